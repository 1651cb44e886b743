"""The in-tree build: which binding is loaded, and builds that are asked for at once."""
import subprocess
import sys
import threading

import pytest
import torch

from triton_msl_b200 import _build, decoder_ops


def test_a_binding_for_another_torch_is_not_loaded(monkeypatch):
    here = _build.binding_path()
    assert torch.__version__ in here.name and here.suffix == ".so"
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    assert _build.binding_path() != here
    monkeypatch.setattr(decoder_ops, "_bound", None)
    monkeypatch.setenv("B2MSL_NO_AUTOBUILD", "1")
    with pytest.raises(RuntimeError, match="torch-0.0.1.so is missing"):
        decoder_ops._native()


def test_a_missing_binding_is_built(monkeypatch, tmp_path):
    monkeypatch.setattr(_build, "binding_path", lambda: tmp_path / "_decoder.so")
    monkeypatch.setattr(decoder_ops, "_bound", None)
    built = []

    def build():
        built.append(1)
        _build._build_binding(False)
    monkeypatch.setattr(_build, "build", build)
    native = decoder_ops._native()
    assert built and native.__file__ == str(tmp_path / "_decoder.so") and hasattr(native, "direct_kv_cache_attn")


def test_builds_exclude_one_another(monkeypatch):
    inside, worst = [], []

    def one(*args):
        inside.append(1)
        worst.append(len(inside))
        threading.Event().wait(0.05)
        inside.pop()
    monkeypatch.setattr(_build, "_build", one)
    threads = [threading.Thread(target=_build.build) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert worst == [1] * 4
    # a process waits as well
    with _build._alone():
        p = subprocess.Popen([sys.executable, "-c", "import fcntl, sys; fcntl.flock(open(sys.argv[1], 'w'), fcntl.LOCK_EX)",
                              str(_build.BUILD / ".lock")])
        with pytest.raises(subprocess.TimeoutExpired):
            p.wait(1)
    assert p.wait(60) == 0
