"""Decoder-serving operators are seen by whatever torch puts between a call and its kernel: tracers,
modes, transforms. Without a GPU a stand-in takes the binding's place."""
import types

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx
from torch.overrides import TorchFunctionMode
from torch.utils._python_dispatch import TorchDispatchMode

import triton_msl_b200 as b2
from triton_msl_b200 import decoder_ops

NAMES = ("qk_norm_rope", "kv_cache_write", "kv_cache_read", "kv_cache_attn", "flash_attn_packed")


class Seen(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.names.append(func.name())
        return func(*args, **(kwargs or {}))


class SeenFunctions(TorchFunctionMode):
    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_function__(self, func, types, args=(), kwargs=None):
        self.names.append(func.name() if hasattr(func, "name") else func.__name__)
        return func(*args, **(kwargs or {}))


def stand_in():
    """Plain arithmetic under the binding's names: what matters is that the inputs are used."""
    def write(kc, ks, vc, vs, k, v, slots):
        ks.copy_(k.detach().sum().expand(ks.shape))
    return types.SimpleNamespace(
        qk_norm_rope=lambda q, k, table, pos, qw, kw, eps, inter: (q * 2 + (0 if qw is None else qw), k * 3),
        kv_cache_write=write,
        kv_cache_read=lambda kc, ks, vc, vs, slots, dtype: (ks.to(dtype).sum() + slots.to(dtype), slots.to(dtype)),
        kv_cache_attn=lambda q, kc, ks, vc, vs, table, lengths, scale: q * lengths.sum(),
        flash_attn_packed=lambda q, k, v, cu_q, cu_k, causal, scale: q + cu_q.sum(),
        **{"direct_" + n: getattr(decoder_ops._native(), "direct_" + n, None) for n in NAMES})


def layer(q, k, slots, device):
    """Every operator once."""
    at = slots.int()
    table = torch.ones(8, 64, device=device)
    cache = b2.KVCache(*(torch.zeros(*s, device=device, dtype=t) for s, t in (
        ((1, 2, 16, 32), torch.uint8), ((1, 2, 16, 1, 2), torch.bfloat16)) * 2))
    a, b = b2.qk_norm_rope(q, k, table, at)
    b2.kv_cache_write(cache, b, k, slots)
    kr, vr = b2.kv_cache_read(cache, slots, torch.float32)
    cu, pages = torch.tensor([0, 6], device=device, dtype=torch.int32), torch.zeros(1, 1, device=device, dtype=torch.int32)
    o = b2.flash_attn_packed(a, b, k, cu)
    return a, b, kr, vr, o, b2.kv_cache_attn(a[-1:], cache, pages, at[-1:] + 1)


def inputs(device, seed):
    g = torch.Generator().manual_seed(seed)
    return (*(torch.randn(6, h, 64, generator=g).half().to(device) for h in (4, 2)),
            torch.randperm(8, generator=g)[:6].to(device))


def names_in(graph):
    return " ".join(str(n) for n in graph.nodes())


def run_all(device):
    def f(q, k, slots):
        return layer(q, k, slots, device)
    one, two = inputs(device, 1), inputs(device, 2)
    want = [f(*one), f(*two)]

    def same(got, ref):
        return all(torch.equal(x, y) for x, y in zip(got, ref))
    # recorded calls are made again with other inputs
    traced = torch.jit.trace(f, one, check_trace=False)
    assert all(f"b2msl::{n}" in names_in(traced.inlined_graph) for n in NAMES)
    assert same(traced(*two), want[1])
    for kw in ({}, dict(pre_dispatch=True), dict(tracing_mode="fake")):
        graph = make_fx(f, **kw)(*one)
        assert all(f"b2msl.{n}" in graph.code for n in NAMES), kw
        assert same(graph(*two), want[1])
    # modes see the calls
    for mode in (Seen(), SeenFunctions()):
        with mode:
            assert same(f(*one), want[0])
        assert {f"b2msl::{n}" for n in NAMES} <= {n.removesuffix(".default") for n in mode.names}
    # transforms take them apart
    table, at = torch.ones(8, 64, device=device), one[2].int()
    got = torch.vmap(lambda x: b2.qk_norm_rope(x, one[1], table, at)[0])(torch.stack([one[0], two[0]]))
    assert same(got, [b2.qk_norm_rope(x[0], one[1], table, at)[0] for x in (one, two)])
    # a default device is nobody who looks on, and leaves the results alone
    with torch.device(device):
        assert same(f(*one), want[0])
    with torch.no_grad(), torch.inference_mode():
        assert same(f(*one), want[0])


@pytest.mark.filterwarnings("ignore")
def test_tracers_modes_and_transforms_see_the_operators(monkeypatch):
    monkeypatch.setattr(decoder_ops, "_bound", stand_in())
    run_all("cpu")


@pytest.mark.gpu
@pytest.mark.filterwarnings("ignore")
def test_tracers_modes_and_transforms_see_the_operators_on_the_gpu():
    run_all("cuda")
    assert b2.device_status(0) == 0


@pytest.mark.gpu
def test_ordinary_calls_go_directly(monkeypatch):
    native = decoder_ops._native()
    calls = []

    def counted(name):
        def call(*args):
            out = getattr(native, name)(*args)
            calls.append((name, out is not NotImplemented))
            return out
        return call
    monkeypatch.setattr(decoder_ops, "_bound", types.SimpleNamespace(
        **{n: counted(n) for m in NAMES for n in (m, "direct_" + m)}))
    args = inputs("cuda", 3)
    for around in (torch.no_grad(), torch.inference_mode(), torch.device("cuda"), torch.autocast("cuda")):
        with around:
            layer(*args, "cuda")
    assert len(calls) == 4 * len(NAMES) and all(n.startswith("direct_") and done for n, done in calls)
    w = torch.nn.Parameter(torch.ones(64, device="cuda").half(), requires_grad=False)
    b2.qk_norm_rope(*args[:2], torch.ones(8, 64, device="cuda"), args[2], w, w)
    assert calls[-1] == ("direct_qk_norm_rope", True)


def gradients(device):
    q, k, slots = inputs(device, 4)
    table, cu, at = torch.ones(8, 64, device=device), torch.tensor([0, 6], device=device, dtype=torch.int32), slots.int()
    cache = b2.KVCache(*(torch.zeros(*s, device=device, dtype=t) for s, t in (
        ((1, 2, 16, 32), torch.uint8), ((1, 2, 16, 1, 2), torch.bfloat16)) * 2))
    pages, w = torch.zeros(1, 1, device=device, dtype=torch.int32), torch.ones(64, device=device).half()
    calls = [lambda q, k, w: b2.qk_norm_rope(q, k, table, at, w, w), lambda q, k, w: b2.flash_attn_packed(q, k, k, cu),
             lambda q, k, w: b2.kv_cache_attn(q[:1], cache, pages, at[:1])]
    for i, call in enumerate(calls):
        for wants in (0, 1, 2)[:(3, 2, 1)[i]]:
            x = [y.detach().requires_grad_(j == wants) for j, y in enumerate((q, k, w))]
            out = call(*x)
            first = out[0] if isinstance(out, tuple) else out
            assert first.requires_grad
            with pytest.raises(RuntimeError, match="b2msl::.* forward-only"):
                first.float().sum().backward()
            with torch.no_grad():
                quiet = call(*x)
            quiet = quiet[0] if isinstance(quiet, tuple) else quiet
            assert not quiet.requires_grad and torch.equal(quiet, first)
    # the cache takes values and no gradients
    b2.kv_cache_write(cache, k.detach().requires_grad_(), k, slots)
    assert not any(t.requires_grad for t in cache)


def test_a_backward_pass_is_refused(monkeypatch):
    monkeypatch.setattr(decoder_ops, "_bound", stand_in())
    gradients("cpu")


@pytest.mark.gpu
def test_a_backward_pass_is_refused_on_the_gpu():
    gradients("cuda")
    b2.device_status(0)
