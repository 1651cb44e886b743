"""Decoder-serving operators without a GPU: the table of rotary angles, the refusals of the C ABI
(validation precedes any CUDA call) and of the Python operators, and their shapes under tracing."""
import ctypes
import math

import pytest
import torch

import triton_msl_b200 as b2
from triton_msl_b200 import _lib

_I64x4, _I64x5, _I64x6, _I64x8, _I64x12 = (ctypes.c_int64 * n for n in (4, 5, 6, 8, 12))


# ------------------------------------------------------------------ rope_table
@pytest.mark.parametrize("length,rot,base", [(0, 8, 1e4), (1, 2, 1e4), (33, 128, 1e4), (100, 64, 5e5)])
def test_rope_table_angles(length, rot, base):
    t = b2.rope_table(length, rot, base, device="cpu")
    assert t.shape == (length, rot) and t.dtype == torch.float32
    for p in range(0, length, 7):
        for i in range(0, rot // 2, 5):
            a = p * base ** (-2 * i / rot)
            # one rounding to fp32 of a value at most 1
            assert abs(t[p, i].item() - math.cos(a)) <= 2.0 ** -24
            assert abs(t[p, rot // 2 + i].item() - math.sin(a)) <= 2.0 ** -24


def test_rope_table_linear_is_a_slower_clock():
    fast, slow = b2.rope_table(16, 32, device="cpu"), b2.rope_table(64, 32, scaling="linear", factor=4, device="cpu")
    assert torch.equal(fast, slow[::4])


def test_rope_table_ntk_keeps_the_fastest_pair_and_stretches_the_slowest():
    rot, f = 64, 8.0
    plain, ntk = b2.rope_table(4096, rot, device="cpu"), b2.rope_table(4096, rot, scaling="ntk", factor=f, device="cpu")
    assert torch.equal(plain[:, 0], ntk[:, 0])
    angle = math.acos(ntk[4000, rot // 2 - 1].double().item())
    want = 4000 * 1e4 ** (-(rot - 2) / rot) / f
    # acos of an fp32 cosine near angle `want`: 2^-25 / sin(want)
    assert abs(angle - want) <= 2.0 ** -24 / math.sin(want)


def test_rope_table_by_parts_blends_between_the_two():
    rot, f, orig = 64, 4.0, 2048
    t = b2.rope_table(512, rot, scaling="by_parts", factor=f, original_length=orig, device="cpu").double()
    gain = 0.1 * math.log(f) + 1
    for i in range(rot // 2):
        freq = 1e4 ** (-2 * i / rot)
        turns = orig * freq / (2 * math.pi)
        keep = min(1.0, max(0.0, (turns - 1) / 31))
        a = 300 * (freq * keep + freq / f * (1 - keep))
        assert abs(t[300, i].item() - gain * math.cos(a)) <= 2.0 ** -23
        assert abs(t[300, rot // 2 + i].item() - gain * math.sin(a)) <= 2.0 ** -23


@pytest.mark.parametrize("kw", [dict(rot_dim=7), dict(length=-1), dict(scaling="other"), dict(base=0.0),
                                dict(scaling="by_parts"), dict(scaling="ntk", rot_dim=2)])
def test_rope_table_refusals(kw):
    args = dict(length=8, rot_dim=8, device="cpu") | kw
    with pytest.raises(ValueError):
        b2.rope_table(**args)


# --------------------------------------------------------------- C ABI refusals
ONE = ctypes.c_void_p(16)  # never followed: every call below is refused first


def _rope(T=4, Hq=2, Hk=1, D=64, R=64, P=8, pos=_lib.B2_I32, dt=_lib.B2_BF16, q=ONE, table=ONE):
    return _lib.lib().b2_qk_norm_rope(q, ONE, ONE, ONE, None, None, table, ONE, pos, T, Hq, Hk, D, R, P,
                                      _I64x8(*[64] * 8), 1e-6, 0, dt, None)


@pytest.mark.parametrize("kw,status", [
    (dict(T=-1), _lib.B2_EINVAL), (dict(R=65), _lib.B2_EINVAL), (dict(R=66), _lib.B2_EINVAL),
    (dict(D=63, R=62), _lib.B2_EINVAL), (dict(D=514, R=64), _lib.B2_EUNSUPPORTED),
    (dict(dt=_lib.B2_I64), _lib.B2_EINVAL), (dict(pos=_lib.B2_F32), _lib.B2_EINVAL),
    (dict(q=None), _lib.B2_EINVAL), (dict(table=None), _lib.B2_EINVAL), (dict(T=1 << 31), _lib.B2_EINVAL),
    (dict(T=0), _lib.B2_OK), (dict(Hq=0, Hk=0), _lib.B2_OK)])
def test_rope_abi(kw, status):
    assert _rope(**kw) == status
    assert bool(_lib.lib().b2_last_error()) == (status != _lib.B2_OK)


def _cache_rows(write=True, T=4, pages=4, H=2, page=16, D=128, group=64, dt=_lib.B2_F16, slots=_lib.B2_I64,
                k=ONE, codes=ONE):
    L = _lib.lib()
    shape, strides = _I64x5(pages, H, page, D, group), _I64x4(256, 128, 256, 128)
    if write:
        return L.b2_kv_cache_write(k, ONE, codes, ONE, ONE, ONE, ONE, slots, T, shape, strides, dt, None)
    return L.b2_kv_cache_read(k, ONE, codes, ONE, ONE, ONE, ONE, slots, T, shape, strides, dt, None)


@pytest.mark.parametrize("write", [True, False])
@pytest.mark.parametrize("kw,status", [
    (dict(T=-1), _lib.B2_EINVAL), (dict(D=96), _lib.B2_EUNSUPPORTED), (dict(group=32), _lib.B2_EUNSUPPORTED),
    (dict(D=64, group=128), _lib.B2_EUNSUPPORTED), (dict(H=0), _lib.B2_EINVAL), (dict(page=0), _lib.B2_EINVAL),
    (dict(pages=1 << 28), _lib.B2_EINVAL), (dict(dt=_lib.B2_I32), _lib.B2_EINVAL),
    (dict(slots=_lib.B2_F16), _lib.B2_EINVAL), (dict(k=None), _lib.B2_EINVAL), (dict(codes=None), _lib.B2_EINVAL),
    (dict(codes=ctypes.c_void_p(24)), _lib.B2_EINVAL), (dict(T=1 << 30), _lib.B2_EINVAL), (dict(T=0), _lib.B2_OK)])
def test_cache_rows_abi(write, kw, status):
    assert _cache_rows(write, **kw) == status


def _attn(B=2, N=1, Hq=4, H=2, D=128, group=64, page=16, max_pages=4, scale=0.1, dt=_lib.B2_F16, q=ONE, table=ONE):
    return _lib.lib().b2_kv_cache_attn(q, ONE, ONE, ONE, ONE, ONE, table, ONE, B, N, Hq, max_pages, max_pages,
                                       _I64x5(8, H, page, D, group), _I64x6(*[512] * 6), scale, dt, None, 0, None)


@pytest.mark.parametrize("kw,status", [
    (dict(B=-1), _lib.B2_EINVAL), (dict(Hq=5), _lib.B2_EINVAL), (dict(page=24), _lib.B2_EUNSUPPORTED),
    (dict(D=80), _lib.B2_EUNSUPPORTED), (dict(scale=math.inf), _lib.B2_EINVAL), (dict(scale=math.nan), _lib.B2_EINVAL),
    (dict(dt=9), _lib.B2_EINVAL), (dict(q=None), _lib.B2_EINVAL), (dict(table=None), _lib.B2_EINVAL),
    (dict(B=1 << 31), _lib.B2_EINVAL), (dict(max_pages=1 << 27), _lib.B2_EINVAL), (dict(B=0), _lib.B2_OK),
    (dict(N=0), _lib.B2_OK), (dict(H=1 << 20, Hq=1 << 20, page=1024), _lib.B2_EINVAL)])
def test_cache_attn_abi(kw, status):
    assert _attn(**kw) == status


def _packed(B=2, Tq=8, Tk=8, Hq=4, Hk=2, D=64, scale=0.1, dt=_lib.B2_F16, q=ONE, cu=ONE):
    return _lib.lib().b2_fa_packed(q, ONE, ONE, ONE, cu, ONE, B, Tq, Tk, Hq, Hk, D, _I64x12(*[64] * 12), scale, 1,
                                   dt, None, 0, None)


@pytest.mark.parametrize("kw,status", [
    (dict(B=-1), _lib.B2_EINVAL), (dict(Hq=3), _lib.B2_EINVAL), (dict(Hk=0), _lib.B2_EINVAL),
    (dict(D=129), _lib.B2_EUNSUPPORTED), (dict(D=0), _lib.B2_EINVAL), (dict(scale=math.nan), _lib.B2_EINVAL),
    (dict(dt=_lib.B2_I32), _lib.B2_EINVAL), (dict(q=None), _lib.B2_EINVAL), (dict(cu=None), _lib.B2_EINVAL),
    (dict(Tq=1 << 30), _lib.B2_EINVAL), (dict(Tq=0), _lib.B2_OK), (dict(Hq=0), _lib.B2_OK)])
def test_packed_abi(kw, status):
    assert _packed(**kw) == status


# ------------------------------------------------------------- Python, no device
def test_no_cpu_path():
    x = torch.randn(3, 2, 64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        b2.qk_norm_rope(x, x, b2.rope_table(4, 64, device="cpu"), torch.zeros(3, dtype=torch.int32))
    cache = b2.kv_cache_alloc(2, 2, 64, 16, device="cpu")
    with pytest.raises(RuntimeError, match="no CPU path"):
        b2.kv_cache_write(cache, x, x, torch.arange(3))
    with pytest.raises(RuntimeError, match="no CPU path"):
        b2.kv_cache_attn(x, cache, torch.zeros(3, 1, dtype=torch.int32), torch.ones(3, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="no CPU path"):
        b2.flash_attn_packed(x, x, x, torch.tensor([0, 3], dtype=torch.int32))


@pytest.mark.parametrize("kw", [dict(head_dim=96), dict(group=32), dict(page_size=24), dict(page_size=0),
                                dict(pages=-1), dict(heads=0), dict(head_dim=64, group=128)])
def test_cache_alloc_refusals(kw):
    args = dict(pages=2, heads=2, head_dim=128, page_size=16, group=64, device="cpu") | kw
    with pytest.raises(ValueError):
        b2.kv_cache_alloc(**args)


def test_cache_alloc_layout():
    c = b2.kv_cache_alloc(3, 5, 128, page_size=32, group=64, device="cpu")
    assert c.k_codes.shape == c.v_codes.shape == (3, 5, 32, 64) and c.k_codes.dtype == torch.uint8
    assert c.k_scales.shape == c.v_scales.shape == (3, 5, 32, 2, 2) and c.k_scales.dtype == torch.bfloat16
    assert c.page_size == 32 and c.head_dim == 128


def test_shapes_under_tracing():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        q, k = torch.empty(6, 8, 64, device="cuda"), torch.empty(6, 2, 64, device="cuda")
        table = torch.empty(32, 64, device="cuda")
        qo, ko = b2.qk_norm_rope(q, k, table, torch.empty(6, dtype=torch.int32, device="cuda"))
        assert qo.shape == q.shape and ko.shape == k.shape
        c = b2.kv_cache_alloc(4, 2, 64, 16, device="cuda")
        slots = torch.empty(6, dtype=torch.int64, device="cuda")
        b2.kv_cache_write(c, k, k, slots)
        kr, vr = b2.kv_cache_read(c, slots, torch.float16)
        assert kr.shape == vr.shape == k.shape and kr.dtype == torch.float16
        o = b2.kv_cache_attn(q.view(6, 1, 8, 64), c, torch.empty(6, 2, dtype=torch.int32, device="cuda"),
                             torch.empty(6, dtype=torch.int32, device="cuda"))
        assert o.shape == (6, 1, 8, 64)
        p = b2.flash_attn_packed(q, k, k, torch.empty(3, dtype=torch.int32, device="cuda"))
        assert p.shape == q.shape
