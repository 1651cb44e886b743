"""Decoder-serving operators on the GPU against plain 64-bit implementations.

Tolerances, derived before the first run. u(T) is half a unit in the last place of the output
type relative to 1: 2^-8 bf16, 2^-11 fp16, 2^-24 fp32.
  * rotation and norm: fp32 arithmetic (a sum of D <= 512 squares, rsqrt, under ten roundings:
    below 1e-5 of the row's largest value), then one rounding to the output type.
  * cache: a code is the nearest integer of (x - low) * (1/scale), so it lies within
    0.5 + 16 * 2^-22 of the quotient; low and scale follow their definition exactly.
  * attention over the cache: a key's weight is rounded to fp16 (2^-11), and its score carries an
    fp32 error below 1e-4 (sums of 128 products, scores below 2^6), so the weight's relative error
    stays below 6e-4; the weights multiply values of at most max|v| twice (codes and lowest value):
    2e-3 * max|v|, then the output's rounding.
  * packed attention: a weight is rounded to the input type (u), its exponential is within 1.1e-4;
    (u + 3e-4) * max|v|, then the output's rounding; fp32 inputs: 1e-4 as everywhere in this suite.
"""
import math

import pytest
import torch

import triton_msl_b200 as b2
from triton_msl_b200 import _lib

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


@pytest.fixture(autouse=True)
def _status():
    b2.device_status(0)
    yield
    assert b2.device_status(0) in (0,), "a kernel left a status bit"


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def check(got, ref, atol, dtype):
    got, ref = got.double(), ref.double()
    assert got.shape == ref.shape
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    # what the output type cannot hold is an infinity in it
    ref = torch.where(ref.abs() > torch.finfo(dtype).max, ref.sign() * math.inf, ref)
    fine = torch.isfinite(ref)
    assert torch.equal(got[~fine & ~torch.isnan(ref)], ref[~fine & ~torch.isnan(ref)])
    over = ((got - ref).abs() - atol - U[dtype] * ref.abs())[fine]
    assert over.numel() == 0 or over.max().item() <= 0, f"exceeds the tolerance by {over.max().item():.3g}"


# ------------------------------------------------------------- q/k norm, rotation
def rope_ref(x, w, table, pos, eps, inter):
    y = x.double()
    if w is not None:
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * w.double()
    R = table.shape[1]
    rows = table.double()[pos.long()][:, None]
    c, s = rows[..., :R // 2], rows[..., R // 2:]
    out = y.clone()
    if inter:
        a, b = y[..., 0:R:2], y[..., 1:R:2]
        out[..., 0:R:2], out[..., 1:R:2] = a * c - b * s, b * c + a * s
    else:
        a, b = y[..., :R // 2], y[..., R // 2:R]
        out[..., :R // 2], out[..., R // 2:R] = a * c - b * s, b * c + a * s
    return out


def rope_check(q, k, table, pos, qw, kw, eps, inter):
    qo, ko = b2.qk_norm_rope(q, k, table, pos, qw, kw, eps=eps, interleaved=inter)
    assert b2.last_kernel() == "qk_norm_rope"
    for got, x, w in ((qo, q, qw), (ko, k, kw)):
        assert got.is_contiguous() and got.dtype == x.dtype
        ref = rope_ref(x, w, table, pos, eps, inter)
        top = ref.abs().nan_to_num(0).amax(-1, keepdim=True) if ref.numel() else ref
        check(got, ref, 1e-5 * top, x.dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("T,Hq,Hk,D,R,norm", [
    (1, 1, 1, 128, 128, True), (5, 32, 8, 128, 128, True), (67, 7, 3, 64, 32, False), (33, 5, 5, 96, 96, True),
    (17, 6, 2, 80, 40, True), (9, 3, 1, 256, 128, True), (4, 2, 2, 512, 512, True), (3, 2, 1, 34, 6, True),
    (2, 9, 1, 64, 0, True), (130, 4, 0, 64, 64, False), (6, 1, 2, 2, 2, True), (3, 1, 1, 510, 254, True)])
def test_rope(dtype, inter, T, Hq, Hk, D, R, norm):
    g = gen(T * 1000 + D + R)
    q, k = (randn(g, T, h, D).mul(2).to(dtype) for h in (Hq, Hk))
    qw, kw = ((1 + 0.3 * randn(g, D)).to(dtype) if norm else None for _ in range(2))
    table = b2.rope_table(300, R)
    pos = torch.randint(0, 300, (T,), generator=g, device="cuda", dtype=torch.int64 if T % 2 else torch.int32)
    rope_check(q, k, table, pos, qw, kw, 1e-6, inter)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("T,Hq,Hk,D,R,norm", [
    (1800, 32, 8, 128, 64, True), (3001, 32, 8, 128, 128, True), (4500, 33, 5, 128, 128, True), (9001, 13, 1, 64, 32, False),
    (9000, 14, 2, 40, 24, True), (1500, 33, 5, 256, 256, True), (9000, 10, 0, 128, 128, True), (18000, 6, 6, 32, 32, False)])
def test_rope_many_heads_at_a_time(dtype, inter, T, Hq, Hk, D, R, norm):
    # enough tokens for lane groups of 8, 16 and 32 heads, whole and not; q and k inside one projection
    g = gen(T + D + R)
    qkv = randn(g, T, Hq + 2 * Hk, D).mul(2).to(dtype)
    qkv[T // 2, 1, D - 1] = math.nan  # stays in its head
    qw, kw = ((1 + 0.3 * randn(g, D)).to(dtype) if norm else None for _ in range(2))
    table = b2.rope_table(300, R)
    pos = torch.randint(0, 300, (T,), generator=g, device="cuda", dtype=torch.int64 if T % 2 else torch.int32)
    rope_check(qkv[:, :Hq], qkv[:, Hq:Hq + Hk], table, pos, qw, kw, 1e-6, inter)


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("shift", [0, 1, 2, 4])
def test_rope_views_and_alignment(inter, shift):
    # q and k as parts of a projection that starts `shift` elements into a buffer; norm of q alone
    g = gen(shift)
    T, Hq, Hk, D = 37, 6, 2, 64
    flat = randn(g, shift + T * (Hq + 2 * Hk) * D + 64).bfloat16()
    qkv = flat[shift:shift + T * (Hq + 2 * Hk) * D].view(T, Hq + 2 * Hk, D)
    w = (1 + 0.1 * randn(g, D)).bfloat16()
    table = b2.rope_table(64, D)
    pos = torch.arange(T, device="cuda", dtype=torch.int32)
    rope_check(qkv[:, :Hq], qkv[:, Hq:Hq + Hk], table, pos, w, None, 1e-5, inter)
    # heads outermost, and a channel stride that is not one
    rope_check(qkv[:, :Hq].transpose(0, 1).contiguous().transpose(0, 1), qkv[:, Hq:Hq + Hk], table, pos, None, w, 1e-5, inter)
    rope_check(qkv[:, :Hq].transpose(1, 2).contiguous().transpose(1, 2), qkv[:, Hq:Hq + Hk], table, pos, w, w, 1e-5, inter)


def test_rope_empty():
    table, e = b2.rope_table(8, 64), torch.empty(0, 4, 64, device="cuda")
    qo, ko = b2.qk_norm_rope(e, e, table, torch.empty(0, dtype=torch.int32, device="cuda"))
    assert qo.shape == ko.shape == e.shape


def test_rope_extremes():
    # a zero row keeps eps in charge; a NaN stays in its own row; an infinity where nothing rotates stays itself
    table = b2.rope_table(16, 32)
    q = torch.ones(4, 2, 64, device="cuda")
    q[0, 0] = 0
    q[1, 1, 3] = math.nan
    q[2, 0, 40] = math.inf
    pos = torch.tensor([3, 4, 5, 15], device="cuda")
    qo, _ = b2.qk_norm_rope(q, q, table, pos)
    check(qo, rope_ref(q, None, table, pos, 1e-6, False), 1e-5, torch.float32)
    w = torch.ones(64, device="cuda")
    qo, _ = b2.qk_norm_rope(q[:2], q[:2], table, pos[:2], w, w)
    assert torch.equal(qo[0, 0], torch.zeros(64, device="cuda"))
    assert torch.isnan(qo[1, 1]).all() and not torch.isnan(qo[1, 0]).any()


def test_rope_position_outside_the_table():
    table = b2.rope_table(16, 32)
    q = torch.ones(4, 2, 64, device="cuda")
    pos = torch.tensor([0, 16, -1, 15], device="cuda", dtype=torch.int32)
    qo, ko = b2.qk_norm_rope(q, q, table, pos)
    assert b2.device_status(0) == _lib.STATUS_BAD_INDEX and b2.device_status(0) == 0
    for o in (qo, ko):
        assert torch.isnan(o[1:3, :, :32]).all() and not torch.isnan(o[1:3, :, 32:]).any()
        assert not torch.isnan(o[0]).any() and not torch.isnan(o[3]).any()


@pytest.mark.parametrize("bad", ["shape", "dtype", "k", "pos", "posdtype", "weight", "table", "odd"])
def test_rope_refusals(bad):
    q = torch.zeros(4, 2, 64, device="cuda")
    a = dict(q=q, k=q, table=b2.rope_table(8, 64), positions=torch.zeros(4, dtype=torch.int32, device="cuda"))
    a |= {"shape": dict(q=q[0]), "dtype": dict(q=q.to(torch.float64), k=q.to(torch.float64)), "k": dict(k=q.half()),
          "pos": dict(positions=torch.zeros(3, dtype=torch.int32, device="cuda")),
          "posdtype": dict(positions=torch.zeros(4, device="cuda")), "weight": dict(q_weight=torch.ones(63, device="cuda")),
          "table": dict(table=b2.rope_table(8, 64).half()), "odd": dict(table=torch.zeros(8, 66, device="cuda"))}[bad]
    with pytest.raises((ValueError, TypeError)):
        b2.qk_norm_rope(**a)


# ------------------------------------------------------------------ 4-bit cache
def down(x):  # fp64 -> the largest bf16 value not above
    y = x.float().to(torch.bfloat16).double()
    lower = torch.nextafter(x.float().to(torch.bfloat16), torch.tensor(-math.inf, device=x.device, dtype=torch.bfloat16)).double()
    return torch.where(y <= x, y, lower)


def row_codes(codes):
    """Codes [..., D/2] as integers [..., D], by the documented layout."""
    D = 2 * codes.shape[-1]
    out = torch.empty(*codes.shape[:-1], D, dtype=torch.int64, device=codes.device)
    for c in range(D):
        word = (c % 64 // 8) * (D // 64) + c // 64
        out[..., c] = (codes[..., 4 * word + (c % 8) // 2] >> (4 * (c % 2))) & 15
    return out


def row_values(codes, scales):
    D, n = 2 * codes.shape[-1], scales.shape[-2]
    s = scales.double().repeat_interleave(D // n, -2)
    return row_codes(codes).double() * s[..., 0] + s[..., 1]


def pick(cache, slots):
    page, off = slots.long() // cache.page_size, slots.long() % cache.page_size
    return [t[page, :, off] for t in cache]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,H,D,group,page", [(1, 1, 64, 64, 16), (1, 8, 128, 128, 16), (77, 3, 128, 64, 32),
                                              (300, 5, 64, 64, 64), (130, 2, 128, 128, 128)])
def test_cache_write_and_read(dtype, T, H, D, group, page):
    g = gen(T + D)
    cache = b2.kv_cache_alloc(T // page + 2, H, D, page, group)
    k, v = (randn(g, T, H, D) * torch.exp(2 * randn(g, T, H, 1))).to(dtype), (randn(g, T, H, D) + 3).to(dtype)
    slots = torch.randperm(cache.k_codes.shape[0] * page, generator=g, device="cuda")[:T]
    if T % 2:
        slots = slots.int()
    b2.kv_cache_write(cache, k, v, slots)
    assert b2.last_kernel() == "kv_cache_write"
    kc, ks, vc, vs = pick(cache, slots)
    for x, codes, scales in ((k, kc, ks), (v, vc, vs)):
        y = x.double().unflatten(-1, (-1, group))
        low, step = scales[..., 1].double(), scales[..., 0].double()
        assert torch.equal(low, down(y.amin(-1)))
        exact = (y.amax(-1) - low) / 15
        # rounded up to bf16 from an fp32 value of three roundings
        assert (step >= exact * (1 - 2.0 ** -22)).all() and (step <= exact * (1 + 2.0 ** -7 + 2.0 ** -21)).all()
        code = row_codes(codes).unflatten(-1, (-1, group)).double()
        off = (code - (y - low[..., None]) / step[..., None]).abs()
        assert off.max().item() <= 0.5 + 16 * 2.0 ** -22
    for out in (torch.float32, dtype):
        kr, vr = b2.kv_cache_read(cache, slots, out)
        assert b2.last_kernel() == "kv_cache_read" and kr.dtype == out
        for got, codes, scales in ((kr, kc, ks), (vr, vc, vs)):
            assert torch.equal(got, row_values(codes, scales).float().to(out))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_cache_codes_follow_their_definition(dtype):
    # bit for bit in fp32, values half way between two codes among them (in 16 bits there are many)
    g = gen(8)
    cache = b2.kv_cache_alloc(64, 4, 128, 16, 64)
    x = (torch.round(randn(g, 1000, 4, 128) * 16) / 8).to(dtype)
    slots = torch.arange(1000, device="cuda")
    b2.kv_cache_write(cache, x, -x, slots)
    kc, ks, vc, vs = pick(cache, slots)
    halves = 0
    for y, codes, scales in ((x, kc, ks), (-x, vc, vs)):
        y = y.float().unflatten(-1, (2, 64))
        step, low = scales[..., :1].float(), scales[..., 1:].float()
        quotient = (y - low) * (1.0 / step)
        halves += (quotient % 1 == 0.5).sum().item()
        assert torch.equal(row_codes(codes).unflatten(-1, (2, 64)), torch.round(quotient).long())
    assert halves > 100


def test_cache_strides_and_alignment():
    g = gen(5)
    T, H, D = 19, 3, 64
    for shift in (0, 1):
        flat = randn(g, T * 3 * H * D + 8).half()
        kv = flat[shift:shift + T * 3 * H * D].view(T, 3 * H, D)
        views = (kv[:, :H], kv[:, H:2 * H])
        hs = tuple(x.transpose(0, 1).contiguous().transpose(0, 1) for x in views)
        cs = tuple(x.transpose(1, 2).contiguous().transpose(1, 2) for x in views)
        slots = torch.arange(T, device="cuda") + 3
        caches = []
        for k, v in (views, hs, cs, tuple(x.contiguous() for x in views)):
            caches.append(b2.kv_cache_alloc(2, H, D, 16, 64))
            b2.kv_cache_write(caches[-1], k, v, slots)
        for c in caches[:-1]:
            assert all(torch.equal(a, b) for a, b in zip(c, caches[-1]))


def test_cache_padding_and_bounds():
    cache = b2.kv_cache_alloc(2, 2, 128, 16, 64)
    g = gen(6)
    k = randn(g, 6, 2, 128)
    before = [t.clone() for t in cache]
    slots = torch.tensor([-1, 5, -7, 31, 32, 1 << 40], device="cuda")
    b2.kv_cache_write(cache, k, k + 1, slots)
    assert b2.device_status(0) == _lib.STATUS_BAD_INDEX
    touched = torch.zeros(2, 16, dtype=torch.bool, device="cuda")
    touched[0, 5] = touched[1, 15] = True
    for now, then in zip(cache, before):
        now, then = now.transpose(1, 2), then.transpose(1, 2)
        assert torch.equal(now[~touched], then[~touched]) and not torch.equal(now[touched], then[touched])
    kr, vr = b2.kv_cache_read(cache, slots, torch.float32)
    assert b2.device_status(0) == _lib.STATUS_BAD_INDEX
    assert (kr[[0, 2]] == 0).all() and (vr[[0, 2]] == 0).all()
    assert torch.isnan(kr[4:]).all() and torch.isnan(vr[4:]).all()
    assert torch.isfinite(kr[[1, 3]]).all()
    e = torch.empty(0, dtype=torch.int64, device="cuda")
    b2.kv_cache_write(cache, k[:0], k[:0], e)
    assert b2.kv_cache_read(cache, e)[0].shape == (0, 2, 128)


def test_cache_extreme_groups():
    cache = b2.kv_cache_alloc(1, 1, 128, 16, 64)
    x = torch.zeros(8, 1, 128, device="cuda")
    x[0] = 7.25                      # constant: held exactly
    x[1, :, 64:] = 1e-40             # denormal range
    x[2, 0, 5] = math.nan
    x[3, 0, 70] = math.inf
    x[4, 0, 3] = -math.inf
    x[5] = torch.linspace(-3e38, 3e38, 128, device="cuda")   # the range itself overflows
    x[6] = torch.linspace(-1e38, 1e38, 128, device="cuda")
    x[7] = torch.linspace(100, 101, 128, device="cuda")      # a range far below the values
    b2.kv_cache_write(cache, x, x, torch.arange(8, device="cuda"))
    for y in b2.kv_cache_read(cache, torch.arange(8, device="cuda"), torch.float32):
        y = y[:, 0]
        assert (y[0] == 7.25).all()
        assert (y[1, :64] == 0).all() and (y[1, 64:] - 1e-40).abs().max() <= 2e-40
        for r, bad in ((2, 0), (3, 1), (4, 0)):
            assert torch.isnan(y[r, 64 * bad:64 * bad + 64]).all()
            assert not torch.isnan(y[r, 64 - 64 * bad:128 - 64 * bad]).any()
        step = (x[6, 0, 63] - x[6, 0, 0]) / 15
        assert ((y[6] - x[6, 0]).abs() <= 0.52 * step).all()
        # low is at most one bf16 step (0.5) under 100, so a code is at most (0.5 + 0.5)/15
        assert ((y[7] - x[7, 0]).abs() <= 0.52 / 15).all()


@pytest.mark.parametrize("bad", ["heads", "dtype", "v", "slots", "slotdtype", "cache", "scales", "strided"])
def test_cache_refusals(bad):
    c = b2.kv_cache_alloc(2, 2, 64, 16)
    k = torch.zeros(4, 2, 64, device="cuda")
    a = dict(cache=c, k=k, v=k, slots=torch.arange(4, device="cuda"))
    a |= {"heads": dict(k=k[:, :1], v=k[:, :1]), "dtype": dict(k=k.double(), v=k.double()), "v": dict(v=k.half()),
          "slots": dict(slots=torch.arange(3, device="cuda")), "slotdtype": dict(slots=torch.zeros(4, device="cuda")),
          "cache": dict(cache=c._replace(v_codes=c.v_codes[:1])), "scales": dict(cache=c._replace(k_scales=c.k_scales.half())),
          "strided": dict(cache=c._replace(k_codes=c.k_codes.transpose(0, 2).contiguous().transpose(0, 2)))}[bad]
    with pytest.raises((ValueError, TypeError)):
        b2.kv_cache_write(**a)
    if bad in ("cache", "scales", "strided", "slotdtype"):
        with pytest.raises((ValueError, TypeError)):
            b2.kv_cache_read(a["cache"], a["slots"])
    with pytest.raises(TypeError):
        b2.kv_cache_read(c, torch.arange(4, device="cuda"), torch.float64)


# ----------------------------------------------------- attention over the cache
def filled(g, lens, H, D, group, page, extra=1, garbage=True):
    """A cache of sequences of these lengths in shuffled pages; what lies past a length is garbage."""
    need = [max(1, -(-n // page)) for n in lens]
    pages = sum(need) + extra
    cache = b2.kv_cache_alloc(pages, H, D, page, group)
    if garbage:
        cache.k_codes.fill_(0xff)
        cache.v_codes.fill_(0xff)
        cache.k_scales.fill_(math.nan)
        cache.v_scales.fill_(math.inf)
    order = torch.randperm(pages, generator=g, device="cuda", dtype=torch.int32)
    table = torch.full((len(lens), max(need) + 1), 1 << 30, dtype=torch.int32, device="cuda")  # unused entries: no page
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
        t = torch.arange(lens[i], device="cuda")
        slots = table[i].long()[t // page] * page + t % page
        b2.kv_cache_write(cache, randn(g, lens[i], H, D) * 2, randn(g, lens[i], H, D) + 0.5, slots)
    return cache, table


def attn_ref(q, cache, table, lens, scale):
    B, N, Hq, D = q.shape
    H = cache.k_codes.shape[1]
    o = torch.zeros(B, N, Hq, D, dtype=torch.float64, device="cuda")
    top = torch.zeros(B, 1, 1, 1, dtype=torch.float64, device="cuda")
    for b, L in enumerate(lens):
        t = torch.arange(L, device="cuda")
        slots = table[b].long()[t // cache.page_size] * cache.page_size + t % cache.page_size
        kc, ks, vc, vs = pick(cache, slots)
        k, v = row_values(kc, ks), row_values(vc, vs)  # [L, H, D]
        top[b] = v.abs().max() if v.numel() else 0
        for n in range(N):
            keys = max(0, L - N + 1 + n)
            for h in range(Hq if keys else 0):
                kh = h // (Hq // H)
                p = torch.softmax(k[:keys, kh] @ q[b, n, h].double() * scale, 0)
                o[b, n, h] = p @ v[:keys, kh]
    return o, top


def attn_check(q, cache, table, lens, scale=None, kernel=None):
    got = b2.kv_cache_attn(q, cache, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), scale)
    if kernel:
        assert b2.last_kernel() == kernel
    ref, top = attn_ref(q, cache, table, lens, q.shape[-1] ** -0.5 if scale is None else scale)
    assert got.is_contiguous() and got.dtype == q.dtype
    check(got, ref, 2e-3 * top, q.dtype)
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("lens,N,Hq,H,D,group,page", [
    ([1], 1, 1, 1, 64, 64, 16), ([0, 1, 2, 17], 1, 4, 2, 128, 64, 16), ([16, 15, 129, 128], 1, 8, 1, 128, 128, 16),
    ([300, 5], 1, 12, 4, 64, 64, 32), ([700], 1, 32, 8, 128, 64, 64), ([1000, 1, 250], 1, 5, 5, 128, 128, 128),
    ([0, 1, 3, 4, 200], 4, 4, 2, 64, 64, 16), ([130, 2], 3, 14, 2, 128, 64, 16), ([513], 8, 8, 1, 128, 128, 64),
    ([90, 33], 5, 32, 1, 64, 64, 32), ([2500, 40], 2, 6, 2, 128, 64, 48)])
def test_cache_attn(dtype, lens, N, Hq, H, D, group, page):
    g = gen(sum(lens) + N + Hq)
    cache, table = filled(g, lens, H, D, group, page)
    attn_check(randn(g, len(lens), N, Hq, D).to(dtype), cache, table, lens,
               kernel="kv_attn_row" if dtype == torch.float32 else "kv_attn_mma")


def test_cache_attn_many_sequences():
    # more sequences than one scan of the lengths takes at once, most of them short or empty
    g = gen(21)
    lens = [(i * 37) % 61 if i % 5 else 0 for i in range(700)] + [900]
    cache, table = filled(g, lens, 1, 64, 64, 16)
    attn_check(randn(g, len(lens), 1, 2, 64).half(), cache, table, lens)


@pytest.mark.parametrize("D,group,Hq", [(64, 64, 16), (128, 64, 16), (128, 128, 96)])
def test_cache_attn_sums_are_not_shifted(D, group, Hq):
    # results far smaller than the values they are sums of, weights far apart: what rounds the products must not shift
    # their sum. Independent errors of 4e-4 (weights and result rounded to fp16) average out over
    # H * D channels, at 6 sigma; a shift may reach 2^-21 of the values.
    g = gen(23 + D + Hq)
    L, H = 30000, 16
    cache, table = filled(g, [L], H, D, group, 64, extra=0)
    t = torch.arange(L, device="cuda")
    slots = table[0].long()[t // 64] * 64 + t % 64
    b2.kv_cache_write(cache, randn(g, L, H, D) * 2, randn(g, L, H, D), slots)
    q = randn(g, 1, 1, Hq, D).half()
    ref, top = attn_ref(q, cache, table, [L], D ** -0.5)
    got = b2.kv_cache_attn(q, cache, table, torch.tensor([L], dtype=torch.int32, device="cuda"))
    shift = (got.double() - ref).mean().abs().item()
    assert shift <= 2.0**-21 * top.item() + 6 * 4e-4 * ref.square().mean().sqrt().item() / math.sqrt(H * D)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_cache_attn_scales(dtype):
    # large and tiny queries, keys of very different steps, values from 1e-6 to 1e4
    g = gen(22)
    lens, H, D = [333], 2, 128
    cache, table = filled(g, lens, H, D, 64, 16)
    t = torch.arange(333, device="cuda")
    slots = table[0].long()[t // 16] * 16 + t % 16
    k = randn(g, 333, H, D) * torch.exp(randn(g, 333, H, 1))
    v = randn(g, 333, H, D) * torch.exp(randn(g, 333, H, 1) * 4)
    b2.kv_cache_write(cache, k, v, slots)
    for mul in (1e-4, 1.0, 30.0):
        attn_check((randn(g, 1, 2, 8, D) * mul).to(dtype), cache, table, lens)
    attn_check(randn(g, 1, 2, 8, D).to(dtype), cache, table, lens, scale=-0.1)
    attn_check(randn(g, 1, 2, 8, D).to(dtype), cache, table, lens, scale=0.0)
    attn_check(torch.zeros(1, 2, 8, D, device="cuda", dtype=dtype), cache, table, lens)


def test_cache_attn_rising_scores():
    # each later key scores higher, so the running maximum moves all along the sequence
    g = gen(23)
    lens, D = [2000], 64
    cache, table = filled(g, lens, 1, D, 64, 16)
    t = torch.arange(2000, device="cuda")
    slots = table[0].long()[t // 16] * 16 + t % 16
    k = torch.ones(2000, 1, D, device="cuda") * (t[:, None, None] / 200) + 0.1 * randn(g, 2000, 1, D)
    b2.kv_cache_write(cache, k, randn(g, 2000, 1, D), slots)
    q = torch.ones(1, 1, 4, D, device="cuda").half()
    attn_check(q, cache, table, lens)
    attn_check(-q, cache, table, lens)


def test_cache_attn_many_small_weights():
    # one key takes half of the weight, 60000 others share the rest at 2^-16 of it each
    g = gen(29)
    L, D = 60001, 64
    cache, table = filled(g, [L], 1, D, 64, 128)
    t = torch.arange(L, device="cuda")
    slots = table[0].long()[t // 128] * 128 + t % 128
    k = torch.zeros(L, 1, D, device="cuda")
    k[5] = 1.0  # score 11 against 0 with the query below
    b2.kv_cache_write(cache, k, randn(g, L, 1, D) + 2, slots)
    q = torch.full((1, 1, 4, D), 11 * D ** 0.5 / D, device="cuda")
    for dtype in (torch.float16, torch.bfloat16):
        attn_check(q.to(dtype), cache, table, [L])


def test_cache_attn_strides_and_dims():
    g = gen(24)
    lens, Hq, H, D = [40, 70], 4, 2, 64
    cache, table = filled(g, lens, H, D, 64, 16)
    qkv = randn(g, 2, 3, Hq + 2 * H, D).half()
    a = attn_check(qkv[:, :, :Hq], cache, table, lens)
    b = b2.kv_cache_attn(qkv[:, :, :Hq].contiguous(), cache, table.clone(), torch.tensor(lens, dtype=torch.int32, device="cuda"))
    assert torch.equal(a, b)
    odd = randn(g, 2 * 3 * Hq * D + 1).half()[1:].view(2, 3, Hq, D)  # not on a 16-byte boundary
    attn_check(odd, cache, table, lens)
    attn_check(qkv[:, :, :Hq].transpose(2, 3).contiguous().transpose(2, 3), cache, table, lens)
    wide = torch.full((2, 50), 7, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    one = b2.kv_cache_attn(qkv[:, 0, :Hq], cache, wide[:, :table.shape[1]], torch.tensor(lens, dtype=torch.int32, device="cuda"))
    assert one.shape == (2, Hq, D)
    check(one, attn_ref(qkv[:, :1, :Hq], cache, table, lens, D ** -0.5)[0][:, 0], 2e-3 * 20, torch.float16)
    e = b2.kv_cache_attn(qkv[:0, :, :Hq], cache, table[:0], torch.empty(0, dtype=torch.int32, device="cuda"))
    assert e.shape == (0, 3, Hq, D)


def test_cache_attn_poisoned_tokens():
    # a NaN in a token's values reaches the rows that attend it and no others
    g = gen(25)
    lens, Hq, H, D = [50, 60], 4, 2, 128
    cache, table = filled(g, lens, H, D, 64, 16)
    q = randn(g, 2, 4, Hq, D).half()
    lt = torch.tensor(lens, dtype=torch.int32, device="cuda")
    last = table[0].long()[48 // 16] * 16 + 48 % 16  # token 48 of sequence 0: rows 2 and 3 attend it
    k, v = randn(g, 1, H, D), randn(g, 1, H, D)
    b2.kv_cache_write(cache, k, v, last[None])
    clean = b2.kv_cache_attn(q, cache, table, lt)
    v[0, 1, 70] = math.nan  # head 1, second group
    b2.kv_cache_write(cache, k, v, last[None])
    got = b2.kv_cache_attn(q, cache, table, lt)
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[0, 2:, 2:, 64:] = True
    assert torch.isnan(got[bad]).all() and torch.equal(got[~bad], clean[~bad])
    k[0, 0] = math.inf  # now the keys of head 0 as well
    b2.kv_cache_write(cache, k, v, last[None])
    got = b2.kv_cache_attn(q, cache, table, lt)
    bad[0, 2:, :2] = True
    assert torch.isnan(got[bad]).all() and torch.equal(got[~bad], clean[~bad])
    q2 = q.clone()
    q2[1, 1, 3, 9] = math.nan
    got = b2.kv_cache_attn(q2, cache, table, lt)
    bad[1, 1, 3] = True
    assert torch.isnan(got[bad]).all() and torch.equal(got[~bad], clean[~bad])


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_cache_attn_bad_indices(dtype):
    g = gen(26)
    lens, Hq, H, D = [50, 60, 20], 4, 2, 64
    cache, table = filled(g, lens, H, D, 64, 16)
    q = randn(g, 3, 1, Hq, D).to(dtype)
    lt = torch.tensor(lens, dtype=torch.int32, device="cuda")
    clean = b2.kv_cache_attn(q, cache, table, lt)
    for page in (-1, cache.k_codes.shape[0]):
        t2 = table.clone()
        t2[1, 2] = page
        got = b2.kv_cache_attn(q, cache, t2, lt)
        assert b2.device_status(0) == _lib.STATUS_BAD_INDEX
        assert torch.isnan(got[1]).all() and torch.equal(got[[0, 2]], clean[[0, 2]])
    for length in (-3, 16 * table.shape[1] + 1):
        l2 = lt.clone()
        l2[0] = length
        got = b2.kv_cache_attn(q, cache, table, l2)
        assert b2.device_status(0) == _lib.STATUS_BAD_INDEX
        assert torch.isnan(got[0]).all() and torch.equal(got[1:], clean[1:])


def test_cache_past_32_bit_offsets():
    # 70,000 pages of 64 KB of codes: the last ones lie past 2^32 bytes
    H, D, page = 8, 128, 128
    cache = b2.kv_cache_alloc(70000, H, D, page, 128)
    assert cache.k_codes.numel() > 1 << 32
    g = gen(27)
    table = torch.tensor([[69999, 65537, 3]], dtype=torch.int32, device="cuda")
    t = torch.arange(300, device="cuda")
    slots = table[0].long()[t // page] * page + t % page
    k, v = randn(g, 300, H, D).half(), randn(g, 300, H, D).half()
    b2.kv_cache_write(cache, k, v, slots)
    kr, vr = b2.kv_cache_read(cache, slots, torch.float16)
    # half a step of a range of at most 2 * max, plus the widening of the step
    assert (kr - k).abs().max() <= 0.51 * 2 * k.abs().max() / 15 and (vr - v).abs().max() <= 0.51 * 2 * v.abs().max() / 15
    attn_check(randn(g, 1, 1, 32, D).half(), cache, table, [300])


def test_cache_attn_on_another_stream():
    g = gen(28)
    lens, Hq, H, D = [777], 8, 2, 128
    cache, table = filled(g, lens, H, D, 64, 16)
    q = randn(g, 1, 1, Hq, D).bfloat16()
    lt = torch.tensor(lens, dtype=torch.int32, device="cuda")
    want = b2.kv_cache_attn(q, cache, table, lt)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [b2.kv_cache_attn(q, cache, table, lt) for _ in range(8)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(o, want) for o in outs)


@pytest.mark.parametrize("bad", ["dim", "heads", "table", "lengths", "dtype", "lendtype"])
def test_cache_attn_refusals(bad):
    c = b2.kv_cache_alloc(2, 2, 64, 16)
    a = dict(q=torch.zeros(3, 1, 4, 64, device="cuda").half(), cache=c, page_table=torch.zeros(3, 2, dtype=torch.int32, device="cuda"),
             lengths=torch.ones(3, dtype=torch.int32, device="cuda"))
    a |= {"dim": dict(q=torch.zeros(3, 1, 4, 128, device="cuda").half()), "heads": dict(q=torch.zeros(3, 1, 3, 64, device="cuda").half()),
          "table": dict(page_table=a["page_table"][:2]), "lengths": dict(lengths=a["lengths"][:2]),
          "dtype": dict(q=a["q"].double()), "lendtype": dict(lengths=a["lengths"].long())}[bad]
    with pytest.raises((ValueError, TypeError)):
        b2.kv_cache_attn(**a)


# -------------------------------------------------------------- packed prompts
def packed_ref(q, k, v, cu_q, cu_k, causal, scale):
    o = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    top = torch.zeros(q.shape[0], 1, 1, dtype=torch.float64, device="cuda")
    G = q.shape[1] // k.shape[1]
    for b in range(len(cu_q) - 1):
        qs, ks = slice(cu_q[b], cu_q[b + 1]), slice(cu_k[b], cu_k[b + 1])
        Lq, Lk = cu_q[b + 1] - cu_q[b], cu_k[b + 1] - cu_k[b]
        if Lq == 0 or Lk == 0:
            continue
        i, j = torch.arange(Lq, device="cuda")[:, None], torch.arange(Lk, device="cuda")
        kept = (j <= i + Lk - Lq) if causal else torch.ones(Lq, Lk, dtype=torch.bool, device="cuda")
        vv = v[ks].double().repeat_interleave(G, 1).transpose(0, 1)
        s = q[qs].double().transpose(0, 1) @ k[ks].double().repeat_interleave(G, 1).permute(1, 2, 0) * scale
        p = torch.softmax(s.masked_fill(~kept, -math.inf), -1).masked_fill(~kept.any(-1, keepdim=True), 0)
        o[qs] = (p @ vv).transpose(0, 1)
        top[qs] = v[ks].abs().max().double()
    return o, top


def packed_check(q, k, v, lens_q, lens_k=None, causal=True, scale=None, lead=0, kernel=None):
    cu_q = [lead + sum(lens_q[:i]) for i in range(len(lens_q) + 1)]
    lens_k = lens_q if lens_k is None else lens_k
    cu_k = [lead + sum(lens_k[:i]) for i in range(len(lens_k) + 1)] if lens_k is not lens_q else cu_q
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    got = b2.flash_attn_packed(q, k, v, dev(cu_q), None if cu_k is cu_q else dev(cu_k), causal=causal, sm_scale=scale)
    if kernel:
        assert b2.last_kernel() == kernel
    assert got.is_contiguous() and got.dtype == q.dtype
    ref, top = packed_ref(q, k, v, cu_q, cu_k, causal, q.shape[-1] ** -0.5 if scale is None else scale)
    check(got, ref, 1e-4 if q.dtype == torch.float32 else (U[q.dtype] + 3e-4) * top, q.dtype)
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,Hq,Hk,D", [
    ([1], 1, 1, 64), ([1, 2, 3], 4, 2, 128), ([127, 128, 129], 2, 2, 64), ([5, 0, 260, 0, 33], 8, 2, 128),
    ([64, 300], 6, 2, 64), ([513], 8, 1, 128), ([200, 71], 5, 1, 96), ([31, 90], 7, 1, 80), ([40, 17], 3, 3, 40),
    ([257, 1], 12, 4, 32), ([100], 32, 2, 64), ([150], 4, 4, 8), ([640, 300], 4, 1, 128)])
def test_packed(dtype, causal, lens, Hq, Hk, D):
    g = gen(sum(lens) + Hq + D)
    T = sum(lens)
    qkv = randn(g, T, Hq + 2 * Hk, D).to(dtype)
    packed_check(qkv[:, :Hq], qkv[:, Hq:Hq + Hk], qkv[:, Hq + Hk:], lens, causal=causal,
                 kernel="fa_packed_simt" if dtype == torch.float32 else "fa_packed_sm100")


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens_q,lens_k", [([1, 1], [300, 1]), ([5, 130], [260, 400]), ([10, 64], [3, 0]),
                                           ([300, 20], [129, 20]), ([0, 4], [9, 700]), ([140], [1000])])
def test_packed_different_lengths(dtype, causal, lens_q, lens_k):
    g = gen(sum(lens_q) + sum(lens_k))
    q = randn(g, sum(lens_q), 8, 64).to(dtype)
    k, v = randn(g, sum(lens_k), 2, 64).to(dtype), randn(g, sum(lens_k), 2, 64).to(dtype)
    packed_check(q, k, v, lens_q, lens_k, causal=causal)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_packed_tokens_outside_every_sequence(dtype):
    g = gen(31)
    q, k, v = (randn(g, 420, h, 64).to(dtype) for h in (4, 2, 2))
    for x in (q, k, v):  # padding before and after the batch holds anything
        x[:7] = math.nan
        x[7 + 300:] = math.nan
    packed_check(q, k, v, [100, 200], lead=7)
    q[:] = 1
    got = b2.flash_attn_packed(q, k, v, torch.tensor([0], dtype=torch.int32, device="cuda"))
    assert (got == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_packed_masked_values_do_not_reach_a_result(dtype, D, value):
    # tokens after a query, and the neighbouring sequences, hold NaN or infinities
    g = gen(32)
    lens = [70, 200, 61]
    q, k, v = (randn(g, sum(lens), h, D).to(dtype) for h in (4, 2, 2))
    cu = torch.tensor([0, 70, 270, 331], dtype=torch.int32, device="cuda")
    clean = b2.flash_attn_packed(q, k, v, cu)
    k2, v2 = k.clone(), v.clone()
    for t in (0, 3, 69):
        k2[t], v2[t] = value, value
    v2[70 + 150, 1, 5] = value     # queries 150.. of sequence 1, heads 2 and 3, see it
    got = b2.flash_attn_packed(q, k2, v2, cu)
    seen = torch.zeros_like(got, dtype=torch.bool)
    seen[:70] = True
    seen[70 + 150:270, 2:, 5] = True
    # a row beside a poisoned key may be summed in another order than in the clean run
    tol = 1e-4 if dtype == torch.float32 else (U[dtype] + 3e-4) * v.abs().max().double().item()
    check(got[~seen], clean[~seen], 2 * tol, dtype)
    want = torch.full_like(got[70 + 150:270, 2:, 5], value)
    assert torch.equal(torch.isnan(got[220:270, 2:, 5]), torch.isnan(want))
    if not math.isnan(value):
        assert torch.equal(got[220:270, 2:, 5], want)
    assert torch.isnan(got[:70]).all()  # their own first key is not finite


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
def test_packed_non_finite_scores(dtype, D):
    # one NaN in a key makes every query that sees it NaN, wherever the key stands in its block
    g = gen(33)
    for at in range(0, 128, 9):
        q, k, v = (randn(g, 128, 1, D).to(dtype) for _ in range(3))
        cu = torch.tensor([0, 128], dtype=torch.int32, device="cuda")
        clean = b2.flash_attn_packed(q, k, v, cu)
        k[at, 0, 3] = math.nan
        got = b2.flash_attn_packed(q, k, v, cu)
        assert torch.isnan(got[at:]).all() and torch.equal(got[:at], clean[:at])


def test_packed_scores_of_every_size():
    g = gen(34)
    for mul in (0.0, 1e-3, 8.0, 40.0):
        for dtype in (torch.bfloat16, torch.float16):
            q, k, v = (randn(g, 333, h, 128) for h in (4, 2, 2))
            packed_check((q * mul).to(dtype), k.to(dtype), v.to(dtype), [300, 33])
    packed_check(q.half(), k.half(), v.half(), [300, 33], scale=-0.2)
    packed_check(q.half(), k.half(), v.half(), [300, 33], scale=0.0)
    rising = torch.ones(600, 1, 64, device="cuda") * (torch.arange(600, device="cuda")[:, None, None] / 50)
    packed_check(torch.ones(600, 1, 64, device="cuda").half(), rising.half(), randn(g, 600, 1, 64).half(), [600])


def test_packed_alignment_and_strides():
    g = gen(35)
    lens, T = [150, 60], 210
    flat = randn(g, T * 6 * 64 + 1).half()
    for base in (flat[:-1], flat[1:]):
        qkv = base.view(T, 6, 64)
        packed_check(qkv[:, :4], qkv[:, 4:5], qkv[:, 5:], lens)
    qkv = flat[:-1].view(6, T, 64).transpose(0, 1)  # heads outermost
    packed_check(qkv[:, :4], qkv[:, 4:5], qkv[:, 5:], lens)
    ch = randn(g, T, 64, 6).half().transpose(1, 2)   # channels strided
    packed_check(ch[:, :4], ch[:, 4:5], ch[:, 5:], lens)


def test_packed_bad_offsets():
    g = gen(36)
    q, k, v = (randn(g, 300, h, 64).half() for h in (4, 2, 2))
    for cu in ([0, 100, 400], [0, 200, 100], [-5, 100, 300]):
        got = b2.flash_attn_packed(q, k, v, torch.tensor(cu, dtype=torch.int32, device="cuda"))
        assert b2.device_status(0) == _lib.STATUS_BAD_INDEX
        assert got.shape == q.shape


def test_packed_many_sequences():
    g = gen(37)
    lens = [(i * 13) % 40 for i in range(300)]
    q, k, v = (randn(g, sum(lens), h, 64).bfloat16() for h in (4, 1, 1))
    packed_check(q, k, v, lens)


def test_packed_equals_padded_attention():
    # one sequence per batch entry, equal heads: the framework's padded attention is the same operator
    g = gen(38)
    q, k, v = (randn(g, 4 * 512, 8, 128).half() for _ in range(3))
    a = packed_check(q, k, v, [512] * 4)
    b = b2.flash_attn_fwd(*(x.view(4, 512, 8, 128).transpose(1, 2) for x in (q, k, v)), causal=True)
    check(b.transpose(1, 2).reshape(2048, 8, 128), a.double(), 2 * (U[torch.float16] + 3e-4) * v.abs().max().double(), torch.float16)


@pytest.mark.parametrize("bad", ["shape", "heads", "dtype", "v", "cu", "cudtype", "cuk"])
def test_packed_refusals(bad):
    q, k = torch.zeros(8, 4, 64, device="cuda").half(), torch.zeros(8, 2, 64, device="cuda").half()
    cu = torch.tensor([0, 8], dtype=torch.int32, device="cuda")
    a = dict(q=q, k=k, v=k, cu_q=cu)
    a |= {"shape": dict(q=q[0]), "heads": dict(q=q[:, :3]), "dtype": dict(q=q.double(), k=k.double(), v=k.double()),
          "v": dict(v=k.float()), "cu": dict(cu_q=cu[:0]), "cudtype": dict(cu_q=cu.long()),
          "cuk": dict(cu_k=torch.zeros(3, dtype=torch.int32, device="cuda"))}[bad]
    with pytest.raises((ValueError, TypeError)):
        b2.flash_attn_packed(**a)
    with pytest.raises(NotImplementedError):
        x = torch.zeros(8, 2, 136, device="cuda").half()
        b2.flash_attn_packed(x, x, x, cu)


# ------------------------------------------------------------------ how they are called
def a_step(g):
    """Inputs of one decode step and of one prompt call, and the step as a function."""
    T, Hq, Hk, D = 24, 8, 2, 64
    q, k, v = randn(g, T, Hq, D).bfloat16(), randn(g, T, Hk, D).bfloat16(), randn(g, T, Hk, D).bfloat16()
    table, pos = b2.rope_table(64, D), torch.arange(T, device="cuda", dtype=torch.int32)
    w = (1 + 0.1 * randn(g, D)).bfloat16()
    cu = torch.tensor([0, 9, T], device="cuda", dtype=torch.int32)
    cache = b2.kv_cache_alloc(4, Hk, D, 16)
    slots = torch.arange(T, device="cuda") + 16
    pages, lengths = torch.tensor([[1, 2]], device="cuda", dtype=torch.int32), torch.tensor([T], device="cuda", dtype=torch.int32)

    def run():
        qr, kr = b2.qk_norm_rope(q, k, table, pos, w, w)
        b2.kv_cache_write(cache, kr, v, slots)
        o = b2.flash_attn_packed(qr, kr, v, cu)
        o4 = b2.kv_cache_attn(qr[-1:], cache, pages, lengths)
        return (qr, kr, o, o4, *b2.kv_cache_read(cache, slots, torch.float32))
    return run, (q, k, v)


def test_operators_in_a_cuda_graph():
    run, (q, k, v) = a_step(gen(40))
    run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    g = gen(41)
    for x in (q, k, v):  # new inputs in the same buffers
        x.copy_(randn(g, *x.shape))
    graph.replay()
    got = [o.clone() for o in outs]
    assert all(torch.equal(a, b) for a, b in zip(got, run()))


def test_operators_repeat_bit_for_bit():
    run, _ = a_step(gen(42))
    first = run()
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, run()))
    g = gen(43)  # parts of a sequence are joined in the order of its keys, whichever CTA ends first
    lens = [5000, 3, 1700]
    cache, table = filled(g, lens, 2, 128, 64, 16)
    q, lt = randn(g, 3, 2, 8, 128).half(), torch.tensor(lens, dtype=torch.int32, device="cuda")
    want = b2.kv_cache_attn(q, cache, table, lt)
    assert all(torch.equal(b2.kv_cache_attn(q, cache, table, lt), want) for _ in range(10))


def test_operators_on_their_own_streams_and_threads():
    import threading
    runs = [a_step(gen(50 + i))[0] for i in range(4)]
    want = [r() for r in runs]
    torch.cuda.synchronize()
    failed = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got = runs[i]()
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    failed.append(i)
        except Exception as e:  # noqa: BLE001
            failed.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed


def test_rope_in_place_through_the_c_entry():
    import ctypes
    g = gen(44)
    T, Hq, Hk, D, R = 13, 5, 2, 96, 64
    q, k = randn(g, T, Hq, D).bfloat16(), randn(g, T, Hk, D).bfloat16()
    w = (1 + 0.1 * randn(g, D)).bfloat16()
    table, pos = b2.rope_table(32, R), torch.arange(T, device="cuda", dtype=torch.int64)
    for inter in (0, 1):
        want = b2.qk_norm_rope(q, k, table, pos, w, w, interleaved=bool(inter))
        x, y = q.clone(), k.clone()
        strides = (ctypes.c_int64 * 8)(Hq * D, D, Hk * D, D, Hq * D, D, Hk * D, D)
        st = _lib.lib().b2_qk_norm_rope(x.data_ptr(), y.data_ptr(), x.data_ptr(), y.data_ptr(), w.data_ptr(), w.data_ptr(),
                                        table.data_ptr(), pos.data_ptr(), _lib.B2_I64, T, Hq, Hk, D, R, 32, strides, 1e-6,
                                        inter, _lib.B2_BF16, torch.cuda.current_stream().cuda_stream)
        assert st == _lib.B2_OK
        assert torch.equal(x, want[0]) and torch.equal(y, want[1])


def test_cache_attn_needs_its_workspace():
    import ctypes
    c = b2.kv_cache_alloc(2, 2, 64, 16)
    q = torch.zeros(1, 1, 4, 64, device="cuda").half()
    o, table, lengths = torch.empty_like(q), torch.zeros(1, 2, device="cuda", dtype=torch.int32), torch.ones(1, device="cuda", dtype=torch.int32)
    shape, strides = (ctypes.c_int64 * 5)(2, 2, 16, 64, 64), (ctypes.c_int64 * 6)(256, 256, 64, 256, 256, 64)
    args = [x.data_ptr() for x in (q, o, *c, table, lengths)] + [1, 1, 4, 2, 2, shape, strides, 0.1, _lib.B2_F16]
    stream = torch.cuda.current_stream().cuda_stream
    need = _lib.lib().b2_query_workspace(4, 1, 2, 2, 64)
    assert need > 0
    assert _lib.lib().b2_kv_cache_attn(*args, None, 0, stream) == _lib.B2_EINVAL
    ws = torch.empty(need + 16, dtype=torch.uint8, device="cuda")
    assert _lib.lib().b2_kv_cache_attn(*args, ws.data_ptr(), need - 1, stream) == _lib.B2_EINVAL
    assert _lib.lib().b2_kv_cache_attn(*args, ws.data_ptr() + 8, need, stream) == _lib.B2_EINVAL
    assert _lib.lib().b2_kv_cache_attn(*args, ws.data_ptr(), need, stream) == _lib.B2_OK
    assert (o == 0).all()
