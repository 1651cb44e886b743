"""Decoder-serving operators at the edges of what their inputs may hold.

The tolerances are those of test_gpu_decoder_ops.py, for the reasons given there, unless a test
says otherwise.
"""
import math

import pytest
import torch

import triton_msl_b200 as b2
from test_gpu_decoder_ops import U, attn_check, attn_ref, check, filled, gen, packed_check, packed_ref, pick, randn, row_values
from triton_msl_b200 import _lib

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _status():
    b2.device_status(0)
    yield
    assert b2.device_status(0) == 0, "a kernel left a status bit"


def slots_of(table, b, t, page):
    return table[b].long()[t // page] * page + t % page


# ----------------------------------------------------- attention over the cache
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("level", [-100.0, -200.0, -1000.0])
@pytest.mark.parametrize("Hq,D,group", [(1, 64, 64), (4, 128, 64), (4, 128, 128), (8, 64, 64), (8, 128, 64), (16, 128, 128),
                                        (24, 64, 64)])
def test_cache_attn_scores_far_below_zero(dtype, level, Hq, D, group):
    # 2^score is zero for every key; only the scores' differences count. One key, one warp's part of a
    # tile and one more, and a sequence that is cut between CTAs
    g = gen(60 + Hq)
    lens = [1, 33, 5000]
    cache, table = filled(g, lens, 1, D, group, 16)
    for b, n in enumerate(lens):
        k = -level / D**0.5 + 0.3 * randn(g, n, 1, D)
        b2.kv_cache_write(cache, k, randn(g, n, 1, D), slots_of(table, b, torch.arange(n, device="cuda"), 16))
    attn_check(torch.full((3, 1, Hq, D), -1.0, device="cuda").to(dtype), cache, table, lens)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hq,N", [(4, 1), (4, 2), (8, 2)])
@pytest.mark.parametrize("low", [(0, 32), (32, 64), (96, 128), (0, 96), (200, 256)])
def test_cache_attn_some_keys_far_below_the_others(dtype, Hq, N, low):
    g = gen(61)
    D = 128
    cache, table = filled(g, [256], 1, D, 64, 16)
    t = torch.arange(256, device="cuda")
    k = 0.3 * randn(g, 256, 1, D)
    k[low[0]:low[1]] += 300 / D**0.5
    b2.kv_cache_write(cache, k, randn(g, 256, 1, D), slots_of(table, 0, t, 16))
    attn_check(torch.full((1, N, Hq, D), -1.0, device="cuda").to(dtype), cache, table, [256])


@pytest.mark.parametrize("Hq", [4, 8, 16])
def test_cache_attn_tiny_queries_of_huge_keys(Hq):
    # bf16 has fp32's exponents: queries of 2^-118 against keys of 2^118 have scores of about 1
    g = gen(62)
    lens, D = [300], 128
    cache, table = filled(g, lens, 1, D, 64, 16)
    t = torch.arange(300, device="cuda")
    b2.kv_cache_write(cache, randn(g, 300, 1, D) * 2.0**118, randn(g, 300, 1, D), slots_of(table, 0, t, 16))
    attn_check((randn(g, 1, 1, Hq, D) * 2.0**-118).bfloat16(), cache, table, lens)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,group,N", [(64, 64, 1), (128, 64, 1), (128, 128, 1), (128, 64, 2), (128, 128, 4), (64, 64, 4)])
@pytest.mark.parametrize("large", [1e4, 1e6])
def test_cache_attn_large_values_of_small_weight(dtype, D, group, N, large):
    # In heads 0 and 2 a few tokens with values 1e6 times the others' weigh nothing, one key half of the
    # sum and the others, 2^-11.5 of it each, the rest: those products have to keep their bits. Heads 1 and
    # 3 attend the large ones, so no bound that the heads share can serve both.
    g = gen(63 + D)
    B, H, L, page = 24, 8, 4097, 64
    if dtype == torch.float16 and large > 6e4:
        large = 6e4 / 5  # what a result of fp16 can hold
    cache, table = filled(g, [L] * B, H, D, group, page, garbage=False)
    t = torch.arange(L, device="cuda")
    outlier = (t % 1024 < 128) & (t % 32 == 7)
    heavy = torch.zeros(L, dtype=torch.bool, device="cuda")
    heavy[40] = True
    q = torch.zeros(B, N, 4 * H, D, device="cuda")
    q[..., 1] = 8 * D**0.5
    q[:, :, 0::2, 0], q[:, :, 1::2, 0] = -40 * D**0.5, 40 * D**0.5
    plain = []
    for b in range(B):
        k, v = torch.zeros(L, H, D, device="cuda"), randn(g, L, H, D) + 1
        k[outlier, :, 0] = 1.0
        k[heavy, :, 1] = 1.0
        v[outlier] *= large
        plain.append(v[~outlier].abs().max().item())
        b2.kv_cache_write(cache, k, v, slots_of(table, b, t, page))
    q = q.to(dtype)
    got = b2.kv_cache_attn(q, cache, table, torch.full((B,), L, dtype=torch.int32, device="cuda"))
    ref, top = attn_ref(q, cache, table, [L] * B, D**-0.5)
    check(got[:, :, 1::2], ref[:, :, 1::2], 2e-3 * top, dtype)
    # the outliers' own part: weight e^-40
    check(got[:, :, 0::2], ref[:, :, 0::2], 2e-3 * max(plain), dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,group,Hq", [(128, 64, 4), (128, 64, 8), (128, 128, 16), (64, 64, 12)])
def test_cache_attn_scores_of_large_terms(dtype, D, group, Hq):
    # Queries of 30, nearly orthogonal to their sequence's key, beside a key of zeros whose value is 0 where the
    # other's is 1: the result is the logistic function of a score whose terms reach hundreds. In log2 units the
    # score is off by 2^-18 (the tensor core's sums of subnormal codes are low by that) + 2^-20 (its cut sums
    # and the fp32 ones) of its parts; the function's slope is at most 1/4, the weights are rounded by 2^-11 each.
    g = gen(68)
    B = 200
    cache, table = filled(g, [2] * B, 1, D, group, 16, garbage=False)
    slots = table[:, 0].long()[:, None] * 16 + torch.arange(2, device="cuda")
    k, v = torch.zeros(B, 2, 1, D, device="cuda"), torch.zeros(B, 2, 1, D, device="cuda")
    k[:, 1, 0] = 2 * randn(g, B, D)
    v[:, 1] = 1.0
    b2.kv_cache_write(cache, k.view(2 * B, 1, D), v.view(2 * B, 1, D), slots.flatten())
    kc, ks, _, _ = pick(cache, slots[:, 1])
    held = row_values(kc, ks)[:, 0]  # [B, D]
    q = 30 * randn(g, B, 1, Hq, D).double()
    q = q - (q @ held[:, None, :, None]) / held.square().sum(-1)[:, None, None, None] * held[:, None, None]
    q = q.to(dtype)
    low = ks[:, 0, :, 1].double().repeat_interleave(group, -1)
    size = max((q.double() @ part[:, None, :, None]).abs().max().item() for part in (low, held - low)) * D**-0.5 / math.log(2)
    got = b2.kv_cache_attn(q, cache, table, torch.full((B,), 2, dtype=torch.int32, device="cuda"))
    ref, _ = attn_ref(q, cache, table, [2] * B, D**-0.5)
    assert 100 < size and 0.05 < ref.min() and ref.max() < 0.95
    check(got, ref, 0.25 * math.log(2) * (2.0**-18 + 2.0**-20) * size + 2 * 2.0**-11 * 0.25, dtype)


@pytest.mark.parametrize("D,group,Hq", [(64, 64, 16), (128, 64, 16), (128, 128, 96)])
def test_cache_attn_sums_of_bf16_are_hardly_shifted(D, group, Hq):
    # results far smaller than the values they are sums of. bf16's codes are subnormal operands: their sums, of
    # the size of the values, come out low by 2^-18, and by 2^-25 for each 16 keys that a warp adds (some 16
    # times here): together below 2^-17 of the largest value. Independent errors, of the weights (2^-11) and of
    # the result (2^-9), average out over H * D channels, at 6 sigma.
    g = gen(69 + D + Hq)
    L, H = 30000, 16
    cache, table = filled(g, [L], H, D, group, 64, extra=0)
    b2.kv_cache_write(cache, randn(g, L, H, D) * 2, randn(g, L, H, D), slots_of(table, 0, torch.arange(L, device="cuda"), 64))
    q = randn(g, 1, 1, Hq, D).bfloat16()
    ref, top = attn_ref(q, cache, table, [L], D**-0.5)
    got = b2.kv_cache_attn(q, cache, table, torch.tensor([L], dtype=torch.int32, device="cuda"))
    shift = (got.double() - ref).mean().abs().item()
    rms = ref.square().mean().sqrt().item()
    assert shift <= 2.0**-17 * top.item() + 6 * (2.0**-11 + 2.0**-9) * rms / math.sqrt(H * D)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,group,Hq,N", [(64, 64, 4, 1), (128, 64, 4, 1), (128, 128, 8, 1), (128, 64, 4, 4), (64, 64, 24, 1)])
def test_cache_attn_one_key_gives_its_value(dtype, D, group, Hq, N):
    # The largest weight is a power of two, so its product with the value's scale is exact and not rounded by
    # 2^-11. Left are the tensor core's sums of subnormal codes, low by 2^-18 of at most twice max|v|, and the
    # result's one rounding.
    g = gen(71)
    lens = [N] * 40
    cache, table = filled(g, lens, 1, D, group, 16)
    q = randn(g, 40, N, Hq, D).to(dtype)
    got = b2.kv_cache_attn(q, cache, table, torch.tensor(lens, dtype=torch.int32, device="cuda"))
    _, _, vc, vs = pick(cache, table[:, 0].long() * 16)
    want = row_values(vc, vs)  # [40, 1, D], token 0: all that the first new token sees
    check(got[:, 0], want.expand(40, Hq, D), 2.0**-17 * want.abs().max(), dtype)


@pytest.mark.parametrize("D,group,Hq", [(128, 64, 4), (64, 64, 8), (128, 128, 24)])
@pytest.mark.parametrize("size", [1e-25, 1e-12, 1e12, 1e30, 2e37])
def test_cache_attn_values_of_every_size(D, group, Hq, size):
    g = gen(72)
    lens = [1, 300, 2000]
    cache, table = filled(g, lens, 1, D, group, 16)
    for b, n in enumerate(lens):
        v = randn(g, n, 1, D).clamp(-4, 4) * size
        v[n // 3:n // 2] = 0  # a part without any
        b2.kv_cache_write(cache, randn(g, n, 1, D) * 2, v, slots_of(table, b, torch.arange(n, device="cuda"), 16))
    attn_check(randn(g, 3, 1, Hq, D).bfloat16(), cache, table, lens)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("value", [0.0, 1.0, -6e4])
def test_cache_attn_constant_values(dtype, value):
    # every group's scale is 0: the result is the value itself, however the scores are spread
    g = gen(73)
    lens, D = [1, 50, 20000], 128
    cache, table = filled(g, lens, 1, D, 64, 64)
    for b, n in enumerate(lens):
        k = randn(g, n, 1, D) * torch.linspace(0.1, 4, n, device="cuda")[:, None, None]
        b2.kv_cache_write(cache, k, torch.full((n, 1, D), value, device="cuda").bfloat16().float(),
                          slots_of(table, b, torch.arange(n, device="cuda"), 64))
    attn_check(randn(g, 3, 2, 4, D).to(dtype)[:, 1:], cache, table, lens)
    attn_check(3 * randn(g, 3, 2, 8, D).to(dtype)[:, 1:], cache, table, lens)


# -------------------------------------------------------------- packed prompts
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_packed_queries_without_a_key_are_zero(dtype, D, value):
    # causal with more queries than keys: query i keeps the keys j <= i - 171, so queries 0..170 keep none,
    # whatever the values hold that later queries of the same tile attend
    g = gen(64)
    Lq, Lk, none = 300, 129, 171
    q, k, v = randn(g, Lq, 8, D).to(dtype), randn(g, Lk, 2, D).to(dtype), randn(g, Lk, 2, D).to(dtype)
    cu_q, cu_k = (torch.tensor([0, n], dtype=torch.int32, device="cuda") for n in (Lq, Lk))
    clean = packed_check(q, k, v, [Lq], [Lk])
    for at in (0, 5, 128):
        w = v.clone()
        w[at, 1] = value
        got = b2.flash_attn_packed(q, k, w, cu_q, cu_k)
        assert (got[:none] == 0).all()
        seen = torch.zeros_like(got, dtype=torch.bool)
        seen[none + at:, 4:] = True
        tol = 1e-4 if dtype == torch.float32 else (U[dtype] + 3e-4) * v.abs().max().double().item()
        check(got[~seen], clean[~seen], 2 * tol, dtype)
        assert not torch.isfinite(got[seen]).any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
def test_masked_values_of_any_size_do_not_reach_a_result(dtype, D):
    # a masked key's weight is 0 and not the smallest normal number, which a value of 1e38 would bring back
    g = gen(65)
    n = 300
    q, k, v = (randn(g, n, h, D).to(dtype) for h in (4, 2, 2))
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    w = v.clone()
    w[250:] = 1e38
    assert torch.equal(b2.flash_attn_packed(q, k, w, cu)[:250], b2.flash_attn_packed(q, k, v, cu)[:250])
    x = [y.transpose(0, 1)[None].repeat_interleave(4 // y.shape[1], 1) for y in (q, k, v, w)]
    assert torch.equal(b2.flash_attn_fwd(x[0], x[1], x[3], causal=True)[:, :, :250],
                       b2.flash_attn_fwd(x[0], x[1], x[2], causal=True)[:, :, :250])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
def test_packed_scores_that_are_all_minus_infinity_have_no_softmax(dtype, D):
    g = gen(66)
    n = 150
    q, k, v = (randn(g, n, h, D).abs().to(dtype) for h in (4, 2, 2))
    k[:70, :, 3] = -math.inf  # queries 0..69 see no other key
    got = b2.flash_attn_packed(q, k, v, torch.tensor([0, n], dtype=torch.int32, device="cuda"))
    assert torch.isnan(got[:70]).all() and torch.isfinite(got[70:]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cu,clamped", [
    ([0, 200, 100], [0, 200, 200]), ([0, 200, 100, 250], [0, 200, 200, 250]), ([150, 20, 220], [150, 150, 220]),
    ([0, 300] * 40, [0, 300] + [300] * 78), ([-5, 100, 400], [0, 100, 300]), ([0, 120, -7, 290, 5], [0, 120, 120, 290, 290]),
    ([0] * 40 + [300, 10, 20, 300], [0] * 40 + [300] * 4)])
def test_packed_offsets_that_descend(dtype, cu, clamped):
    # a sequence begins no earlier than the ones before it end: every token belongs to one, and the work
    # is bounded by the tokens, whatever the offsets hold
    g = gen(67)
    q, k, v = (randn(g, 300, h, 64).to(dtype) for h in (4, 2, 2))
    keys = [i * 300 // (len(cu) - 1) for i in range(len(cu))]
    got = b2.flash_attn_packed(q, k, v, *(torch.tensor(x, dtype=torch.int32, device="cuda") for x in (cu, keys)))
    assert b2.device_status(0) == _lib.STATUS_BAD_INDEX
    ref, top = packed_ref(q, k, v, clamped, keys, True, 64**-0.5)
    check(got, ref, 1e-4 if dtype == torch.float32 else (U[dtype] + 3e-4) * top, dtype)


def test_packed_prompts_of_millions_of_tokens():
    # seconds of units whose last key block is full, between others where it is not: no wait that spans them
    # may take that for a stalled pipeline
    g = gen(74)
    lens, H, D = [2097152, 1200005], 4, 64
    T = sum(lens)
    q, k, v = (torch.empty(T, H, D, device="cuda", dtype=torch.bfloat16).normal_(generator=g) for _ in range(3))
    cu = [0, lens[0], T]
    got = b2.flash_attn_packed(q, k, v, torch.tensor(cu, dtype=torch.int32, device="cuda"))
    assert b2.last_kernel() == "fa_packed_sm100" and b2.device_status(0) == 0
    for b, i in ((0, 5), (0, lens[0] // 2 + 3), (0, lens[0] - 1), (1, 0), (1, 700001), (1, lens[1] - 1)):
        keys = slice(cu[b], cu[b] + i + 1)
        p = torch.softmax(torch.einsum("hd,jhd->hj", q[cu[b] + i].double(), k[keys].double()) * D**-0.5, 1)
        ref = torch.einsum("hj,jhd->hd", p, v[keys].double())
        check(got[cu[b] + i], ref, (U[torch.bfloat16] + 3e-4) * v[keys].abs().max().double().item(), torch.bfloat16)


# ------------------------------------------------------------------ how they are called
def test_the_binding_refuses_tensors_without_storage():
    # what a transform wraps has no storage: an exception, and not the end of the process
    from triton_msl_b200 import decoder_ops
    native = decoder_ops._native()
    q, k = torch.ones(2, 6, 4, 64, device="cuda").half(), torch.ones(6, 2, 64, device="cuda").half()
    table, at = b2.rope_table(8, 64), torch.arange(6, device="cuda", dtype=torch.int32)
    cache = b2.kv_cache_alloc(1, 2, 64, 16)
    cu, one = torch.tensor([0, 6], device="cuda", dtype=torch.int32), torch.ones(1, 1, device="cuda", dtype=torch.int32)
    calls = [lambda x: native.flash_attn_packed(x, k, k, cu, cu, True, 0.1),
             lambda x: native.qk_norm_rope(x, k, table, at, None, None, 1e-6, False)[0],
             lambda x: native.kv_cache_attn(x[None], *cache, one, one[0], 0.1),
             lambda x: native.kv_cache_write(*cache, x[:, :2], x[:, :2], at),
             lambda x: native.kv_cache_read(*cache, at + x.sum().int() * 0, torch.float16)[0]]
    for call in calls:
        with pytest.raises(RuntimeError, match="storage"):
            torch.vmap(call)(q)
        with pytest.raises(RuntimeError, match="storage"):
            torch.func.grad(lambda x: call(x).float().sum())(q[0].float().half())
    assert torch.equal(b2.flash_attn_packed(q[0], k, k, cu), torch.ones_like(q[0]))
