"""Workloads of the decoder-serving operators: q/k norm with rotary positions, the 4-bit paged
key/value cache (write, read back), attention over that cache, and causal attention over packed
prompts.

``listed()`` names the cases, ``prepare`` makes a case's inputs, ``run`` makes one pass: with
``own`` false in elementary torch operations in 32 bits, with ``own`` true through this
repository's operators. ``exact`` gives the same outputs from the definitions in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # a decode step of 16 sequences: the latency of one small launch
        dict(name="rope_decode", op="rope", tokens=16, q_heads=32, kv_heads=8, dim=128, rot=128,
             norm=True, interleaved=False, dtype="bf16", longest=8192),
        # the prompt phase: a long batch of tokens, bound by memory
        dict(name="rope_prompt", op="rope", tokens=16384, q_heads=32, kv_heads=8, dim=128, rot=128,
             norm=True, interleaved=False, dtype="bf16", longest=16384),
        # rotation alone, of half the head, neighbouring pairs, an odd number of tokens
        dict(name="rope_part_odd", op="rope", tokens=5001, q_heads=16, kv_heads=16, dim=64, rot=32,
             norm=False, interleaved=True, dtype="fp16", longest=8192),
        # one new token of each of 32 sequences goes into the cache
        dict(name="cache_decode", op="cache", tokens=32, kv_heads=8, dim=128, group=64, page=16,
             skipped=0, dtype="bf16"),
        # a prompt batch goes into the cache and is read back for the next part of the prompt
        dict(name="cache_prompt", op="cache", tokens=32768, kv_heads=8, dim=128, group=64, page=64,
             skipped=7, dtype="bf16"),
        # a single sequence being answered: latency
        dict(name="attn4_single", op="attn4", batch=1, new=1, q_heads=32, kv_heads=8, dim=128, group=64,
             page=16, longest=2048, dtype="bf16"),
        # an ordinary serving batch of ragged lengths
        dict(name="attn4_batch", op="attn4", batch=32, new=1, q_heads=32, kv_heads=8, dim=128, group=64,
             page=64, longest=8192, dtype="bf16"),
        # four drafted tokens of each sequence are checked at once; small heads, many sharing one
        dict(name="attn4_drafted", op="attn4", batch=16, new=4, q_heads=32, kv_heads=4, dim=64, group=64,
             page=16, longest=4095, dtype="fp16"),
        # few sequences with long contexts
        dict(name="attn4_long", op="attn4", batch=4, new=1, q_heads=32, kv_heads=8, dim=128, group=128,
             page=128, longest=131072, dtype="bf16"),
        # many short prompts, one of a single token
        dict(name="packed_short", op="packed", lengths="1,17,130,64,255,33,97,200,5,128,77,256",
             q_heads=16, kv_heads=16, dim=64, dtype="fp16"),
        # four prompts of 2048 tokens, four query heads to a key head
        dict(name="packed_2048", op="packed", lengths="2048,2048,2048,2048",
             q_heads=32, kv_heads=8, dim=128, dtype="bf16"),
        # a long prompt of odd length beside shorter ones
        dict(name="packed_long", op="packed", lengths="8191,2500,511",
             q_heads=32, kv_heads=8, dim=128, dtype="bf16"),
    ]


def _between(rng, lo, hi):
    """A whole number spread over [lo, hi] evenly in its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "cache", "attn4", "attn4", "packed", "packed"])
    heads, share = rng.choice([1, 2, 4, 5, 8]), rng.choice([1, 2, 3, 4, 6, 7, 8])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "rope":
        dim = rng.choice([64, 80, 96, 128])
        return dict(op=op, tokens=_between(rng, 1, 16384), q_heads=min(32, heads * share), kv_heads=heads,
                    dim=dim, rot=rng.choice([dim, dim // 2]), norm=rng.random() < 0.7,
                    interleaved=rng.random() < 0.4, dtype=rng.choice(["bf16", "fp16", "fp32"]),
                    longest=_between(rng, 1024, 16384))
    if op == "cache":
        dim = rng.choice([64, 128])
        return dict(op=op, tokens=_between(rng, 1, 32768), kv_heads=heads, dim=dim,
                    group=rng.choice([64, dim]), page=rng.choice([16, 32, 64, 128]),
                    skipped=rng.choice([0, 3, 11]), dtype=dtype)
    if op == "attn4":
        dim, batch = rng.choice([64, 128]), _between(rng, 1, 64)
        return dict(op=op, batch=batch, new=rng.choice([1, 1, 1, 2, 3, 4]), q_heads=heads * share,
                    kv_heads=heads, dim=dim, group=rng.choice([64, dim]), page=rng.choice([16, 32, 64, 128]),
                    longest=_between(rng, 1, 262144 // batch), dtype=dtype)
    left, lengths = _between(rng, 1, 8191), []
    while left > 0 and len(lengths) < 24:
        lengths.append(rng.randint(1, left))
        left -= lengths[-1]
    rng.shuffle(lengths)
    heads, share = min(heads, 4), rng.choice([1, 2, 3, 4, 8])
    return dict(op=op, lengths=",".join(map(str, lengths)), q_heads=heads * share, kv_heads=heads,
                dim=rng.choice([64, 96, 128]), dtype=dtype)


def _lengths(case):
    """Lengths of the sequences in the cache: the longest first, the others ragged below it."""
    longest, n = case["longest"], case["batch"]
    return [longest] + [1 + int((longest - 1) * (i * 0.6180339887 % 1.0)) for i in range(1, n)]


def _packed(case):
    return [int(x) for x in case["lengths"].split(",")]


def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    d = case["dim"]
    if case["op"] == "rope":
        rows = case["tokens"] * (case["q_heads"] + case["kv_heads"])
        return dict(bytes=2 * rows * d * e + case["tokens"] * (4 * case["rot"] + 4),
                    flops=rows * (3 * case["rot"] + (4 * d if case["norm"] else 0)))
    if case["op"] == "cache":
        t, h = case["tokens"], case["kv_heads"]
        held = d // 2 + 4 * (d // case["group"])
        return dict(bytes=2 * 2 * t * h * (d * e + held) + 2 * 8 * t, flops=2 * t * h * d * 8)
    if case["op"] == "attn4":
        total = sum(_lengths(case))
        held = d // 2 + 4 * (d // case["group"])
        rows = case["batch"] * case["new"] * case["q_heads"]
        return dict(bytes=2 * total * case["kv_heads"] * held + 2 * rows * d * e,
                    flops=4 * case["new"] * case["q_heads"] * d * total)
    lens = _packed(case)
    pairs = sum(n * (n + 1) // 2 for n in lens)
    return dict(bytes=sum(lens) * d * e * (2 * case["q_heads"] + 2 * case["kv_heads"]),
                flops=4 * case["q_heads"] * d * pairs)


# ------------------------------------------------------------------ the cache's format
# A row of `dim` values of one token and head is held as dim/8 words of 8 values of 4 bits (the
# first value in the lowest bits); word i of the 64-value group g is stored at i*(dim/64) + g.
# Each group of `group` values has a scale and a lowest value in bfloat16: x = code*scale + low.
def _bf16_down(x):
    bits = x.contiguous().view(torch.int32)
    cut = bits & -65536
    return torch.where((bits < 0) & (cut != bits), cut + 65536, cut).view(torch.float32)


def _bf16_up(x):
    return ((x.contiguous().view(torch.int32) + 65535) & -65536).view(torch.float32)


def _quantise(x, group):
    """[..., dim] -> codes uint8 [..., dim/2], scales bf16 [..., dim/group, 2]."""
    dim = x.shape[-1]
    g = x.float().reshape(*x.shape[:-1], dim // group, group)
    low = _bf16_down(g.amin(-1))
    scale = _bf16_up((g.amax(-1) - low) * (1.0 / 15.0))
    fine = torch.isfinite(scale)
    inv = torch.where(scale >= 2.0**-126, 1.0 / scale, torch.zeros_like(scale))
    code = torch.round((g - low[..., None]) * inv[..., None]).clamp(0, 15)
    code = torch.where(fine[..., None], code, torch.zeros_like(code)).to(torch.uint8)
    scale = torch.where(fine, scale, torch.full_like(scale, math.nan))
    pairs = code.reshape(*x.shape[:-1], dim // 64, 8, 4, 2)
    held = (pairs[..., 0] | (pairs[..., 1] << 4)).transpose(-3, -2)
    return held.reshape(*x.shape[:-1], dim // 2), torch.stack((scale, low), -1).to(torch.bfloat16)


def _values(codes, scales, dtype):
    """The values that codes [..., dim/2] and scales [..., dim/group, 2] stand for."""
    half, groups = codes.shape[-1], scales.shape[-2]
    held = codes.reshape(*codes.shape[:-1], 8, half // 32, 4).transpose(-3, -2)
    code = torch.stack((held & 15, held >> 4), -1).reshape(*codes.shape[:-1], groups, 2 * half // groups)
    scales = scales.to(dtype)
    return (code.to(dtype) * scales[..., :1] + scales[..., 1:]).reshape(*codes.shape[:-1], 2 * half)


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, d = DTYPES[case["dtype"]], case["dim"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if case["op"] == "rope":
        t, hq, hk = case["tokens"], case["q_heads"], case["kv_heads"]
        # q and k are parts of the projection's output, which also holds v
        qkv = (normal(t, hq + 2 * hk, d) * 1.5).to(dtype)
        half = case["rot"] // 2
        freq = 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
        angle = torch.arange(case["longest"], device="cuda", dtype=torch.float64)[:, None] * freq
        return dict(case=case, q=qkv[:, :hq], k=qkv[:, hq:hq + hk],
                    table=torch.cat((angle.cos(), angle.sin()), 1).float(),
                    positions=torch.randint(0, case["longest"], (t,), generator=g, device="cuda",
                                            dtype=torch.int32),
                    q_weight=(1 + 0.1 * normal(d)).to(dtype) if case["norm"] else None,
                    k_weight=(1 + 0.1 * normal(d)).to(dtype) if case["norm"] else None)
    if case["op"] == "cache":
        t, h, page = case["tokens"], case["kv_heads"], case["page"]
        pages = (t + page - 1) // page + 3
        slots = torch.randperm(pages * page, generator=g, device="cuda")[:t]
        if case["skipped"]:
            slots[::case["skipped"]] = -1  # padding of the batch: not written
        return dict(case=case, k=(normal(t, h, d) * 2).to(dtype), v=normal(t, h, d).to(dtype), slots=slots,
                    cache=tuple(torch.zeros(pages, h, page, *s, device="cuda", dtype=p) for s, p in (
                        ((d // 2,), torch.uint8), ((d // case["group"], 2), torch.bfloat16)) * 2))
    if case["op"] == "attn4":
        lens, page, h = _lengths(case), case["page"], case["kv_heads"]
        need = [(n + page - 1) // page for n in lens]
        pages = sum(need) + 1
        order = torch.randperm(pages, generator=g, device="cuda", dtype=torch.int32)
        table = torch.zeros(len(lens), max(need), device="cuda", dtype=torch.int32)
        at = 0
        for i, n in enumerate(need):
            table[i, :n] = order[at:at + n]
            at += n
        cache = ()
        for spread in (2.0, 1.0):
            codes = torch.empty(pages, h, page, d // 2, device="cuda", dtype=torch.uint8)
            scales = torch.empty(pages, h, page, d // case["group"], 2, device="cuda", dtype=torch.bfloat16)
            step = max(1, (1 << 27) // (h * page * d))
            for p in range(0, pages, step):
                c, s = _quantise(normal(min(step, pages - p), h, page, d) * spread, case["group"])
                codes[p:p + step], scales[p:p + step] = c, s
            cache += (codes, scales)
        return dict(case=case, q=normal(len(lens), case["new"], case["q_heads"], d).to(dtype), cache=cache,
                    pages=table, lengths=torch.tensor(lens, device="cuda", dtype=torch.int32))
    lens, hq, hk = _packed(case), case["q_heads"], case["kv_heads"]
    qkv = normal(sum(lens), hq + 2 * hk, d).to(dtype)
    starts = [sum(lens[:i]) for i in range(len(lens) + 1)]
    return dict(case=case, q=qkv[:, :hq], k=qkv[:, hq:hq + hk], v=qkv[:, hq + hk:],
                starts=torch.tensor(starts, device="cuda", dtype=torch.int32), longest=max(lens))


# ------------------------------------------------------------------ plain forms
def _turn(x, weight, rows, interleaved, eps, dtype):
    y, rot = x.to(dtype), rows.shape[-1]
    if weight is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps) * weight.to(dtype)
    cos, sin = rows[:, None, :rot // 2], rows[:, None, rot // 2:]
    a, b = (y[..., 0:rot:2], y[..., 1:rot:2]) if interleaved else (y[..., :rot // 2], y[..., rot // 2:rot])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((turned, y[..., rot:]), -1)


def _attend(q, k, v, kept, scale):
    """q [B, H, G, N, D], k and v [B, H, 1, L, D], kept [B, 1, 1, N, L]."""
    s = torch.matmul(q, k.transpose(-1, -2))
    s.mul_(scale).masked_fill_(~kept, -math.inf)
    top = s.amax(-1, keepdim=True)
    s.sub_(torch.where(top > -math.inf, top, torch.zeros_like(top))).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s, v)
    return torch.where(total > 0, o / total, torch.zeros_like(o))


def _cache_attention(s, dtype):
    case, q = s["case"], s["q"]
    b, n, hq, d = q.shape
    h, page = case["kv_heads"], case["page"]
    length = s["pages"].shape[1] * page
    at = s["pages"].long()

    def gathered(codes, scales):
        x = _values(codes[at], scales[at], dtype)  # [B, pages, H, page, D]
        return x.transpose(1, 2).reshape(b, h, 1, length, d)

    limit = s["lengths"].long()[:, None] - n + 1 + torch.arange(n, device=q.device)
    kept = torch.arange(length, device=q.device) < limit[..., None]
    qs = q.to(dtype).reshape(b, n, h, hq // h, d).permute(0, 2, 3, 1, 4)
    o = _attend(qs, gathered(*s["cache"][:2]), gathered(*s["cache"][2:]), kept[:, None, None], d**-0.5)
    return o.permute(0, 3, 1, 2, 4).reshape(b, n, hq, d)


def _packed_attention(s, dtype):
    q, k, v, starts = s["q"], s["k"], s["v"], s["starts"].long()
    t, hq, d = q.shape
    h, longest = k.shape[1], s["longest"]
    place = torch.arange(longest, device=q.device)
    at = (starts[:-1, None] + place).clamp(max=t - 1)  # [B, longest]
    inside = place < (starts[1:] - starts[:-1])[:, None]
    kept = (place[:, None] >= place) & inside[:, None, :]
    qs = q[at].to(dtype).reshape(*at.shape, h, hq // h, d).permute(0, 2, 3, 1, 4)
    ks, vs = (x[at].to(dtype).permute(0, 2, 1, 3)[:, :, None] for x in (k, v))
    o = _attend(qs, ks, vs, kept[:, None, None], d**-0.5)
    return o.permute(0, 3, 1, 2, 4).reshape(*at.shape, hq, d)[inside]


def _through_cache(x, codes, scales, slots, case):
    """Writes x [T, H, D] to its slots of the cache and reads the same slots back."""
    written = slots >= 0
    c, m = _quantise(x, case["group"])
    # padding rows (slot -1) are neither written nor read
    at, c, m = (slots[written], c[written], m[written]) if case["skipped"] else (slots, c, m)
    page, place = at // case["page"], at % case["page"]
    codes[page, :, place], scales[page, :, place] = c, m
    page, place = slots.clamp(min=0) // case["page"], slots.clamp(min=0) % case["page"]
    y = _values(codes[page, :, place], scales[page, :, place], torch.float32)
    return torch.where(written[:, None, None], y, torch.zeros_like(y)).to(x.dtype)


def _plain(s):
    case = s["case"]
    if case["op"] == "rope":
        rows = s["table"][s["positions"].long()]
        return tuple(_turn(x, w, rows, case["interleaved"], 1e-6, torch.float32).to(x.dtype)
                     for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])))
    if case["op"] == "cache":
        return (_through_cache(s["k"], *s["cache"][:2], s["slots"], case),
                _through_cache(s["v"], *s["cache"][2:], s["slots"], case))
    if case["op"] == "attn4":
        return _cache_attention(s, torch.float32).to(s["q"].dtype)
    return _packed_attention(s, torch.float32).to(s["q"].dtype)


# ------------------------------------------------------------------ the repository's operators
def _own(s):
    import triton_msl_b200 as b2

    case = s["case"]
    if case["op"] == "rope":
        return b2.qk_norm_rope(s["q"], s["k"], s["table"], s["positions"], s["q_weight"], s["k_weight"],
                               eps=1e-6, interleaved=case["interleaved"])
    if case["op"] == "cache":
        cache = b2.KVCache(*s["cache"])
        b2.kv_cache_write(cache, s["k"], s["v"], s["slots"])
        return b2.kv_cache_read(cache, s["slots"], dtype=s["k"].dtype)
    if case["op"] == "attn4":
        return b2.kv_cache_attn(s["q"], b2.KVCache(*s["cache"]), s["pages"], s["lengths"])
    return b2.flash_attn_packed(s["q"], s["k"], s["v"], s["starts"], causal=True)


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ 64 bits
def _exact_attention(q, k, v, kept, scale):
    """One head: q [N, D], k and v [L, D], kept [N, L]."""
    s = (q @ k.T * scale).masked_fill(~kept, -math.inf)
    return torch.softmax(s, -1).nan_to_num(0.0) @ v


def exact(case, seed):
    def values(codes, scales):
        """The values of rows of codes [N, dim/2], scales [N, dim/group, 2], value by value from the format."""
        dim, group = 2 * codes.shape[1], 2 * codes.shape[1] // scales.shape[1]
        x = torch.empty(codes.shape[0], dim, device=codes.device, dtype=torch.float64)
        for c in range(dim):
            word = (c % 64 // 8) * (dim // 64) + c // 64
            byte = codes[:, 4 * word + c % 8 // 2].to(torch.float64)
            code = torch.remainder(byte, 16) if c % 2 == 0 else torch.floor(byte / 16)
            x[:, c] = code * scales[:, c // group, 0].double() + scales[:, c // group, 1].double()
        return x

    s = prepare(case, seed)
    d = case["dim"]
    if case["op"] == "rope":
        half, dev = case["rot"] // 2, s["q"].device
        freq = torch.pow(torch.tensor(10000.0, dtype=torch.float64, device=dev),
                         -torch.arange(half, dtype=torch.float64, device=dev) / half)
        turn = torch.polar(torch.ones((), dtype=torch.float64, device=dev), s["positions"].double()[:, None, None] * freq)
        out = ()
        for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])):
            y = x.double()
            if w is not None:
                y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / d + 1e-6) * w.double()
            pairs = y[..., :2 * half].unflatten(-1, (half, 2) if case["interleaved"] else (2, half))
            axis = -1 if case["interleaved"] else -2
            z = torch.complex(pairs.select(axis, 0), pairs.select(axis, 1)) * turn
            out += (torch.cat((torch.stack((z.real, z.imag), axis).flatten(-2), y[..., 2 * half:]), -1),)
        return out
    if case["op"] == "cache":
        out = ()
        for x in (s["k"], s["v"]):
            y = x.double().unflatten(-1, (-1, case["group"]))
            low = _bf16_down(y.amin(-1, keepdim=True).float())
            scale = _bf16_up(((y.amax(-1, keepdim=True) - low.double()) / 15).float()).double()
            # a value half way between two codes may go to either: 32 and 64 bits decide some apart
            code = torch.round((y - low) / scale).clamp(0, 15)
            y = torch.where(scale > 0, code * scale + low, low.double()).flatten(-2)
            out += (torch.where((s["slots"] >= 0)[:, None, None], y, torch.zeros_like(y)),)
        return out
    if case["op"] == "attn4":
        n, share, page = case["new"], case["q_heads"] // case["kv_heads"], case["page"]
        o = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64)
        codes_k, scales_k, codes_v, scales_v = s["cache"]
        for i, length in enumerate(_lengths(case)):
            at = s["pages"][i, :(length + page - 1) // page].long()
            limit = length - n + 1 + torch.arange(n, device="cuda")
            kept = (torch.arange(length, device="cuda") < limit[:, None]).repeat_interleave(share, 0)
            for h in range(case["kv_heads"]):
                k, v = (values(c[at, h].flatten(0, 1)[:length], m[at, h].flatten(0, 1)[:length])
                        for c, m in ((codes_k, scales_k), (codes_v, scales_v)))
                q = s["q"][i, :, h * share:(h + 1) * share].reshape(n * share, d).double()
                o[i, :, h * share:(h + 1) * share] = _exact_attention(q, k, v, kept, d**-0.5).view(n, share, d)
        return o
    share = case["q_heads"] // case["kv_heads"]
    o = torch.empty(s["q"].shape, device="cuda", dtype=torch.float64)
    at = 0
    for n in _packed(case):
        kept = torch.ones(n, n, device="cuda", dtype=torch.bool).tril()
        for h in range(case["q_heads"]):
            q, k, v = (x[at:at + n, i].double() for x, i in ((s["q"], h), (s["k"], h // share), (s["v"], h // share)))
            o[at:at + n, h] = _exact_attention(q, k, v, kept, d**-0.5)
        at += n
    return o
