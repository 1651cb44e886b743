"""PyTorch operators around a decoder layer's attention, for serving.

Operators (namespace ``b2msl``), each one C-ABI call on the tensors' device and
current stream:
  * ``qk_norm_rope``: per-head RMSNorm of queries and keys and their rotary
    positions in one pass; ``rope_table`` makes its table of angles
  * ``kv_cache_write`` / ``kv_cache_read``: a paged key/value cache held in 4 bits
    (``KVCache``, ``kv_cache_alloc``)
  * ``kv_cache_attn``: attention of each sequence's newest tokens over that cache
  * ``flash_attn_packed``: attention over prompts packed without padding, causal,
    with grouped heads

They have no counterparts in the reference. They are forward-only, like the
attention next to them. Index tensors (positions, slots, pages, lengths, offsets)
are read on the device and never copied to the host; one that points outside what
it indexes sets ``STATUS_BAD_INDEX`` in ``device_status()``.

A decode step makes each of these calls once per layer on a few tokens, where the
host's cost is the call's. So the operators are registered with
``torch.library.Library`` (about 3 us per call on the host; ``custom_op`` takes 12),
and the functions below call the implementation directly where nothing traces:
the registered operator serves ``torch.compile`` and other tracers.
"""
from __future__ import annotations

import math
from ctypes import c_int64
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from .ops import _DT, _dtype_code, _require_cuda

_IDX = {torch.int32: _lib.B2_I32, torch.int64: _lib.B2_I64}
_I64x4, _I64x5, _I64x6, _I64x8, _I64x12 = (c_int64 * n for n in (4, 5, 6, 8, 12))

_library = torch.library.Library("b2msl", "FRAGMENT")


def _register(schema: str, impl, fake) -> None:
    name = schema.split("(")[0]
    _library.define(schema)
    _library.impl(name, impl, "CUDA")
    # the same checks raise the package's "no CPU path" error on CPU tensors
    _library.impl(name, impl, "CPU")
    torch.library.register_fake(f"b2msl::{name}", fake, lib=_library)


def _traced(x: torch.Tensor) -> bool:
    """Whether a call on x goes through the registered operator."""
    return type(x) is not torch.Tensor or torch.compiler.is_compiling()


def _call(dev: torch.device, fn: str, *args) -> None:
    """One C call with `dev` current and its current stream as the last argument."""
    f = getattr(_lib.lib(), fn)
    index = dev.index
    # the stream's handle without a Stream object around it (0.1 us against 2)
    stream = torch._C._cuda_getCurrentRawStream(index)
    if index == torch.cuda.current_device():
        st = f(*args, stream)
    else:
        with torch.cuda.device(dev):
            st = f(*args, stream)
    if st != _lib.B2_OK:
        _lib.check(fn, st)


def _unit(x: torch.Tensor) -> torch.Tensor:
    """x with unit channel stride (a copy only where it has another)."""
    return x if x.stride(-1) == 1 or x.shape[-1] <= 1 else x.contiguous()


def _index(t: torch.Tensor, what: str, name: str, size: int, dtypes=_IDX) -> int:
    code = dtypes.get(t.dtype)
    if code is None:
        raise TypeError(f"{what}: {name} must be {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")
    if t.dim() != 1 or t.shape[0] != size:
        raise ValueError(f"{what}: {name} must have shape {(size,)}, got {tuple(t.shape)}")
    if size > 1 and t.stride(0) != 1:
        raise ValueError(f"{what}: {name} must be contiguous")
    return code


_I32 = {torch.int32: _lib.B2_I32}


# ------------------------------------------------------- q/k norm and rotation
def rope_table(length: int, rot_dim: int, base: float = 10000.0, scaling: str = "none",
               factor: float = 1.0, original_length: int = 0, slow: float = 1.0, fast: float = 32.0,
               device="cuda") -> torch.Tensor:
    """Angles of rotary positions 0..length-1: fp32 [length, rot_dim], cosines then sines.

    The angle of pair i at position p is p * base**(-2i/rot_dim), computed in 64
    bits (in 32, an angle of 1e5 is off by 4e-3). For contexts longer than a model
    was trained on, ``scaling``:
      * ``"linear"``: positions divided by ``factor``
      * ``"ntk"``: base * factor**(rot_dim/(rot_dim-2)), which stretches the
        slowest pair by ``factor`` and leaves the fastest
      * ``"by_parts"``: a pair that turns fewer than ``slow`` times in
        ``original_length`` positions is divided by ``factor``, one that turns more
        than ``fast`` times is left, those between are blended; the table is
        multiplied by 0.1*ln(factor) + 1 (YaRN, Peng et al. 2023)
    Made once per model and kept; ``qk_norm_rope`` reads the rows of its positions.
    """
    what = "rope_table"
    if length < 0 or rot_dim < 0 or rot_dim % 2:
        raise ValueError(f"{what}: need length >= 0 and an even rot_dim >= 0")
    if scaling not in ("none", "linear", "ntk", "by_parts"):
        raise ValueError(f"{what}: scaling must be none, linear, ntk or by_parts, got {scaling!r}")
    if not (base > 0 and factor > 0):
        raise ValueError(f"{what}: base and factor must be positive")
    gain = 1.0
    if scaling == "ntk":
        if rot_dim < 4:
            raise ValueError(f"{what}: ntk scaling needs rot_dim >= 4")
        base = base * factor ** (rot_dim / (rot_dim - 2))
    pair = torch.arange(rot_dim // 2, dtype=torch.float64, device=device)
    freq = base ** (-2.0 * pair / max(rot_dim, 1))
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "by_parts":
        if original_length <= 0 or not slow < fast:
            raise ValueError(f"{what}: by_parts needs original_length > 0 and slow < fast")
        turns = original_length * freq / (2 * math.pi)
        keep = ((turns - slow) / (fast - slow)).clamp(0, 1)
        freq = freq * keep + freq / factor * (1 - keep)
        gain = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    angle = torch.arange(length, dtype=torch.float64, device=device)[:, None] * freq
    return (torch.cat((angle.cos(), angle.sin()), 1) * gain).float()


def _weight(w: Optional[torch.Tensor], name: str, D: int, dtype: torch.dtype):
    if w is None:
        return None
    if w.dtype != dtype or w.dim() != 1 or w.shape[0] != D or not w.is_contiguous():
        raise ValueError(f"qk_norm_rope: {name} must be contiguous [{D}] of dtype {dtype}")
    return w.data_ptr()


def _rope_impl(q, k, table, positions, q_weight, k_weight, eps, interleaved):
    what = "qk_norm_rope"
    dev = _require_cuda(q, k, table, positions, q_weight, k_weight, what=what)
    dt = _dtype_code(q, what)
    if q.dim() != 3 or k.dim() != 3:
        raise ValueError(f"{what}: need q [T, Hq, D] and k [T, Hk, D]; got {tuple(q.shape)}, {tuple(k.shape)}")
    T, Hq, D = q.shape
    Tk, Hk, Dk = k.shape
    if T != Tk or D != Dk:
        raise ValueError(f"{what}: need q [T, Hq, D] and k [T, Hk, D]; got {tuple(q.shape)}, {tuple(k.shape)}")
    dtype = q.dtype
    if k.dtype != dtype:
        raise TypeError(f"{what}: q and k must share a dtype ({dtype} vs {k.dtype})")
    if table.dim() != 2 or table.dtype != torch.float32 or not table.is_contiguous():
        raise ValueError(f"{what}: table must be contiguous float32 [positions, rot_dim]")
    P, R = table.shape
    if R % 2 or R > D or D % 2:
        raise ValueError(f"{what}: rot_dim {R} must be even and at most head_dim {D} (even)")
    pos = _index(positions, what, "positions", T)
    qw, kw = _weight(q_weight, "q_weight", D, dtype), _weight(k_weight, "k_weight", D, dtype)
    q, k = _unit(q), _unit(k)
    qo, ko = q.new_empty((T, Hq, D)), k.new_empty((T, Hk, D))
    qt, qh, _ = q.stride()
    kt, kh, _ = k.stride()
    _call(dev, "b2_qk_norm_rope", q.data_ptr(), k.data_ptr(), qo.data_ptr(), ko.data_ptr(), qw, kw,
          table.data_ptr(), positions.data_ptr(), pos, T, Hq, Hk, D, R, P,
          _I64x8(qt, qh, kt, kh, Hq * D, D, Hk * D, D), eps, interleaved, dt)
    return qo, ko


_register("qk_norm_rope(Tensor q, Tensor k, Tensor table, Tensor positions, Tensor? q_weight, "
          "Tensor? k_weight, float eps, bool interleaved) -> (Tensor, Tensor)", _rope_impl,
          lambda q, k, table, positions, q_weight, k_weight, eps, interleaved: (
              q.new_empty(q.shape), k.new_empty(k.shape)))


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, table: torch.Tensor, positions: torch.Tensor,
                 q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                 eps: float = 1e-6, interleaved: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """RMSNorm of each head of q [T, Hq, D] and k [T, Hk, D], then their rotation.

    table: fp32 [P, R] from ``rope_table``; positions: int32 or int64 [T]. The
    first R channels are rotated in pairs (i, i + R/2), or (2i, 2i+1) when
    ``interleaved``; the others are only normed. Without a weight that tensor is
    rotated and not normed. q and k may be strided views (parts of one projection);
    the results are contiguous. A position outside the table gives NaN.
    """
    call = torch.ops.b2msl.qk_norm_rope.default if _traced(q) else _rope_impl
    return call(q, k, table, positions, q_weight, k_weight, eps, interleaved)


# ------------------------------------------------------------- the 4-bit cache
class KVCache(NamedTuple):
    """A paged key/value cache in 4 bits (``kv_cache_alloc``); its layout is in include/b2msl.h.

    codes: uint8 [pages, H, page_size, D/2]; scales: bfloat16 [pages, H, page_size,
    D/group, 2], the step and the lowest value of each group of channels. Slot s is
    token s % page_size of page s // page_size.
    """
    k_codes: torch.Tensor
    k_scales: torch.Tensor
    v_codes: torch.Tensor
    v_scales: torch.Tensor

    @property
    def page_size(self) -> int:
        return self.k_codes.shape[2]

    @property
    def head_dim(self) -> int:
        return 2 * self.k_codes.shape[3]


def kv_cache_alloc(pages: int, heads: int, head_dim: int, page_size: int = 64, group: int = 64,
                   device="cuda") -> KVCache:
    """An empty cache of pages * page_size tokens. head_dim 64 or 128, group 64 or head_dim,
    page_size a multiple of 16. A token takes heads * (head_dim + 8 * head_dim/group) bytes."""
    what = "kv_cache_alloc"
    if head_dim not in (64, 128) or group not in (64, head_dim):
        raise ValueError(f"{what}: head_dim must be 64 or 128 and group 64 or head_dim; got {head_dim}, {group}")
    if page_size <= 0 or page_size % 16 or pages < 0 or heads <= 0:
        raise ValueError(f"{what}: need page_size a positive multiple of 16, pages >= 0, heads > 0")

    def half():
        return (torch.zeros((pages, heads, page_size, head_dim // 2), dtype=torch.uint8, device=device),
                torch.zeros((pages, heads, page_size, head_dim // group, 2), dtype=torch.bfloat16, device=device))
    return KVCache(*half(), *half())


def _cache_shape(what, kc, ks, vc, vs):
    """(H, D, the C ABI's shape array) of a cache."""
    shape, scales = kc.shape, ks.shape
    if len(shape) != 4 or len(scales) != 5 or vc.shape != shape or vs.shape != scales:
        raise ValueError(f"{what}: not a KVCache: codes {tuple(kc.shape)}, {tuple(vc.shape)}, "
                         f"scales {tuple(ks.shape)}, {tuple(vs.shape)}")
    pages, H, page, half = shape
    spages, sH, spage, groups, two = scales
    if spages != pages or sH != H or spage != page or two != 2 or groups == 0:
        raise ValueError(f"{what}: not a KVCache: codes {tuple(shape)}, scales {tuple(scales)}")
    if kc.dtype != torch.uint8 or vc.dtype != torch.uint8 or ks.dtype != torch.bfloat16 \
            or vs.dtype != torch.bfloat16:
        raise TypeError(f"{what}: the cache holds uint8 codes and bfloat16 scales")
    if not (kc.is_contiguous() and ks.is_contiguous() and vc.is_contiguous() and vs.is_contiguous()):
        raise ValueError(f"{what}: the cache's tensors must be contiguous")
    return H, 2 * half, _I64x5(pages, H, page, 2 * half, 2 * half // groups)


def _write_impl(kc, ks, vc, vs, k, v, slots):
    what = "kv_cache_write"
    dev = _require_cuda(kc, ks, vc, vs, k, v, slots, what=what)
    H, D, shape = _cache_shape(what, kc, ks, vc, vs)
    size = k.shape
    if len(size) != 3 or v.shape != size or size[1] != H or size[2] != D:
        raise ValueError(f"{what}: k and v must be [T, {H}, {D}]; got {tuple(k.shape)}, {tuple(v.shape)}")
    if v.dtype != k.dtype:
        raise TypeError(f"{what}: k and v must share a dtype ({k.dtype} vs {v.dtype})")
    dt = _dtype_code(k, what)
    T = size[0]
    sdt = _index(slots, what, "slots", T)
    k, v = _unit(k), _unit(v)
    kt, kh, _ = k.stride()
    vt, vh, _ = v.stride()
    _call(dev, "b2_kv_cache_write", k.data_ptr(), v.data_ptr(), kc.data_ptr(), ks.data_ptr(), vc.data_ptr(),
          vs.data_ptr(), slots.data_ptr(), sdt, T, shape, _I64x4(kt, kh, vt, vh), dt)


_register("kv_cache_write(Tensor(a!) k_codes, Tensor(b!) k_scales, Tensor(c!) v_codes, Tensor(d!) v_scales, "
          "Tensor k, Tensor v, Tensor slots) -> ()", _write_impl,
          lambda kc, ks, vc, vs, k, v, slots: None)


def kv_cache_write(cache: KVCache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Quantises k, v [T, H, D] (any float type, strided) into the cache's slots [T], in place.

    slots: int32 or int64, all different; a negative one marks padding and is skipped.
    """
    (torch.ops.b2msl.kv_cache_write.default if _traced(k) else _write_impl)(*cache, k, v, slots)


def _read_impl(kc, ks, vc, vs, slots, dtype):
    what = "kv_cache_read"
    dev = _require_cuda(kc, ks, vc, vs, slots, what=what)
    H, D, shape = _cache_shape(what, kc, ks, vc, vs)
    if slots.dim() != 1:
        raise ValueError(f"{what}: slots must be [T], got {tuple(slots.shape)}")
    dt = _DT.get(dtype)
    if dt is None:
        raise TypeError(f"{what}: unsupported dtype {dtype} (float32/float16/bfloat16)")
    T = slots.shape[0]
    sdt = _index(slots, what, "slots", T)
    k = slots.new_empty((T, H, D), dtype=dtype)
    v = slots.new_empty((T, H, D), dtype=dtype)
    _call(dev, "b2_kv_cache_read", k.data_ptr(), v.data_ptr(), kc.data_ptr(), ks.data_ptr(), vc.data_ptr(),
          vs.data_ptr(), slots.data_ptr(), sdt, T, shape, _I64x4(H * D, D, H * D, D), dt)
    return k, v


def _read_fake(kc, ks, vc, vs, slots, dtype):
    shape = (slots.shape[0], kc.shape[1], 2 * kc.shape[3])
    return kc.new_empty(shape, dtype=dtype), kc.new_empty(shape, dtype=dtype)


_register("kv_cache_read(Tensor k_codes, Tensor k_scales, Tensor v_codes, Tensor v_scales, Tensor slots, "
          "ScalarType dtype) -> (Tensor, Tensor)", _read_impl, _read_fake)


def kv_cache_read(cache: KVCache, slots: torch.Tensor,
                  dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
    """k, v [T, H, D] of the cache's slots [T]: zeros where a slot is negative.

    For the part of a prompt that is already cached: its keys and values, packed
    before the new ones, go to ``flash_attn_packed``.
    """
    return (torch.ops.b2msl.kv_cache_read.default if _traced(slots) else _read_impl)(*cache, slots, dtype)


# ------------------------------------------------------ attention over the cache
def _attn_impl(q, kc, ks, vc, vs, page_table, lengths, sm_scale):
    what = "kv_cache_attn"
    dev = _require_cuda(q, kc, ks, vc, vs, page_table, lengths, what=what)
    dt = _dtype_code(q, what)
    H, D, shape = _cache_shape(what, kc, ks, vc, vs)
    if q.dim() != 4 or q.shape[3] != D or q.shape[2] % H:
        raise ValueError(f"{what}: q must be [B, N, Hq, {D}] with Hq a multiple of {H}; got {tuple(q.shape)}")
    B, N, Hq, _ = q.shape
    if page_table.dim() != 2 or page_table.shape[0] != B or page_table.dtype != torch.int32:
        raise ValueError(f"{what}: page_table must be int32 [{B}, max_pages]")
    max_pages = page_table.shape[1]
    row, unit = page_table.stride()
    if max_pages > 1 and unit != 1:
        raise ValueError(f"{what}: page_table must have unit stride along a row")
    _index(lengths, what, "lengths", B, _I32)
    q = _unit(q)
    o = q.new_empty((B, N, Hq, D))
    n_ws = _lib.lib().b2_query_workspace(4, B, N * (Hq // H), H, D)
    ws = q.new_empty((n_ws,), dtype=torch.uint8) if n_ws else None
    qb, qn, qh, _ = q.stride()
    _call(dev, "b2_kv_cache_attn", q.data_ptr(), o.data_ptr(), kc.data_ptr(), ks.data_ptr(), vc.data_ptr(),
          vs.data_ptr(), page_table.data_ptr(), lengths.data_ptr(), B, N, Hq, max_pages, row, shape,
          _I64x6(qb, qn, qh, N * Hq * D, Hq * D, D), sm_scale, dt, None if ws is None else ws.data_ptr(), n_ws)
    return o


_register("kv_cache_attn(Tensor q, Tensor k_codes, Tensor k_scales, Tensor v_codes, Tensor v_scales, "
          "Tensor page_table, Tensor lengths, float sm_scale) -> Tensor", _attn_impl,
          lambda q, kc, ks, vc, vs, page_table, lengths, sm_scale: q.new_empty(q.shape))


def kv_cache_attn(q: torch.Tensor, cache: KVCache, page_table: torch.Tensor, lengths: torch.Tensor,
                  sm_scale: Optional[float] = None) -> torch.Tensor:
    """Attention of the newest N tokens of each sequence, q [B, N, Hq, D] or [B, Hq, D] (N = 1).

    page_table: int32 [B, max_pages], the pages of each sequence in order; lengths:
    int32 [B], the tokens of each sequence in the cache, the N new ones included.
    Token n of the N attends everything up to its own position. A token without a
    key gives zeros. sm_scale defaults to 1/sqrt(D).
    """
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(q.shape[-1])
    call = torch.ops.b2msl.kv_cache_attn.default if _traced(q) else _attn_impl
    if q.dim() == 3:
        return call(q.unsqueeze(1), *cache, page_table, lengths, sm_scale).squeeze(1)
    return call(q, *cache, page_table, lengths, sm_scale)


# ------------------------------------------------------------- packed prompts
def _packed_impl(q, k, v, cu_q, cu_k, causal, sm_scale):
    what = "flash_attn_packed"
    dev = _require_cuda(q, k, v, cu_q, cu_k, what=what)
    dt = _dtype_code(q, what)
    if q.dim() != 3 or k.dim() != 3 or v.shape != k.shape:
        raise ValueError(f"{what}: need q [Tq, Hq, D] and k, v [Tk, Hk, D]; got "
                         f"{tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    Tq, Hq, D = q.shape
    Tk, Hk, Dk = k.shape
    if D != Dk or Hk == 0 or Hq % Hk:
        raise ValueError(f"{what}: need q [Tq, Hq, D] and k, v [Tk, Hk, D] with Hq a multiple of Hk; got "
                         f"{tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if not (q.dtype == k.dtype == v.dtype):
        raise TypeError(f"{what}: q, k, v must share a dtype")
    if cu_q.dim() != 1 or cu_q.shape[0] < 1:
        raise ValueError(f"{what}: cu_q must hold the B + 1 offsets of B sequences")
    B = cu_q.shape[0] - 1
    _index(cu_q, what, "cu_q", B + 1, _I32)
    if cu_k is not cu_q:
        _index(cu_k, what, "cu_k", B + 1, _I32)
    o = q.new_empty((Tq, Hq, D))
    n_ws = _lib.lib().b2_query_workspace(5, B, Tq, Hq // Hk, 0)
    ws = q.new_empty((n_ws,), dtype=torch.uint8) if n_ws else None
    _call(dev, "b2_fa_packed", q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), cu_q.data_ptr(),
          cu_k.data_ptr(), B, Tq, Tk, Hq, Hk, D, _I64x12(*q.stride(), *k.stride(), *v.stride(), Hq * D, D, 1),
          sm_scale, causal, dt, None if ws is None else ws.data_ptr(), n_ws)
    return o


_register("flash_attn_packed(Tensor q, Tensor k, Tensor v, Tensor cu_q, Tensor cu_k, bool causal, "
          "float sm_scale) -> Tensor", _packed_impl,
          lambda q, k, v, cu_q, cu_k, causal, sm_scale: q.new_empty(q.shape))


def flash_attn_packed(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor,
                      cu_k: Optional[torch.Tensor] = None, causal: bool = True,
                      sm_scale: Optional[float] = None) -> torch.Tensor:
    """Attention within each of B sequences packed along the token axis.

    q [Tq, Hq, D], k and v [Tk, Hk, D], Hq a multiple of Hk (query head h reads key
    head h // (Hq // Hk)); cu_q, cu_k: int32 [B+1], the offset at which each sequence
    starts and the end of the last (cu_k defaults to cu_q). Causal: with Lq queries
    and Lk keys, query i keeps keys j <= i + Lk - Lq. Queries without a key, and
    tokens outside every sequence, give zeros. sm_scale defaults to 1/sqrt(D).
    """
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(q.shape[-1])
    call = torch.ops.b2msl.flash_attn_packed.default if _traced(q) else _packed_impl
    return call(q, k, v, cu_q, cu_q if cu_k is None else cu_k, causal, sm_scale)
