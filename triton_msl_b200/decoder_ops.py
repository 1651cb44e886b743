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
attention next to them: a backward pass through one raises. What is written into the
cache is held there without its gradient. Index tensors (positions, slots, pages, lengths, offsets)
are read on the device and never copied to the host; one that points outside what
it indexes sets ``STATUS_BAD_INDEX`` in ``device_status()``.

A decode step makes each of these calls once per layer on a few tokens, where the
host's cost is the call's. So their checks and calls are native
(``csrc/binding.cpp``), and the functions below go there directly where torch's
dispatcher would do nothing else. Under ``torch.compile``, a tracer, a mode or a
transform, for tensors of a subclass and where a gradient is wanted, they call the operators registered with torch.
"""
from __future__ import annotations

import importlib.util
import math
from typing import NamedTuple, Optional, Tuple

import torch
from torch.utils._device import DeviceContext

from . import _build, _lib

_bound = None


def _native():
    """The native binding, with the kernel library's entry points."""
    global _bound
    if _bound is None:
        path = _build.binding_path()
        if not path.exists() and _lib.autobuild():
            _build.build()
        if not path.exists():
            raise RuntimeError(f"{path} is missing: build it with `python -m triton_msl_b200._build`")
        spec = importlib.util.spec_from_file_location(f"{__package__}._decoder", path)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        lib = _lib.lib()
        module.bind(*(_lib.address(getattr(lib, f)) for f in (
            "b2_qk_norm_rope", "b2_kv_cache_write", "b2_kv_cache_read", "b2_kv_cache_attn", "b2_fa_packed",
            "b2_query_workspace")), DeviceContext)
        _bound = module
    return _bound


_library = torch.library.Library("b2msl", "FRAGMENT")


def _register(schema: str, fake) -> None:
    name = schema.split("(")[0]

    def impl(*args):
        return getattr(_native(), name)(*args)
    _library.define(schema)
    _library.impl(name, impl, "CUDA")
    # the same checks raise the package's "no CPU path" error on CPU tensors
    _library.impl(name, impl, "CPU")
    torch.library.register_fake(f"b2msl::{name}", fake, lib=_library)
    if "!" in schema:  # changes its arguments and returns nothing
        return

    def backward(ctx, *grads):
        raise RuntimeError(f"b2msl::{name} is forward-only: nothing can be differentiated through it")
    torch.library.register_autograd(f"b2msl::{name}", backward, lib=_library)


# Each function below asks the binding's direct_... first, which makes the call where nothing
# but the operator's kernel would see it and otherwise returns NotImplemented. The two are
# written out in each: a shared function for it cost 0.15 us of a call.
_compiling = torch.compiler.is_compiling


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
        than ``fast`` times is left, those between are blended linearly in the number
        of turns; the table is multiplied by 0.1*ln(factor) + 1 (YaRN as published,
        Peng et al. 2023). Models that blend by the channel's place instead, or leave
        the table unscaled, bring a table of their own, which ``qk_norm_rope`` takes as well.
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


_register("qk_norm_rope(Tensor q, Tensor k, Tensor table, Tensor positions, Tensor? q_weight, "
          "Tensor? k_weight, float eps, bool interleaved) -> (Tensor, Tensor)",
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
    if type(q) is torch.Tensor and not _compiling():
        out = (_bound or _native()).direct_qk_norm_rope(q, k, table, positions, q_weight, k_weight, eps, interleaved)
        if out is not NotImplemented:
            return out
    return torch.ops.b2msl.qk_norm_rope.default(q, k, table, positions, q_weight, k_weight, eps, interleaved)


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


_register("kv_cache_write(Tensor(a!) k_codes, Tensor(b!) k_scales, Tensor(c!) v_codes, Tensor(d!) v_scales, "
          "Tensor k, Tensor v, Tensor slots) -> ()",
          lambda kc, ks, vc, vs, k, v, slots: None)


def kv_cache_write(cache: KVCache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Quantises k, v [T, H, D] (any float type, strided) into the cache's slots [T], in place.

    slots: int32 or int64, all different; a negative one marks padding and is skipped.
    """
    if type(k) is torch.Tensor and not _compiling():
        out = (_bound or _native()).direct_kv_cache_write(*cache, k, v, slots)
        if out is not NotImplemented:
            return
    torch.ops.b2msl.kv_cache_write.default(*cache, k, v, slots)


def _read_fake(kc, ks, vc, vs, slots, dtype):
    shape = (slots.shape[0], kc.shape[1], 2 * kc.shape[3])
    return kc.new_empty(shape, dtype=dtype), kc.new_empty(shape, dtype=dtype)


_register("kv_cache_read(Tensor k_codes, Tensor k_scales, Tensor v_codes, Tensor v_scales, Tensor slots, "
          "ScalarType dtype) -> (Tensor, Tensor)", _read_fake)


def kv_cache_read(cache: KVCache, slots: torch.Tensor,
                  dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
    """k, v [T, H, D] of the cache's slots [T]: zeros where a slot is negative.

    For the part of a prompt that is already cached: its keys and values, packed
    before the new ones, go to ``flash_attn_packed``.
    """
    if type(slots) is torch.Tensor and not _compiling():
        out = (_bound or _native()).direct_kv_cache_read(*cache, slots, dtype)
        if out is not NotImplemented:
            return out
    return torch.ops.b2msl.kv_cache_read.default(*cache, slots, dtype)


# ------------------------------------------------------ attention over the cache
_register("kv_cache_attn(Tensor q, Tensor k_codes, Tensor k_scales, Tensor v_codes, Tensor v_scales, "
          "Tensor page_table, Tensor lengths, float sm_scale) -> Tensor",
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
    if q.dim() == 3:
        return kv_cache_attn(q.unsqueeze(1), cache, page_table, lengths, sm_scale).squeeze(1)
    if type(q) is torch.Tensor and not _compiling():
        out = (_bound or _native()).direct_kv_cache_attn(q, *cache, page_table, lengths, sm_scale)
        if out is not NotImplemented:
            return out
    return torch.ops.b2msl.kv_cache_attn.default(q, *cache, page_table, lengths, sm_scale)


# ------------------------------------------------------------- packed prompts
_register("flash_attn_packed(Tensor q, Tensor k, Tensor v, Tensor cu_q, Tensor cu_k, bool causal, "
          "float sm_scale) -> Tensor",
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
    if cu_k is None:
        cu_k = cu_q
    if type(q) is torch.Tensor and not _compiling():
        out = (_bound or _native()).direct_flash_attn_packed(q, k, v, cu_q, cu_k, causal, sm_scale)
        if out is not NotImplemented:
            return out
    return torch.ops.b2msl.flash_attn_packed.default(q, k, v, cu_q, cu_k, causal, sm_scale)
