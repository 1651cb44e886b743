"""One decoder attention layer served with this package's operators.

Prompts of different lengths come in packed, are attended in one call and leave their
keys and values in a paged 4-bit cache; each later step adds one token to every
sequence, or the next part of a prompt to one. Every matrix product, norm, rotation,
cache access and attention is an operator of ``triton_msl_b200``:

    x -> gemm (q, k, v) -> qk_norm_rope -> kv_cache_write -> flash_attn_packed | kv_cache_attn -> gemm

Run ``python examples/decoder_serving.py`` on a B200: it serves three sequences and
prints how far the result is from the same layer in 64 bits without a cache.
"""
from __future__ import annotations

import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
import triton_msl_b200 as b2  # noqa: E402


class Pages:
    """Which pages of the cache each sequence holds."""

    def __init__(self, pages: int, page_size: int, max_sequences: int, max_length: int):
        self.free = list(range(pages))
        self.page_size = page_size
        self.table = torch.zeros(max_sequences, -(-max_length // page_size), dtype=torch.int32)
        self.lengths = [0] * max_sequences

    def extend(self, sequence: int, tokens: int) -> list[int]:
        """Slots for the next `tokens` tokens of a sequence."""
        at, self.lengths[sequence] = self.lengths[sequence], self.lengths[sequence] + tokens
        slots = []
        for t in range(at, at + tokens):
            if t % self.page_size == 0:
                self.table[sequence, t // self.page_size] = self.free.pop()
            slots.append(int(self.table[sequence, t // self.page_size]) * self.page_size + t % self.page_size)
        return slots

    def slots(self, sequence: int, tokens: int) -> list[int]:
        return [int(self.table[sequence, t // self.page_size]) * self.page_size + t % self.page_size
                for t in range(tokens)]


class DecoderAttention:
    """The attention block of a decoder layer: projections, q/k norm, rotation, cache, output."""

    def __init__(self, hidden=256, q_heads=8, kv_heads=2, head_dim=64, max_length=1024, max_sequences=8,
                 page_size=16, seed=0, device="cuda"):
        g = torch.Generator().manual_seed(seed)
        self.q_heads, self.kv_heads, self.head_dim, self.device = q_heads, kv_heads, head_dim, device
        width = (q_heads + 2 * kv_heads) * head_dim

        def weight(*shape):
            return (torch.randn(*shape, generator=g) * shape[0] ** -0.5).to(device, torch.bfloat16)
        self.w_qkv, self.w_out = weight(hidden, width), weight(q_heads * head_dim, hidden)
        self.q_norm, self.k_norm = ((1 + 0.1 * torch.randn(head_dim, generator=g)).to(device, torch.bfloat16)
                                    for _ in range(2))
        self.table = b2.rope_table(max_length, head_dim, device=device)
        self.pages = Pages(max_sequences * max_length // page_size, page_size, max_sequences, max_length)
        self.cache = b2.kv_cache_alloc(len(self.pages.free), kv_heads, head_dim, page_size, device=device)

    def _int(self, values, dtype=torch.int32):
        return torch.tensor(values, dtype=dtype).to(self.device)

    def _qkv(self, x, positions):
        """Queries and keys normed and rotated, values, each [tokens, heads, head_dim]."""
        qkv = b2.gemm(x, self.w_qkv).view(x.shape[0], -1, self.head_dim)
        q, k, v = qkv.split([self.q_heads, self.kv_heads, self.kv_heads], 1)
        q, k = b2.qk_norm_rope(q, k, self.table, positions, self.q_norm, self.k_norm)
        return q, k, v

    def _out(self, o):
        return b2.gemm(o.reshape(-1, self.q_heads * self.head_dim), self.w_out)

    def prompts(self, xs: dict[int, torch.Tensor]) -> torch.Tensor:
        """New prompts {sequence: [tokens, hidden]}, packed; the layer's output for all their tokens."""
        lens = [x.shape[0] for x in xs.values()]
        starts = self._int([sum(lens[:i]) for i in range(len(lens) + 1)])
        q, k, v = self._qkv(torch.cat(list(xs.values())), self._int([t for n in lens for t in range(n)]))
        slots = [s for i, n in zip(xs, lens) for s in self.pages.extend(i, n)]
        b2.kv_cache_write(self.cache, k, v, self._int(slots, torch.int64))
        return self._out(b2.flash_attn_packed(q, k, v, starts))

    def more_of_a_prompt(self, sequence: int, x: torch.Tensor) -> torch.Tensor:
        """The next part of one prompt: its cached tokens are read back before the new ones."""
        held = self.pages.lengths[sequence]
        q, k, v = self._qkv(x, self._int(range(held, held + x.shape[0])))
        old_k, old_v = b2.kv_cache_read(self.cache, self._int(self.pages.slots(sequence, held), torch.int64), k.dtype)
        b2.kv_cache_write(self.cache, k, v, self._int(self.pages.extend(sequence, x.shape[0]), torch.int64))
        return self._out(b2.flash_attn_packed(q, torch.cat((old_k, k)), torch.cat((old_v, v)), self._int([0, x.shape[0]]),
                                              self._int([0, held + x.shape[0]])))

    def step(self, sequences: list[int], x: torch.Tensor) -> torch.Tensor:
        """One new token of each of these sequences, x [sequences, hidden]."""
        q, k, v = self._qkv(x, self._int([self.pages.lengths[i] for i in sequences]))
        slots = [self.pages.extend(i, 1)[0] for i in sequences]
        b2.kv_cache_write(self.cache, k, v, self._int(slots, torch.int64))
        table = self.pages.table[sequences].to(self.device)
        return self._out(b2.kv_cache_attn(q, self.cache, table, self._int([self.pages.lengths[i] for i in sequences])))


def exact(layer: DecoderAttention, x: torch.Tensor) -> torch.Tensor:
    """The layer over one whole sequence x [tokens, hidden] in 64 bits, nothing cached."""
    D, n = layer.head_dim, x.shape[0]
    q, k, v = (x.double() @ layer.w_qkv.double()).view(n, -1, D).split([layer.q_heads, layer.kv_heads, layer.kv_heads], 1)
    angle = torch.arange(n, device=x.device)[:, None] * 10000.0 ** (-torch.arange(D // 2, device=x.device).double() * 2 / D)
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]

    def rotated(y, w):
        y = y * (y.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w.double()
        z = torch.complex(y[..., :D // 2], y[..., D // 2:]) * turn
        return torch.cat((z.real, z.imag), -1)
    q, k = rotated(q, layer.q_norm), rotated(k, layer.k_norm)
    k, v = (y.repeat_interleave(layer.q_heads // layer.kv_heads, 1) for y in (k, v))
    s = torch.einsum("ihd,jhd->hij", q, k) * D ** -0.5
    s = s.masked_fill(torch.ones(n, n, device=x.device, dtype=torch.bool).triu(1), float("-inf"))
    return torch.einsum("hij,jhd->ihd", s.softmax(-1), v).reshape(n, -1) @ layer.w_out.double()


def serve(seed=0, lengths=(37, 130, 5), steps=12) -> dict[str, float]:
    """Serves sequences of these prompt lengths for some steps; the relative error of each phase."""
    layer = DecoderAttention(seed=seed)
    g = torch.Generator().manual_seed(seed + 1)
    total = [n + steps + 9 for n in lengths]
    xs = [torch.randn(n, layer.w_qkv.shape[0], generator=g).to("cuda", torch.bfloat16) for n in total]
    want = [exact(layer, x) for x in xs]

    def error(got, ref):
        return ((got.double() - ref).norm() / ref.norm()).item()
    got = layer.prompts({i: x[:n] for i, (x, n) in enumerate(zip(xs, lengths))})
    errors = {"prompts": error(got, torch.cat([w[:n] for w, n in zip(want, lengths)]))}
    part = layer.more_of_a_prompt(1, xs[1][lengths[1]:lengths[1] + 9])
    errors["more of a prompt"] = error(part, want[1][lengths[1]:lengths[1] + 9])
    at = [n + (9 if i == 1 else 0) for i, n in enumerate(lengths)]
    outs, refs = [], []
    for s in range(steps):
        outs.append(layer.step(list(range(len(xs))), torch.stack([x[a + s] for x, a in zip(xs, at)])))
        refs.append(torch.stack([w[a + s] for w, a in zip(want, at)]))
    errors["steps"] = error(torch.cat(outs), torch.cat(refs))
    return errors


if __name__ == "__main__":
    for phase, e in serve().items():
        print(f"{phase:18s} relative error against 64 bits {e:.4f}")
