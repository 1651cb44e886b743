"""The decoder-serving operators together, as examples/decoder_serving.py uses them."""
import sys
from pathlib import Path

import pytest
import torch

import triton_msl_b200 as b2

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seed,lengths", [(0, (37, 130, 5)), (1, (1, 300, 64, 16))])
def test_serving_a_layer(seed, lengths):
    import decoder_serving
    b2.device_status(0)
    errors = decoder_serving.serve(seed, lengths)
    # bf16 inputs, weights and activations: each of the five roundings on the way (projection, norm and
    # rotation, weights of the softmax, output, projection) is 2^-9 in the mean square, scores of a few
    # units pass theirs on to the weights: under 2 %
    assert errors["prompts"] < 0.02
    # 4-bit keys and values: a group of 64 normal values spans about 5 deviations in 15 steps, so a
    # value is off by 0.33 / sqrt(12) = 0.1 deviations; keys (through scores) and values each add that
    # relative to an average of the values: within 0.25
    assert errors["more of a prompt"] < 0.25
    assert errors["steps"] < 0.25
    assert b2.device_status(0) == 0


def test_operators_under_torch_compile():
    """The registered operators survive tracing and give what the direct calls give."""
    q, k = torch.randn(9, 8, 64, device="cuda").bfloat16(), torch.randn(9, 2, 64, device="cuda").bfloat16()
    table, pos = b2.rope_table(32, 64), torch.arange(9, device="cuda", dtype=torch.int32)
    cu = torch.tensor([0, 4, 9], device="cuda", dtype=torch.int32)
    slots = torch.arange(9, device="cuda")
    pages, lengths = torch.zeros(1, 1, device="cuda", dtype=torch.int32), torch.tensor([9], device="cuda", dtype=torch.int32)

    def layer(cache):
        a, b = b2.qk_norm_rope(q, k, table, pos)
        b2.kv_cache_write(cache, b, k, slots)
        return b2.flash_attn_packed(a, b, k, cu), b2.kv_cache_attn(a[8:].unsqueeze(0), cache, pages, lengths), \
            *b2.kv_cache_read(cache, slots)
    caches = [b2.kv_cache_alloc(1, 2, 64, 16) for _ in range(2)]
    with torch.no_grad():
        want = layer(caches[0])
        got = torch.compile(layer, backend="aot_eager")(caches[1])
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    assert all(torch.equal(x, y) for x, y in zip(*caches))
