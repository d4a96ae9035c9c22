"""Tree attention in 16 bits against float64, with bounds that a softmax weight
rounded to the inputs' type does not meet.

The weights enter the product with V in two parts. The first is off by at most
half a step (eps / 2 of the type, relative), which the second part holds with
the same relative error: (eps / 2)^2 is left of each weight, 2^-16 in bf16 and
2^-22 in fp16, where parts below the normal numbers add 2^-25 per key for
weights lifted to 2^7 or more: n 2^-32 of the row's sum. The sum of the row is
taken over the fp32 weights. The output's own rounding and the fp32 terms are
those of ``_tree_reference.allowed``. Where values of V cancel, an output is far
smaller than what is added up, and a weight's rounding shows."""

from __future__ import annotations

import pytest
import torch

from _tree_reference import build, random_tree, reference
from micro_vllm_amd.attention.operators.mi355x_tree import hip_tree_attention

pytestmark = pytest.mark.gpu


def bound(dtype, out, size, biggest, most, d):
    u = torch.finfo(dtype).eps / 2
    return u * out.abs() + (u * u + most * 2.0**-32 + 2 * (d + 4) * 2.0**-24 * biggest + most * 2.0**-23 + 2.0**-19) * size + 1e-30


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("nodes", [1, 7, 14, 60])
@pytest.mark.parametrize("contexts", [[150, 40], [2000, 5]], ids=["whole", "split"])
def test_weights_keep_more_bits_than_the_type(device, dtype, d, nodes, contexts):
    gen = torch.Generator().manual_seed(nodes)
    b = build(device, dtype, contexts, [random_tree(nodes, 3, gen) for _ in contexts], 8, 2, d, 16, seed=nodes, scale=0.5)
    out, size, biggest, most = reference(b)
    got = hip_tree_attention(b.query, b.key, b.value, b.cache, b.metadata).cpu().double()
    off, allow = (got - out).abs(), bound(dtype, out, size, biggest, most, d)
    assert not (off > allow).any(), f"worst {float((off / allow).max()):.2f} x the bound"
