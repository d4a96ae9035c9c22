"""Caches with the token dimension outermost: a block's 16-token groups lie
further apart than 32 bits of byte offset reach, while one group's rows do not.
What a batch gives there is, bit for bit, what it gives in a tight cache."""

from __future__ import annotations

import pytest
import torch

from _tree_reference import build, check, random_tree
from micro_vllm_amd.attention.operators.mi355x_tree import hip_tree_attention
from test_gpu_attention import build_case, operator, run_and_check

pytestmark = pytest.mark.gpu

# (tokens of a block, elements between tokens): the last group of a block begins
# 2 (block - 16) stride bytes behind its first one.
WIDE = [(64, 3 * 2**24), (128, 5 * 2**22), (256, 9 * 2**20)]


def spread(cache, token):
    """``cache`` with ``token`` elements between neighbouring tokens."""

    planes, blocks, block, heads, dim = cache.shape
    assert 2 * (block - 16) * token >= 2**32 > 2 * 16 * token
    page = planes * heads * dim
    memory = torch.empty((block - 1) * token + blocks * page, dtype=cache.dtype, device=cache.device)
    wide = memory.as_strided(cache.shape, (heads * dim, page, token, dim, 1))
    wide.copy_(cache)
    return wide


@pytest.mark.parametrize(("block", "token"), WIDE, ids=str)
@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize(("dtype", "nodes"), [(torch.bfloat16, 5), (torch.float16, 13), (torch.bfloat16, 40)], ids=str)
def test_trees_over_groups_far_apart(device, dtype, nodes, d, block, token):
    gen = torch.Generator().manual_seed(nodes)
    trees = [random_tree(n, 3, gen) for n in (nodes, 1, nodes)]
    b = build(device, dtype, [700, 3, 290], trees, 8, 2, d, block, seed=nodes)
    wide = spread(b.cache, token)
    expected = hip_tree_attention(b.query, b.key, b.value, b.cache, b.metadata)
    check(b, expected)
    got = hip_tree_attention(b.query, b.key, b.value, wide, b.metadata)
    assert torch.equal(got, expected)
    assert torch.equal(wide.contiguous().view(torch.int16), b.cache.view(torch.int16))


@pytest.mark.parametrize(("block", "token"), WIDE, ids=str)
@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("qlens", [[200, 33], [70, 1, 2]], ids=["chunks", "mixed"])
def test_chunks_over_groups_far_apart(device, qlens, d, block, token):
    q, k, v, cache, md = build_case(device, torch.bfloat16, [300, 500, 40][: len(qlens)], qlens, 8, 2, d, block, seed=6)
    wide = spread(cache, token)
    got = run_and_check(q, k, v, wide, md, torch.bfloat16)
    assert torch.equal(got, operator()(q, k, v, cache, md))
