"""Tree attention where a launch of its own lists the items (more row blocks than
the chip takes in two rounds), at every number of rows per item; head_dim 96 in
each of them; lengths that do not fit their trees, by value. Bounds as in
``_tree_reference``."""

from __future__ import annotations

import math

import pytest
import torch

from _tree_reference import build, check, random_tree
from micro_vllm_amd import layers
from micro_vllm_amd.attention.operators.mi355x_paged import hip_write_kv_cache
from micro_vllm_amd.attention.operators.mi355x_tree import hip_tree_attention, hip_tree_attention_over_cache

pytestmark = pytest.mark.gpu

# (requests, nodes at most): 32, 64 and 128 rows per item with four heads per KV
# head; 8 KV heads leave 64 workgroups per head at once, and two rounds are 128.
LISTED = [(150, 8), (100, 16), (60, 40)]


def many(device, dtype, requests, most, d, tail=0):
    gen = torch.Generator().manual_seed(requests)
    contexts = torch.randint(0, 50, (requests,), generator=gen).tolist()
    contexts[1], contexts[requests // 2] = 1500, 700
    sizes = torch.randint(max(1, most - 6), most + 1, (requests,), generator=gen).tolist()
    sizes[3] = 0
    return build(device, dtype, contexts, [random_tree(n, 3, gen) if n else [] for n in sizes], 32, 8, d, 16, seed=most, tail=tail)


def run(b):
    return hip_tree_attention(b.query, b.key, b.value, b.cache, b.metadata)


@pytest.mark.parametrize(("dtype", "d"), [(torch.bfloat16, 128), (torch.float16, 96), (torch.bfloat16, 64)], ids=str)
@pytest.mark.parametrize(("requests", "most"), LISTED, ids=str)
def test_listed_items(device, dtype, d, requests, most):
    b = many(device, dtype, requests, most, d, tail=5)
    written = b.cache.clone()
    got = run(b)
    assert (got[-5:] == 0).all()
    check(b, got)
    hip_write_kv_cache(b.key, b.value, written, b.metadata)
    assert torch.equal(written.view(torch.int16), b.cache.view(torch.int16))
    assert torch.equal(hip_tree_attention_over_cache(b.query, written, b.metadata), got)


@pytest.mark.parametrize(("requests", "most"), LISTED, ids=str)
def test_graphs_of_listed_items(device, requests, most):
    b = many(device, torch.bfloat16, requests, most, 96)
    run(b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(b)
    for _ in range(3):
        b.query.mul_(0.9)
        b.value.add_(0.25)
        expected = run(b)
        out.fill_(7)
        b.cache.view(2, -1, 8, 96)[:, b.metadata.slot_mapping] = math.nan  # the replay writes the rows anew
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, expected)
    del graph


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("nodes", [6, 14, 40])
def test_nonfinite_rows_at_every_item_size(device, dtype, bad, d, nodes):
    """One request split over its keys, one whole: rows that see the bad value get
    it, the others none of it."""

    gen = torch.Generator().manual_seed(nodes)
    b = build(device, dtype, [1700, 60], [random_tree(nodes, 3, gen) for _ in range(2)], 8, 2, d, 16, seed=nodes)
    b.value[2] = bad
    b.key[nodes + 3] = bad
    got = run(b)
    bad_at = [1700 + 2] * nodes + [60 + 3] * nodes
    touched = torch.tensor([at in seen for at, seen in zip(bad_at, b.visible)], device=device)
    assert 0 < int(touched.sum()) < 2 * nodes
    assert torch.isfinite(got[~touched]).all()
    check(b, got)


@pytest.mark.parametrize(("dtype", "d"), [(torch.bfloat16, 64), (torch.float16, 128), (torch.float32, 128), (torch.bfloat16, 80)], ids=str)
@pytest.mark.parametrize("length", [5, 1, 8])
def test_nodes_before_position_zero_are_seen_by_nobody(device, dtype, d, length):
    """A length below the number of nodes: node j lies at position length - 8 + j."""

    gen = torch.Generator().manual_seed(1)
    tree = random_tree(8, 2, gen)
    b = build(device, dtype, [40], [tree], 4, 2, d, 16, seed=2)
    run(b)
    nodes = [[p - 40 for p in seen if p >= 40] for seen in b.visible]
    b.metadata.context_lengths[0] = length
    b.visible = [[length - 8 + j for j in seen if length - 8 + j >= 0] for seen in nodes]
    got = hip_tree_attention_over_cache(b.query, b.cache, b.metadata)
    assert length == 8 or torch.isnan(got).any()
    check(b, got)


@pytest.mark.parametrize(("dtype", "d"), [(torch.bfloat16, 64), (torch.float16, 128), (torch.float32, 128), (torch.bfloat16, 80)], ids=str)
@pytest.mark.parametrize("length", [2**62, 10**6, 2**31 + 8, 50])
def test_lengths_past_the_table_are_cut_there(device, dtype, d, length):
    """Every position of the table that a block holds is a cached one then."""

    gen = torch.Generator().manual_seed(1)
    b = build(device, dtype, [40], [random_tree(8, 2, gen)], 4, 2, d, 16, seed=2, table_extra=0)
    run(b)
    b.metadata.context_lengths[0] = length
    nodes = [[p - 40 for p in seen if p >= 40] for seen in b.visible]
    prefix = length - 8
    b.visible = [[p for p in range(48) if p < prefix or p - prefix in seen] for seen in nodes]
    check(b, hip_tree_attention_over_cache(b.query, b.cache, b.metadata))


def test_replays_of_an_acceptance_over_new_rows(device):
    """Each replay moves rows that the last one did not leave there."""

    n = 20
    tree = [-1, -1, 0, 1] + list(range(3, n - 1))
    b = build(device, torch.bfloat16, [10], [tree], 1, 1, 8, 16)
    ints = lambda x: torch.tensor(x, dtype=torch.int64, device=device)  # noqa: E731
    parents, targets, drafts, first = ints(tree), ints([1] * n), ints([7] + [1] * (n - 1)), ints([1])
    cache = torch.zeros(b.cache.shape, dtype=torch.bfloat16, device=device)
    call = lambda: layers.accept_tree(drafts, targets, parents, first, b.metadata, max_accepted=32, kv_caches=[cache])  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    table = b.metadata.block_table[0].tolist()
    place = lambda p: (table[p // 16], p % 16)  # noqa: E731
    for turn, stop in enumerate((5, 12, 19, 3)):
        targets.fill_(1)
        targets[stop - 1] = 9
        cache.copy_(torch.randn(cache.shape, generator=torch.Generator().manual_seed(turn)).to(torch.bfloat16))
        path = [1] + list(range(3, stop)) if stop > 3 else [1]
        if stop == 3:
            targets.fill_(1)
            targets[1] = 9
        want = cache.clone()
        for k, i in enumerate(path):
            (sb, so), (db, do) = place(10 + i), place(10 + k)
            want[:, db, do] = cache[:, sb, so]
        graph.replay()
        torch.cuda.synchronize()
        assert got.nodes[0, : int(got.counts)].tolist() == path
        assert got.next_tokens.tolist() == [9] and got.context_lengths.tolist() == [10 + len(path)]
        assert torch.equal(cache, want), turn
    del graph
