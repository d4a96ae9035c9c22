"""Drafted decoding over a pool that is too small, and past a request's table:
requests that a step does not serve keep their rows, their cached K/V and their
place, and go on once there is room.

The copy model (``_copy_model``) makes every continuation known, and a row that
was released, overwritten or moved would change a token."""

from __future__ import annotations

import random

import pytest
import torch

from _copy_model import make_copy_model
from micro_vllm_amd import layers
from micro_vllm_amd.attention import FullAttentionSpec
from micro_vllm_amd.attention.operators.registry import get_attention_operator_class
from micro_vllm_amd.harness.model import DecoderConfig, DecoderModel
from micro_vllm_amd.worker.block_tables import NO_BLOCKS, REFUSED, SERVED, DeviceBlockTables
from test_gpu_tree_decoding import BLOCK, OFFSET, VOCAB, drafted

pytestmark = pytest.mark.gpu

PROMPTS = [60, 17, 76, 33]
BLOCKS = 15  # and the null block: the prompts take 4 + 2 + 5 + 3
WIDTH = 6


@pytest.mark.parametrize("fused", [True, False], ids=["fused", "torch"])
def test_requests_that_are_not_served_go_on_later(device, fused):
    rng = random.Random(11)
    config = DecoderConfig.qwen3_0_6b(num_hidden_layers=2, vocab_size=VOCAB, intermediate_size=512)
    paged, tree = (get_attention_operator_class(n)() for n in ("mi355x_paged", "mi355x_tree"))
    model = DecoderModel(config, paged, device=device, fused_layers=fused)
    make_copy_model(model, offset=OFFSET)
    prompts = [[rng.randrange(VOCAB) for _ in range(n)] for n in PROMPTS]
    wanted = []
    for prompt in prompts:
        tokens = list(prompt)
        for _ in range(300):
            tokens.append(tokens[len(tokens) - 1 - OFFSET])
        wanted.append(tokens)
    count = len(prompts)
    tables = DeviceBlockTables.create(BLOCKS + 1, count, WIDTH, BLOCK, device)
    caches = [torch.zeros((2, BLOCKS + 1, BLOCK, 8, 128), dtype=torch.bfloat16, device=device) for _ in range(2)]
    ints = lambda x: torch.tensor(x, dtype=torch.int64, device=device)  # noqa: E731
    starts = lambda sizes: ints([sum(sizes[:i]) for i in range(len(sizes) + 1)])  # noqa: E731
    slots, spec = ints([2, 0, 3, 1]), FullAttentionSpec()
    seen = set()
    waited = [0] * count
    with torch.inference_mode():
        cached = ints(PROMPTS)
        metadata, status = tables.pack(slots, cached, starts(PROMPTS), sum(PROMPTS), spec, max_query_len=max(PROMPTS))
        assert status.tolist() == [SERVED] * count
        hidden = model.forward(ints([t for p in prompts for t in p]), metadata.query_positions, caches, metadata)
        first = layers.argmax_rows(model.logits(hidden[starts(PROMPTS)[1:] - 1]))
        model.operator = tree
        done, live = list(PROMPTS), [True] * count
        for step in range(60):
            assert [t for t, alive in zip(first.tolist(), live) if alive] == [w[d] for w, d, alive in zip(wanted, done, live) if alive]
            # Request 0 once asks for more than its table holds.
            trees = [drafted(w[d:], rng, VOCAB) if alive else ([], []) for w, d, alive in zip(wanted, done, live)]
            if step == 3:
                trees[0] = ([-1] * (WIDTH * BLOCK), [0] * (WIDTH * BLOCK))
            sizes = [len(p) for p, _ in trees]
            parents, tokens = (ints([x for t in trees for x in t[k]]) for k in (0, 1))
            before = [r.clone() for r in tables.rows[slots]], tables.counts[slots].tolist()
            metadata, status = tables.pack_tree(slots, cached + ints(sizes), starts(sizes), parents, spec, max_nodes=max(sizes + [1]))
            hidden = model.forward(tokens, metadata.query_positions, caches, metadata)
            chosen = layers.argmax_rows(model.logits(hidden))
            accepted = layers.accept_tree(tokens, chosen, parents, first, metadata, max_accepted=16, kv_caches=caches)
            first = accepted.next_tokens
            cached = torch.where(status == 0, accepted.context_lengths, cached)
            assert (tables.resize(slots, cached) == SERVED).all()
            for r, got in enumerate(status.tolist()):
                seen.add(got)
                waited[r] += got != SERVED
                if got != SERVED:
                    assert int(cached[r]) == done[r] and int(accepted.counts[r]) == 0
                    assert torch.equal(tables.rows[slots[r]], before[0][r]) and int(tables.counts[slots[r]]) == before[1][r]
                elif live[r]:
                    done[r] += int(accepted.counts[r])
                    assert int(cached[r]) == done[r]
            # A request that is done, or that everyone waits for, leaves; its blocks serve the others.
            starved = all(got != SERVED for got, alive in zip(status.tolist(), live) if alive)
            for r in range(count):
                if live[r] and (done[r] > WIDTH * BLOCK - 12 or starved):
                    live[r], starved = False, False
                    cached[r] = 0
            assert (tables.resize(slots, cached) == SERVED).all()
            if not any(live):
                break
    assert seen == {SERVED, NO_BLOCKS, REFUSED}
    assert sum(d - p for d, p in zip(done, PROMPTS)) > 60 and sum(w > 0 for w in waited) >= 2
    assert sorted(tables.free_blocks.tolist()) == list(range(BLOCKS)) and int(tables.num_free) == BLOCKS
