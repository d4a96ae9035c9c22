"""The step over drafted trees that the integration guide shows, run as written
(CPU only): the block tables are their Python model, the other calls check
their arguments against the package's own signatures."""

from __future__ import annotations

import inspect
import re
from pathlib import Path
from types import SimpleNamespace

import pytest
import torch

from _table_model import Tables
from micro_vllm_amd import layers
from micro_vllm_amd.attention import FullAttentionSpec
from micro_vllm_amd.worker.block_tables import NO_BLOCKS, REFUSED, SERVED, DeviceBlockTables

DOC = Path(__file__).resolve().parents[1] / "INTEGRATION.md"
BLOCK, WIDTH = 16, 6


def snippet():
    if not DOC.exists():
        pytest.skip("the integration guide is not in this copy of the tree")
    section = DOC.read_text().split("steps over drafted trees", 1)[1]
    return re.search(r"```python\n(.*?)```", section, flags=re.S).group(1)


def bound(function, *args, **kwargs):
    return inspect.signature(function).bind(None, *args, **kwargs).arguments


class ListTables:
    """``DeviceBlockTables`` over the Python model."""

    def __init__(self, num_blocks, num_slots, width, block_size):
        self.model = Tables(num_blocks, num_slots, width, block_size)

    def pack_tree(self, *args, **kwargs):
        a = bound(DeviceBlockTables.pack_tree, *args, **kwargs)
        starts = a["query_start_locations"].tolist()
        new = [e - s for s, e in zip(starts, starts[1:])]
        status = self.model.resize(a["slots"].tolist(), a["lengths"].tolist(), new)
        lengths = [n if st == SERVED else 0 for n, st in zip(a["lengths"].tolist(), status)]
        metadata = SimpleNamespace(query_positions="positions", context_lengths=torch.tensor(lengths), nodes=new)
        self.packed = status
        return metadata, torch.tensor(status, dtype=torch.int32)

    def resize(self, *args, **kwargs):
        a = bound(DeviceBlockTables.resize, *args, **kwargs)
        return torch.tensor(self.model.resize(a["slots"].tolist(), a["lengths"].tolist()), dtype=torch.int32)


def accept_one(*args, **kwargs):
    """``accept_tree`` where the model confirms node 0 of every served tree."""

    a = inspect.signature(layers.accept_tree).bind(*args, **kwargs).arguments
    lengths, nodes = a["metadata"].context_lengths, torch.tensor(a["metadata"].nodes)
    served = lengths >= nodes
    kept = torch.where(served, lengths - nodes + (nodes > 0).long(), lengths)
    return layers.TreeAcceptance(
        counts=(served & (nodes > 0)).long(), nodes=torch.zeros(len(kept), 1, dtype=torch.int64),
        next_tokens=a["first_tokens"], context_lengths=kept,
    )


def run_step(tables, cached, sizes, forward=lambda *args: None):
    """One pass of the guide's code; returns its namespace."""

    namespace = dict(
        DeviceBlockTables=SimpleNamespace(create=lambda *a: tables), FullAttentionSpec=FullAttentionSpec, torch=torch,
        num_blocks=None, num_slots=None, width=WIDTH, block_size=BLOCK, device=None,
        model=SimpleNamespace(forward=forward, logits=lambda hidden: None), argmax_rows=lambda logits: None, logits=None,
        accept_tree=accept_one, kv_caches=["cache"], drafts=None, first_tokens=torch.zeros(len(sizes), dtype=torch.int64),
        slots=torch.arange(len(sizes)), cached=torch.tensor(cached), sizes=torch.tensor(sizes),
        lengths=torch.tensor(cached) + torch.tensor(sizes), parents=None,
        qsl=torch.tensor([sum(sizes[:i]) for i in range(len(sizes) + 1)]),
    )
    exec(compile(snippet(), str(DOC), "exec"), namespace)
    return namespace


def test_requests_that_are_not_served_keep_their_blocks():
    """A list that runs out, and a length past the table."""

    tables = ListTables(10, 4, WIDTH, BLOCK)
    cached = [40, 90, 30, 14]
    assert tables.model.resize([0, 1, 2, 3], [32, 90, 0, 0]) == [SERVED] * 4  # 2 + 6 of 9 blocks
    tables.model.resize([0], [40])
    tables.model.rows[2], tables.model.rows[3] = [100, 101], [102]  # (blocks from elsewhere, so that the list is empty)
    before = [list(r) for r in tables.model.rows]
    after = run_step(tables, cached, [4, 8, 5, 3])
    assert tables.packed == [SERVED, REFUSED, NO_BLOCKS, NO_BLOCKS]
    assert tables.model.rows == before
    assert after["status"].tolist() == [SERVED] * 4
    assert after["cached"].tolist() == [41, 90, 30, 14]


def test_the_blocks_of_refused_nodes_go_back():
    tables = ListTables(20, 2, WIDTH, BLOCK)
    tables.model.resize([0, 1], [30, 33])
    free = list(tables.model.free)
    after = run_step(tables, [30, 33], [40, 1])
    assert tables.packed == [SERVED, SERVED]
    assert after["cached"].tolist() == [31, 34] and tables.model.free == free


def test_the_model_is_called_as_it_is_declared():
    from micro_vllm_amd.harness.model import DecoderModel

    calls = []
    tables = ListTables(20, 1, WIDTH, BLOCK)
    tables.model.resize([0], [30])
    run_step(tables, [30], [4], forward=lambda *args: calls.append(bound(DecoderModel.forward, *args)))
    (called,) = calls
    assert called["positions"] == "positions" and called["kv_caches"] == ["cache"]
    assert hasattr(called["metadata"], "context_lengths")
