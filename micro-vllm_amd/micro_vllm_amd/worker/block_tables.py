"""Block tables kept on the GPU and changed by lengths that only it knows.

The reference allocates blocks on the host (core/block.py:20-158) and rebuilds
each step's table from Python lists (model_runner.py:833-900); ``DeviceBlockRows``
(packing.py) keeps the rows on the device but still takes their ids from the
host. When a step verifies drafted tokens, how many of them stay is known on
the device first. ``DeviceBlockTables`` holds the free list there too: a step's
blocks, table, slots, positions and tree masks follow from device lengths
without a host read (``mvllm_pack_block_tables``).
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from micro_vllm_amd import _native
from micro_vllm_amd.attention.attention import AttentionMetadata
from micro_vllm_amd.attention.spec import AttentionSpec
from micro_vllm_amd.attention.tree import TreeAttentionMetadata

# What a call did for a request (``status``).
SERVED = 0
NO_BLOCKS = 1
REFUSED = 2


_INT32 = torch.int32
_INT64 = torch.int64


def _int64(t: torch.Tensor, name: str, count: int, device: torch.device) -> torch.Tensor:
    if t.dtype is not _INT64 or t.shape != (count,):
        raise ValueError(f"{name} must be int64 [{count}], got {t.dtype} {tuple(t.shape)}")
    if t.device != device:
        raise RuntimeError(f"{name} is on {t.device}, the block tables on {device}")
    return t if t.is_contiguous() else t.contiguous()


@dataclass(frozen=True, slots=True, eq=False)
class DeviceBlockTables:
    """Rows of block ids, their counts and a free list, all int32 on the GPU.

    ``rows[slot]`` ([slots, width]) holds ``counts[slot]`` ids and -1 behind
    them; ``free_blocks`` holds ``num_free[0]`` free ids, taken from the end,
    and -1 behind them. Which request owns which row is the caller's business.
    Calls change all four in place, in stream order: calls on one object must
    not overlap. Each returns int32 ``status`` per request: ``SERVED`` (also for
    slot -1, which pads a batch), ``NO_BLOCKS`` (the free list is too short; the
    row is as it was) or ``REFUSED`` (a slot out of range or named before in the
    call, a length out of range or below its new tokens; nothing changed).
    """

    rows: torch.Tensor
    counts: torch.Tensor
    free_blocks: torch.Tensor
    num_free: torch.Tensor
    block_size: int
    null_block_id: int

    def __post_init__(self) -> None:
        rows, counts, free, num_free = self.rows, self.counts, self.free_blocks, self.num_free
        device = rows.device
        for t in (rows, counts, free, num_free):
            if t.dtype is not _INT32 or not t.is_contiguous():
                raise ValueError("rows, counts, free_blocks and num_free must be contiguous int32")
            if t.device != device:
                raise RuntimeError(f"block tables lie on {t.device} and {device}")
        if rows.dim() != 2 or rows.shape[0] < 1 or rows.shape[1] < 1 or self.block_size < 1:
            raise ValueError("block tables need rows [slots, width] and a positive block size")
        if counts.shape != rows.shape[:1] or free.dim() != 1 or num_free.shape != (1,):
            raise ValueError("counts needs an entry per row, free_blocks one dimension, num_free one entry")

    @classmethod
    def create(
        cls, num_blocks: int, num_slots: int, width: int, block_size: int, device: torch.device | str
    ) -> "DeviceBlockTables":
        """Empty rows and a full free list over a cache of ``num_blocks``
        blocks, of which the last is the null block; block 0 is taken first."""

        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError("device block tables require a GPU device")
        if num_blocks < 2 or num_slots < 1 or width < 1:
            raise ValueError("block tables need a block besides the null block, rows and a width")
        return cls(
            rows=torch.full((num_slots, width), -1, dtype=torch.int32, device=device),
            counts=torch.zeros(num_slots, dtype=torch.int32, device=device),
            free_blocks=torch.arange(num_blocks - 2, -1, -1, dtype=torch.int32, device=device),
            num_free=torch.tensor([num_blocks - 1], dtype=torch.int32, device=device),
            block_size=block_size,
            null_block_id=num_blocks - 1,
        )

    def _packed(self) -> bytes:
        rows, free = self.rows, self.free_blocks
        return _native.pack_block_tables(
            (rows.data_ptr(), self.counts.data_ptr(), free.data_ptr(), self.num_free.data_ptr()),
            (rows.shape[0], rows.shape[1], free.shape[0], self.block_size),
        )

    def _requests(self, slots: torch.Tensor, lengths: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, int]:
        device = self.rows.device
        if device.type != "cuda":
            raise RuntimeError("device block tables require GPU tensors")
        if slots.dim() != 1:
            raise ValueError(f"slots must be 1-D, got shape {tuple(slots.shape)}")
        count = slots.shape[0]
        if count > _native.MAX_TABLE_REQUESTS:
            raise ValueError(f"{count} requests in one call; at most {_native.MAX_TABLE_REQUESTS}")
        return _int64(slots, "slots", count, device), _int64(lengths, "lengths", count, device), count

    def resize(self, slots: torch.Tensor, lengths: torch.Tensor) -> torch.Tensor:
        """Grow or cut each request's row to the blocks that ``lengths`` need;
        returns the status. Length 0 releases a row, live or not: after a step,
        pass a request that ``pack`` or ``pack_tree`` did not serve the length it
        had before, not the 0 that stands in the step's metadata."""

        slots, lengths, count = self._requests(slots, lengths)
        device = self.rows.device
        status = torch.empty(count, dtype=_INT32, device=device)
        guard = _native.enter_device(device)
        try:
            code = _native.packed("mvllm_resize_block_tables")(
                self._packed(), slots.data_ptr(), lengths.data_ptr(), count, status.data_ptr(),
                _native.stream_handle(device),
            )
        finally:
            if guard is not None:
                guard.__exit__(None, None, None)
        if code:
            _native.check(code, "mvllm_resize_block_tables")
        return status

    def _pack(self, slots, lengths, query_start_locations, parents, num_tokens, spec, words):
        slots, lengths, count = self._requests(slots, lengths)
        device, width = self.rows.device, self.rows.shape[1]
        qsl = _int64(query_start_locations, "query_start_locations", count + 1, device)
        status = torch.empty(count, dtype=_INT32, device=device)
        context_lengths = torch.empty(count, dtype=_INT64, device=device)
        table = torch.empty(count, width, dtype=_INT64, device=device)
        slot_mapping = torch.empty(num_tokens, dtype=_INT64, device=device)
        positions = torch.empty(num_tokens, dtype=_INT64, device=device)
        starts = torch.empty(num_tokens, dtype=_INT64, device=device)
        mask = torch.empty(num_tokens, words, dtype=_INT64, device=device) if words else None
        guard = _native.enter_device(device)
        try:
            code = _native.packed("mvllm_pack_block_tables")(
                self._packed(),
                _native.pack_table_step(
                    (slots.data_ptr(), lengths.data_ptr(), qsl.data_ptr(), parents.data_ptr() if num_tokens and words else 0),
                    (count, num_tokens, self.null_block_id),
                    spec.kernel_code(),
                    (words, width),
                    (
                        context_lengths.data_ptr(), table.data_ptr(), slot_mapping.data_ptr(), positions.data_ptr(),
                        starts.data_ptr(), mask.data_ptr() if words else 0, status.data_ptr(),
                    ),
                ),
                _native.stream_handle(device),
            )
        finally:
            if guard is not None:
                guard.__exit__(None, None, None)
        if code:
            _native.check(code, "mvllm_pack_block_tables")
        return qsl, status, context_lengths, table, slot_mapping, positions, starts, mask

    def pack(
        self,
        slots: torch.Tensor,
        lengths: torch.Tensor,
        query_start_locations: torch.Tensor,
        num_tokens: int,
        spec: AttentionSpec,
        *,
        max_query_len: int | None = None,
    ) -> tuple[AttentionMetadata, torch.Tensor]:
        """``resize``, and the metadata of a step whose new tokens are the last
        ``query_start_locations[r + 1] - query_start_locations[r]`` of each
        request's ``lengths[r]``. A request that is not served gets a null row,
        slots -1 and length 0 in the metadata; its blocks stay its own, and its
        length before the call is the caller's to keep."""

        if num_tokens < 0:
            raise ValueError("num_tokens must not be negative")
        qsl, status, context_lengths, table, slot_mapping, positions, starts, _ = self._pack(
            slots, lengths, query_start_locations, None, num_tokens, spec, 0
        )
        metadata = AttentionMetadata(
            query_positions=positions, query_context_start_positions=starts, query_start_locations=qsl,
            context_lengths=context_lengths, block_table=table, slot_mapping=slot_mapping, block_size=self.block_size,
            max_query_len=max_query_len,
        )
        return metadata, status

    def pack_tree(
        self,
        slots: torch.Tensor,
        lengths: torch.Tensor,
        query_start_locations: torch.Tensor,
        parents: torch.Tensor,
        spec: AttentionSpec,
        *,
        max_nodes: int,
    ) -> tuple[TreeAttentionMetadata, torch.Tensor]:
        """``pack`` for trees: ``parents`` names, for every token, an earlier
        node of its request or -1 (it follows the cached tokens), ``lengths``
        counts the nodes, and ``max_nodes`` (at most 1,024) is the largest tree.
        The mask holds each node and its ancestors, as far back as ``spec``
        reaches."""

        if not 1 <= max_nodes <= _native.MAX_TREE_NODES:
            raise ValueError(f"max_nodes must be 1 to {_native.MAX_TREE_NODES}, got {max_nodes}")
        if parents.dim() != 1:
            raise ValueError(f"parents must be 1-D, got shape {tuple(parents.shape)}")
        num_tokens = parents.shape[0]
        parents = _int64(parents, "parents", num_tokens, self.rows.device)
        qsl, status, context_lengths, table, slot_mapping, positions, starts, mask = self._pack(
            slots, lengths, query_start_locations, parents, num_tokens, spec, -(-max_nodes // 64)
        )
        metadata = TreeAttentionMetadata(
            query_positions=positions, query_context_start_positions=starts, query_start_locations=qsl,
            context_lengths=context_lengths, block_table=table, slot_mapping=slot_mapping, tree_mask=mask,
            block_size=self.block_size, max_query_len=max_nodes,
        )
        return metadata, status
