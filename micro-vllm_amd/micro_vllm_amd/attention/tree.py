"""Metadata of a step whose tokens are trees of drafted nodes.

No counterpart in the reference, whose metadata (attention.py:12-28) describes
one causal sequence per request. The fields that both have carry the same
meaning; ``tree_mask`` takes the place of the causal order among a request's
own tokens.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch


@dataclass(frozen=True, slots=True, eq=False)
class TreeAttentionMetadata:
    """Flattened tree nodes, what they see, and paged-cache inputs.

    The tokens of request r are the nodes of its tree. ``context_lengths[r]``
    counts them: node i lies in the cache at position
    ``context_lengths[r] - nodes + i``, behind the request's cached tokens,
    while ``query_positions`` holds its place in the sequence (cached tokens +
    depth), for the rotary embedding. It sees the cached positions from
    ``query_context_start_positions`` on, and the nodes whose bits are set in
    its row of ``tree_mask`` (int64, 64 nodes per word; its own bit is not
    implied). ``slot_mapping`` names slots that no other request of the call
    reads, where the call writes them.
    """

    query_positions: torch.Tensor
    query_context_start_positions: torch.Tensor
    query_start_locations: torch.Tensor
    context_lengths: torch.Tensor
    block_table: torch.Tensor
    slot_mapping: torch.Tensor
    tree_mask: torch.Tensor
    block_size: int
    # Optional host-side hint: the largest number of nodes of any request. It
    # chooses the kernel's shape, never what is computed.
    max_query_len: int | None = None

    @property
    def num_requests(self) -> int:
        """Number of requests represented by this batch."""

        return self.context_lengths.numel()
