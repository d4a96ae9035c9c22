"""The gfx950 tree-attention operator (registered as ``"mi355x_tree"``).

Attention of drafted trees over the paged cache, with the call and error
conventions of ``"mi355x_paged"``: the same positional signature, the nodes'
K/V written in place, a new output tensor like ``query``; tensors off the GPU
raise ``RuntimeError``, unsupported types ``ValueError``. It takes a
``TreeAttentionMetadata``. Unlike there, the rows that a call writes may be read
by no other request of the same call: a workgroup writes those that it reads, and
is not ordered with the others. (``DeviceBlockTables`` gives every request blocks
of its own.) All work runs in the HIP library on the current
torch stream without host synchronisation, so a call can be captured in a HIP
graph.
"""

from __future__ import annotations

import math

import torch

from micro_vllm_amd import _native
from micro_vllm_amd.attention.operators.base import AttentionOperator
from micro_vllm_amd.attention.operators.mi355x_paged import SUPPORTED_DTYPES, _batch_fields
from micro_vllm_amd.attention.tree import TreeAttentionMetadata


def _tree_attention(
    query: torch.Tensor,
    key: torch.Tensor | None,
    value: torch.Tensor | None,
    layer_kv_cache: torch.Tensor,
    metadata: TreeAttentionMetadata,
) -> torch.Tensor:
    if (key is None) != (value is None):
        raise ValueError("mi355x_tree attention takes key and value together, or neither")
    device, dtype = query.device, query.dtype
    if device.type != "cuda":
        raise RuntimeError("mi355x_tree attention requires GPU tensors")
    if dtype not in SUPPORTED_DTYPES:
        raise ValueError(
            f"mi355x_tree attention supports torch.bfloat16, torch.float16 and torch.float32, got {dtype}"
        )
    if layer_kv_cache.device != device:
        raise RuntimeError(f"layer_kv_cache is on {layer_kv_cache.device}, query on {device}")
    if layer_kv_cache.dtype is not dtype:
        raise ValueError(f"layer_kv_cache dtype {layer_kv_cache.dtype} differs from query dtype {dtype}")
    packed_key = packed_value = None
    if key is not None:
        if key.dtype is not dtype or value.dtype is not dtype:
            raise ValueError(f"key and value dtypes {key.dtype}, {value.dtype} differ from query dtype {dtype}")
        if key.device != device or value.device != device:
            raise RuntimeError(f"key is on {key.device}, value on {value.device}, query on {device}")
        packed_key, packed_value = _native.pack_tensor3(key), _native.pack_tensor3(value)
    mask = getattr(metadata, "tree_mask", None)
    if mask is None:
        raise ValueError("mi355x_tree attention takes a TreeAttentionMetadata")
    if mask.dtype is not torch.int64 or mask.dim() != 2 or mask.shape[0] != query.shape[0] or mask.shape[1] < 1:
        raise ValueError(
            f"metadata.tree_mask must be int64 [tokens, words], got {mask.dtype} {tuple(mask.shape)}"
        )
    if mask.device != device:
        raise RuntimeError(f"metadata.tree_mask is on {mask.device}, expected {device}")
    words = mask.shape[1]
    row, column = mask.stride()
    if column != 1 or row < words:
        mask = mask.contiguous()
        row = words
    *fields, keep = _batch_fields(metadata, device)
    batch = _native.pack_batch(*fields)
    cache = _native.pack_kv_cache(layer_kv_cache)
    output = torch.empty_like(query, memory_format=torch.contiguous_format)
    guard = _native.enter_device(device)
    try:
        nbytes = _native.packed("mvllm_tree_attention_workspace_bytes")(batch, query.shape[1], cache)
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
        status = _native.packed("mvllm_tree_attention")(
            _native.pack_tensor3(query),
            packed_key,
            packed_value,
            cache,
            batch,
            mask.data_ptr(),
            row,
            words,
            _native.pack_tensor3(output),
            1.0 / math.sqrt(query.shape[-1]),
            workspace.data_ptr() if nbytes else None,
            nbytes,
            _native.stream_handle(device),
        )
    finally:
        if guard is not None:
            guard.__exit__(None, None, None)
    if status:
        _native.check(status, "mvllm_tree_attention")
    del keep
    return output


def hip_tree_attention(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    layer_kv_cache: torch.Tensor,
    metadata: TreeAttentionMetadata,
) -> torch.Tensor:
    """Write the nodes' K/V, then attention over cached tokens and trees.

    A slot that this call writes is read by its own request only; where another
    one's table names it, write the rows first (``hip_write_kv_cache``) and use
    ``hip_tree_attention_over_cache``."""

    return _tree_attention(query, key, value, layer_kv_cache, metadata)


def hip_tree_attention_over_cache(
    query: torch.Tensor,
    layer_kv_cache: torch.Tensor,
    metadata: TreeAttentionMetadata,
) -> torch.Tensor:
    """The attention part of ``hip_tree_attention``, over a cache that already
    holds the nodes' K/V (written by ``layers.qk_norm_rope_kv_write``)."""

    return _tree_attention(query, None, None, layer_kv_cache, metadata)


class MI355XTreeAttentionOperator(AttentionOperator):
    """gfx950 HIP attention of drafted trees over the paged cache."""

    def forward(
        self,
        query: torch.Tensor,
        key: torch.Tensor,
        value: torch.Tensor,
        layer_kv_cache: torch.Tensor,
        metadata: TreeAttentionMetadata,
        /,
    ) -> torch.Tensor:
        return hip_tree_attention(query, key, value, layer_kv_cache, metadata)
