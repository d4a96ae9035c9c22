"""Fused decoder-layer steps around the attention call, on the HIP library.

torch-facing wrappers of `mvllm_add_rms_norm`, `mvllm_qk_norm_rope_kv_write`,
`mvllm_silu_mul`, `mvllm_embed_rms_norm` and `mvllm_argmax_rows`
(include/mvllm_amd.h). They replace, for bf16/fp16 activations on the GPU:
* RMSNorm (src/micro_vllm/layers/normalization.py:7-22) and the residual
  adds of the decoder layer (models/qwen.py:136-156, llama.py:120-140);
* Qwen3's per-head q/k RMSNorm and the rotary embedding (models/qwen.py:
  89-91, layers/rotary_embedding.py:14-52) together with the paged-cache
  write (attention/operators/reference.py:84-98);
* the SwiGLU activation (layers/mlp.py:10-21);
* the token embedding with the first layer's input RMSNorm (models/qwen.py:
  227, :144);
* greedy sampling, the per-row argmax (sampling/sampler.py:24-31, 39-46).
`accept_tree` (`mvllm_accept_tree`) follows the argmax where a step verifies
drafted trees, which the reference does not do.
There is no fallback: the HIP library must be present.
"""

from __future__ import annotations

from collections.abc import Sequence
from dataclasses import dataclass

import torch

from micro_vllm_amd import _native
from micro_vllm_amd.attention.tree import TreeAttentionMetadata


def _dtype(t: torch.Tensor) -> int:
    if t.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"fused layer ops support bfloat16 and float16, got {t.dtype}")
    if t.device.type != "cuda":
        raise RuntimeError("fused layer ops require GPU tensors")
    return _native.dtype_code(t.dtype)


def add_rms_norm(
    x: torch.Tensor, weight: torch.Tensor, eps: float, residual: torch.Tensor | None = None
) -> torch.Tensor:
    """RMSNorm of ``residual + x`` (``residual`` is updated in place) or of ``x``."""

    code = _dtype(x)
    if x.dim() != 2 or x.stride(1) != 1 or weight.shape != (x.shape[1],) or weight.dtype != x.dtype:
        raise ValueError("add_rms_norm expects x [rows, dim] with unit column stride and weight [dim]")
    if residual is not None and (residual.shape != x.shape or residual.stride(1) != 1 or residual.dtype != x.dtype):
        raise ValueError("residual must match x")
    out = torch.empty_like(x, memory_format=torch.contiguous_format)
    _native.check(
        _native.load().mvllm_add_rms_norm(
            x.data_ptr(),
            x.stride(0),
            residual.data_ptr() if residual is not None else None,
            residual.stride(0) if residual is not None else 0,
            weight.contiguous().data_ptr(),
            out.data_ptr(),
            out.stride(0),
            x.shape[0],
            x.shape[1],
            eps,
            code,
            _native.stream_handle(x.device),
        ),
        "mvllm_add_rms_norm",
    )
    return out


def qk_norm_rope_kv_write(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    q_weight: torch.Tensor | None,
    k_weight: torch.Tensor | None,
    cos: torch.Tensor | None,
    sin: torch.Tensor | None,
    eps: float,
    layer_kv_cache: torch.Tensor,
    slot_mapping: torch.Tensor,
    positions: torch.Tensor | None = None,
) -> torch.Tensor:
    """Normalised, rotated query [tokens, Hq, 128]; key/value go into the cache.

    Without ``positions`` the cos/sin tables hold one row per token; with
    them, one row per position (token t uses row ``positions[t]``; a position
    outside the table rotates to NaN)."""

    _dtype(query)
    rows = query.shape[0] if positions is None else (cos.shape[0] if cos is not None else 0)
    for name, t in (("cos", cos), ("sin", sin)):
        if t is not None and (t.dtype != torch.float32 or not t.is_contiguous() or t.shape != (rows, 128)):
            raise ValueError(f"{name} must be a contiguous float32 [{'tokens' if positions is None else 'positions'}, 128] table")
    if positions is not None:
        if cos is None or positions.dtype != torch.int64 or positions.numel() != query.shape[0]:
            raise ValueError("positions need cos/sin tables and one int64 entry per token")
        positions = positions.contiguous()
    if slot_mapping.dtype != torch.int64 or slot_mapping.numel() != query.shape[0]:
        raise ValueError("slot_mapping must be int64 with one entry per token")
    q_out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
    _native.check(
        _native.packed("mvllm_qk_norm_rope_kv_write")(
            _native.pack_tensor3(query),
            _native.pack_tensor3(key),
            _native.pack_tensor3(value),
            q_weight.contiguous().data_ptr() if q_weight is not None else None,
            k_weight.contiguous().data_ptr() if k_weight is not None else None,
            cos.data_ptr() if cos is not None else None,
            sin.data_ptr() if sin is not None else None,
            positions.data_ptr() if positions is not None else None,
            rows if positions is not None else 0,
            eps,
            q_out.data_ptr(),
            _native.pack_kv_cache(layer_kv_cache),
            slot_mapping.contiguous().data_ptr(),
            _native.stream_handle(query.device),
        ),
        "mvllm_qk_norm_rope_kv_write",
    )
    return q_out


def silu_mul(gate_up: torch.Tensor) -> torch.Tensor:
    """silu(gate) * up for rows [gate | up]."""

    code = _dtype(gate_up)
    if gate_up.dim() != 2 or gate_up.stride(1) != 1 or gate_up.shape[1] % 4:
        raise ValueError("silu_mul expects [rows, 2 * intermediate] with unit column stride")
    inter = gate_up.shape[1] // 2
    out = torch.empty((gate_up.shape[0], inter), dtype=gate_up.dtype, device=gate_up.device)
    _native.check(
        _native.load().mvllm_silu_mul(
            gate_up.data_ptr(),
            gate_up.stride(0),
            out.data_ptr(),
            out.stride(0),
            gate_up.shape[0],
            inter,
            code,
            _native.stream_handle(gate_up.device),
        ),
        "mvllm_silu_mul",
    )
    return out


def embed_rms_norm(
    ids: torch.Tensor,
    embedding: torch.Tensor,
    weight: torch.Tensor,
    eps: float,
    last_tokens: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """(embedding rows of ``ids``, their RMSNorm): the residual stream and the
    first layer's input. An id ``-(1 + r)`` stands for ``last_tokens[r]``;
    ids outside the vocabulary give zero rows."""

    code = _dtype(embedding)
    if ids.dtype != torch.int64 or ids.dim() != 1:
        raise ValueError("ids must be a 1-D int64 tensor")
    if embedding.dim() != 2 or embedding.stride(1) != 1 or weight.shape != (embedding.shape[1],) or weight.dtype != embedding.dtype:
        raise ValueError("embed_rms_norm expects embedding [vocab, dim] with unit column stride and weight [dim]")
    if last_tokens is not None and (last_tokens.dtype != torch.int64 or not last_tokens.is_contiguous()):
        raise ValueError("last_tokens must be a contiguous int64 tensor")
    n, dim = ids.shape[0], embedding.shape[1]
    residual = torch.empty((n, dim), dtype=embedding.dtype, device=embedding.device)
    out = torch.empty_like(residual)
    ids = ids.contiguous()
    _native.check(
        _native.load().mvllm_embed_rms_norm(
            ids.data_ptr(),
            n,
            last_tokens.data_ptr() if last_tokens is not None else None,
            last_tokens.numel() if last_tokens is not None else 0,
            embedding.data_ptr(),
            embedding.shape[0],
            embedding.stride(0),
            weight.contiguous().data_ptr(),
            residual.data_ptr(),
            residual.stride(0),
            out.data_ptr(),
            out.stride(0),
            dim,
            eps,
            code,
            _native.stream_handle(embedding.device),
        ),
        "mvllm_embed_rms_norm",
    )
    return residual, out


def argmax_rows(logits: torch.Tensor, copy_into: torch.Tensor | None = None) -> torch.Tensor:
    """``logits.argmax(dim=-1)`` for [rows, vocab] logits (int64 [rows]);
    ``copy_into[:rows]`` receives the same indices."""

    if logits.device.type != "cuda":
        raise RuntimeError("argmax_rows requires GPU tensors")
    if logits.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise ValueError(f"argmax_rows supports bfloat16, float16 and float32, got {logits.dtype}")
    if logits.dim() != 2 or logits.stride(1) != 1:
        raise ValueError("argmax_rows expects [rows, vocab] logits with unit column stride")
    rows = logits.shape[0]
    if copy_into is not None and (copy_into.dtype != torch.int64 or not copy_into.is_contiguous() or copy_into.numel() < rows):
        raise ValueError("copy_into must be a contiguous int64 tensor with a slot per row")
    out = torch.empty(rows, dtype=torch.int64, device=logits.device)
    _native.check(
        _native.load().mvllm_argmax_rows(
            logits.data_ptr(),
            rows,
            logits.shape[1],
            logits.stride(0),
            _native.dtype_code(logits.dtype),
            out.data_ptr(),
            copy_into.data_ptr() if copy_into is not None else None,
            _native.stream_handle(logits.device),
        ),
        "mvllm_argmax_rows",
    )
    return out


@dataclass(frozen=True, slots=True, eq=False)
class TreeAcceptance:
    """What a verified step keeps of every request's tree (all int64)."""

    counts: torch.Tensor  # [requests] accepted nodes
    nodes: torch.Tensor  # [requests, max_accepted] which, ascending; -1 behind them
    next_tokens: torch.Tensor  # [requests] the token after the last accepted one
    context_lengths: torch.Tensor  # [requests] cached tokens with the accepted ones


def _tokens(t: torch.Tensor, name: str, count: int, device: torch.device) -> torch.Tensor:
    if t.dtype is not torch.int64 or t.shape != (count,):
        raise ValueError(f"{name} must be int64 [{count}], got {t.dtype} {tuple(t.shape)}")
    if t.device != device:
        raise RuntimeError(f"{name} is on {t.device}, expected {device}")
    return t if t.is_contiguous() else t.contiguous()


def accept_tree(
    draft_tokens: torch.Tensor,
    target_tokens: torch.Tensor,
    parents: torch.Tensor,
    first_tokens: torch.Tensor,
    metadata: TreeAttentionMetadata,
    *,
    max_accepted: int,
    kv_caches: Sequence[torch.Tensor] | torch.Tensor = (),
) -> TreeAcceptance:
    """The longest path of every drafted tree that the model's own tokens
    confirm, its K/V rows moved behind the cached tokens.

    ``target_tokens`` [tokens] is the model's choice after each node
    (``argmax_rows`` of its logits), ``first_tokens`` [requests] the token known
    to follow the cached ones; a node is accepted if its drafted token is its
    parent's choice (or, with parent -1, the request's first token) and its
    parent is accepted. The lowest of equal siblings wins; at most
    ``max_accepted`` (up to 1,024) are taken. ``kv_caches`` (every layer's cache,
    or one tensor with a leading layer dimension; all alike) are changed in
    place: accepted node k's rows go to position cached + k. A request whose
    context length is below its nodes accepts nothing and keeps that length.
    ``pack_tree`` gives 0 to one that it did not serve; that request's own
    length is the caller's to keep, ``torch.where(status == 0,
    accepted.context_lengths, cached)`` with the status of ``pack_tree`` and the
    cached tokens before the step, as ``resize`` would release its row for 0."""

    device = draft_tokens.device
    if device.type != "cuda":
        raise RuntimeError("accept_tree requires GPU tensors")
    if draft_tokens.dim() != 1:
        raise ValueError(f"draft_tokens must be 1-D, got shape {tuple(draft_tokens.shape)}")
    if not 1 <= max_accepted <= _native.MAX_TREE_NODES:
        raise ValueError(f"max_accepted must be 1 to {_native.MAX_TREE_NODES}, got {max_accepted}")
    n, requests = draft_tokens.shape[0], metadata.num_requests
    draft_tokens = _tokens(draft_tokens, "draft_tokens", n, device)
    target_tokens = _tokens(target_tokens, "target_tokens", n, device)
    parents = _tokens(parents, "parents", n, device)
    first_tokens = _tokens(first_tokens, "first_tokens", requests, device)
    qsl = _tokens(metadata.query_start_locations, "query_start_locations", requests + 1, device)
    lengths = _tokens(metadata.context_lengths, "context_lengths", requests, device)
    table = metadata.block_table
    if table.dtype is not torch.int64 or table.dim() != 2 or table.shape[0] < requests:
        raise ValueError(f"block_table must be int64 with a row per request, got {table.dtype} {tuple(table.shape)}")
    if table.device != device:
        raise RuntimeError(f"block_table is on {table.device}, expected {device}")
    packed_cache = None
    if isinstance(kv_caches, torch.Tensor):
        shape = kv_caches.shape
        if len(shape) != 6:
            raise ValueError(f"a cache tensor of all layers has 6 dimensions, got shape {tuple(shape)}")
        layers, base, step = shape[0], kv_caches.data_ptr(), kv_caches.stride(0) * kv_caches.element_size()
        pointers = [base + i * step for i in range(layers)]
        like, shape, strides = kv_caches, shape[1:], kv_caches.stride()[1:]
    elif kv_caches:
        layers = len(kv_caches)
        pointers = [c.data_ptr() for c in kv_caches]
        like = kv_caches[0]
        shape, strides = like.shape, like.stride()
        for c in kv_caches:
            if c.shape != shape or c.stride() != strides or c.dtype is not like.dtype or c.device != device:
                raise ValueError("kv_caches must be alike: shape, strides, dtype and device")
    else:
        layers = 0
    if layers:
        if like.device != device:
            raise RuntimeError(f"kv_caches are on {like.device}, expected {device}")
        if len(shape) != 5 or shape[0] != 2 or shape[2] != metadata.block_size:
            raise ValueError(f"kv_caches shape {tuple(shape)} does not match block_size {metadata.block_size}")
        if len(set(pointers)) != layers:
            raise ValueError("kv_caches names a layer's cache twice: its rows would move twice")
        packed_cache = _native.pack_kv_geometry(pointers[0], like.dtype, shape, strides)
    counts = torch.empty(requests, dtype=torch.int64, device=device)
    nodes = torch.empty(requests, max_accepted, dtype=torch.int64, device=device)
    next_tokens = torch.empty(requests, dtype=torch.int64, device=device)
    new_lengths = torch.empty(requests, dtype=torch.int64, device=device)
    guard = _native.enter_device(device)
    try:
        code = _native.packed("mvllm_accept_tree")(
            _native.pack_accept_args(
                (
                    draft_tokens.data_ptr(), target_tokens.data_ptr(), parents.data_ptr(), first_tokens.data_ptr(),
                    qsl.data_ptr(), lengths.data_ptr(), table.data_ptr(),
                ),
                (n, requests, max_accepted),
                (table.shape[1], *table.stride()),
                (counts.data_ptr(), nodes.data_ptr(), next_tokens.data_ptr(), new_lengths.data_ptr()),
            ),
            packed_cache,
            _native.pack_pointers(pointers) if layers else None,
            layers,
            _native.stream_handle(device),
        )
    finally:
        if guard is not None:
            guard.__exit__(None, None, None)
    if code:
        _native.check(code, "mvllm_accept_tree")
    return TreeAcceptance(counts, nodes, next_tokens, new_lengths)
