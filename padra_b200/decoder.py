"""A decoder layer on the library's kernels: norm, attention over the paged 4-bit cache, norm, routed experts.

`DecoderLayer` strings together what the C ABI offers on either side of the expert projections.  The order is the reference's
(src/cuda/inference.cu:2913-2975 for one row, :3358-3392 for several, :3861-3890 for a chunk); the cache and the attention are this
library's own.  The two dense projections and the router's product are plain library GEMMs.  Nothing is read back to the host: a step
whose row counts stay the same can be captured into a CUDA graph and replayed with new rows, page tables and contexts.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from . import binding as B
from .attention import AttentionKernels, KvCache, Rotary, Sequences
from .experts import EXPERTS, ExpertKernels

MAX_CHUNK_ROWS = 2048  # rows of one routing + scheduling launch


@dataclass
class LayerWeights:
    """Device tensors of one layer; matrices are [outputs][inputs] BF16, norm weights BF16 vectors (q_norm, k_norm may be None)."""

    input_norm: torch.Tensor
    qkv: torch.Tensor  # query heads, then key heads, then value heads
    q_norm: torch.Tensor | None
    k_norm: torch.Tensor | None
    output: torch.Tensor
    post_norm: torch.Tensor
    router: torch.Tensor


class DecoderLayer:
    """One layer over its own cache.  `experts` and `attention` may be shared by the layers of a model (one stream at a time)."""

    def __init__(self, index: int, weights: LayerWeights, attention: AttentionKernels, experts: ExpertKernels, cache: KvCache,
                 rotary: Rotary | None = None, scale: float | None = None, window: int = 0, eps: float = 1e-6):
        w, (hidden, _) = weights, experts.dims
        width = w.output.shape[1]
        self.heads, rest = divmod(width, cache.head_dim)
        if rest or self.heads % cache.kv_heads or tuple(w.output.shape) != (hidden, width):
            raise ValueError("output is [hidden][query heads * head_dim], with query heads a multiple of the cache's KV heads")
        if tuple(w.qkv.shape) != (width + 2 * cache.kv_heads * cache.head_dim, hidden) or tuple(w.router.shape) != (EXPERTS, hidden):
            raise ValueError("qkv is [(query + 2 KV heads) * head_dim][hidden], router [64][hidden]")
        for t in (w.input_norm, w.post_norm):
            if t.dtype != torch.bfloat16 or t.numel() != hidden or not t.is_contiguous():
                raise ValueError("the layer's norm weights are BF16 vectors of `hidden` values")
        self.index, self.weights, self.attention, self.experts, self.cache = index, weights, attention, experts, cache
        self.rotary, self.window, self.eps = rotary, window, eps
        self.scale = 1 / math.sqrt(cache.head_dim) if scale is None else scale

    def project(self, x: torch.Tensor):
        """Queries, keys and values of the rows, as strided views of one product; x is not changed."""
        normalized = torch.empty_like(x)
        self.experts.residual_norm(x, None, normalized, self.weights.input_norm)
        qkv = normalized.bfloat16() @ self.weights.qkv.T
        h, kv, d = self.heads, self.cache.kv_heads, self.cache.head_dim
        return [part.unflatten(1, (-1, d)) for part in qkv.split((h * d, kv * d, kv * d), 1)]

    def attend(self, q, k, v, sequences: Sequences) -> torch.Tensor:
        """Appends the rows to the cache and attends over it; returns [rows][hidden], to be added to the residual stream."""
        w = self.weights
        q = self.attention.append(self.cache, sequences, k, v, self.rotary, w.k_norm, self.eps, q, w.q_norm, torch.zeros_like(q, memory_format=torch.contiguous_format))
        mixed = self.attention.attention(self.cache, sequences, q, self.scale, self.window, torch.zeros_like(q))
        return (mixed.flatten(1) @ w.output.T).float()

    def feed_forward(self, x: torch.Tensor, normalized: torch.Tensor) -> None:
        """Adds the routed experts' output to x: the whole-layer decode kernels for few rows, chunks of grouped GEMMs for many."""
        rows = x.shape[0]
        logits = (normalized.bfloat16() @ self.weights.router.T).float()
        if rows <= B.MAX_DECODE_ROWS:
            ids, routing = self.experts.route(logits)
            self.experts.moe_decode_layer(self.index, ids, routing, normalized, x, rows)
            return
        for at in range(0, rows, MAX_CHUNK_ROWS):
            n = min(MAX_CHUNK_ROWS, rows - at)
            if n > 3:
                self.experts.prefill_chunk(self.index, logits[at:at + n], normalized[at:at + n], x[at:at + n], n)
            else:  # a chunk's tail too short for a grouped GEMM
                ids, routing = self.experts.route(logits[at:at + n])
                self.experts.moe_decode_layer(self.index, ids, routing, normalized[at:at + n], x[at:at + n], n)

    def forward(self, x: torch.Tensor, sequences: Sequences) -> torch.Tensor:
        """One step for the rows of x [rows][hidden] (FP32, the residual stream), updated in place and returned.  Rows of no sequence
        and padding attend to nothing; the rest of the layer treats them like any other."""
        if x.dtype != torch.float32 or x.dim() != 2 or not x.is_contiguous() or tuple(x.shape) != (sequences.rows, self.experts.t.hidden):
            raise ValueError(f"x: want contiguous FP32 [{sequences.rows}][{self.experts.t.hidden}], got {list(x.shape)} of {x.dtype}")
        if not sequences.rows:
            return x
        residual = self.attend(*self.project(x), sequences)
        normalized = torch.empty_like(x)
        self.experts.residual_norm(x, residual, normalized, self.weights.post_norm)
        self.feed_forward(x, normalized)
        return x

    __call__ = forward
