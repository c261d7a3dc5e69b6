"""Paged decode attention over the indexer's block tables.

The reference hands its sparse block table — ``sparse_kv_indptr``,
``sparse_kv_indices`` (entries ``page * H + h``) and ``kv_last_page_len``,
as written by the planner (csrc/utils_sglang.cu:123-184) and top-k
(csrc/topk.cu:56-113) — to FlashInfer's paged decode attention inside its
SGLang fork.  This module is that consumer on gfx950
(``vtx_paged_decode_attention``): one decode token per request, grouped
query heads, the last page of each segment partial.

``sparse_decode_attention`` reads the sparse table from an indexer context,
``dense_decode_attention`` the dense one (full attention over every page).

Requests that share leading pages (a system prompt, samples of one prompt):
``plan_shared_prefix`` finds what they share in a table, once per step, and
``shared_prefix_decode_attention`` reads those pages once for all of them, in
every layer, with ``paged_decode_attention``'s result.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _hip


def paged_decode_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, kv_indptr: torch.Tensor,
                           kv_indices: torch.Tensor, kv_last_page_len: torch.Tensor, batch_size: int,
                           num_kv_heads: int, sm_scale: Optional[float] = None,
                           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of q ([B, H_q, D] or [B*H_kv, G, D], bf16) over the pages of
    each (request, kv head) segment of the table; returns [*q.shape] bf16."""
    D = int(q.shape[-1])
    scale = 1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale)
    o = torch.empty_like(q) if out is None else out
    _hip.paged_decode_attention(q, o, k_cache, v_cache, kv_indptr, kv_indices, kv_last_page_len, batch_size,
                                num_kv_heads, scale)
    return o


def sparse_decode_attention(q, k_cache, v_cache, ctx, sm_scale: Optional[float] = None, out=None):
    """Attention over the pages the indexer selected (ctx's sparse table)."""
    return paged_decode_attention(q, k_cache, v_cache, ctx.sparse_kv_indptr, ctx.sparse_kv_indices,
                                  ctx.kv_last_page_len, ctx.batch_size, ctx.num_kv_heads, sm_scale, out)


def dense_decode_attention(q, k_cache, v_cache, ctx, sm_scale: Optional[float] = None, out=None):
    """Full attention over every page of each request (ctx's dense table)."""
    return paged_decode_attention(q, k_cache, v_cache, ctx.dense_kv_indptr, ctx.dense_kv_indices,
                                  ctx.kv_last_page_len, ctx.batch_size, ctx.num_kv_heads, sm_scale, out)


class SharedPrefixPlan:
    """What ``plan_shared_prefix`` found in a block table, per segment
    ``b * num_kv_heads + h`` (int32, on the GPU): ``leaders``, the first request
    of its run, and ``shared_pages``, the leading pages that the run shares.
    ``buffer`` holds them, and the division of the attention's work."""

    def __init__(self, buffer: torch.Tensor, batch_size: int, num_kv_heads: int, group_size: int, head_dim: int,
                 page_size: int):
        self.buffer = buffer
        self.sizes = (int(batch_size), int(num_kv_heads), int(group_size), int(head_dim), int(page_size))

    def _part(self, i: int) -> torch.Tensor:
        segments = self.sizes[0] * self.sizes[1]
        return self.buffer.narrow(0, 16 + i * ((segments + 7) // 8 * 8), segments)

    @property
    def leaders(self) -> torch.Tensor:
        return self._part(0)

    @property
    def shared_pages(self) -> torch.Tensor:
        return self._part(1)


def plan_shared_prefix(kv_indptr: torch.Tensor, kv_indices: torch.Tensor, batch_size: int, num_kv_heads: int,
                       group_size: int, head_dim: int, page_size: int, group_ids: Optional[torch.Tensor] = None,
                       plan: Optional[SharedPrefixPlan] = None) -> SharedPrefixPlan:
    """Finds the pages that requests of a block table share.  Per kv head,
    consecutive requests form a run while their ``group_ids`` (int32 [batch])
    are equal, or without ids while their first pages are; the run shares its
    longest common prefix of entries (which is looked up: ids promise nothing),
    except each request's own last page.  Sharing has one level: where all requests
    begin with one page (a system prompt) and groups of them share what follows,
    pass the groups' ids, or that page is all that is shared.  group_size: query
    heads per kv head.

    Plan anew whenever entries or lengths in pages change (``kv_last_page_len``
    may).  ``plan``: an earlier plan of the same sizes to write into, as a
    captured step needs it."""
    sizes = (int(batch_size), int(num_kv_heads), int(group_size), int(head_dim), int(page_size))
    if plan is not None and plan.sizes != sizes:
        raise RuntimeError(
            f"vortex_torch: plan is for (batch, kv heads, group, head_dim, page) {plan.sizes}, not {sizes}")
    buffer = _hip.plan_shared_prefix(kv_indptr, kv_indices, group_ids, *sizes, None if plan is None else plan.buffer)
    return SharedPrefixPlan(buffer, *sizes) if plan is None else plan


def shared_prefix_decode_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                                   kv_indptr: torch.Tensor, kv_indices: torch.Tensor, kv_last_page_len: torch.Tensor,
                                   plan: SharedPrefixPlan, sm_scale: Optional[float] = None,
                                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``paged_decode_attention`` over the table that ``plan`` was made of,
    every shared page read once for its run.  The probabilities are rounded to
    bf16 for the matrix cores; sums and outputs are fp32, rounded once."""
    B, H, G, D, P = plan.sizes
    if k_cache.dim() != 3 or k_cache.shape[1] != P or k_cache.shape[2] != D:
        raise RuntimeError(
            f"vortex_torch: k_cache must be [pages * H, {P}, {D}] as planned, got {tuple(k_cache.shape)}")
    scale = 1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale)
    o = torch.empty_like(q) if out is None else out
    _hip.shared_prefix_decode_attention(q, o, k_cache, v_cache, kv_indptr, kv_indices, kv_last_page_len, plan.buffer,
                                        B, H, G, scale)
    return o


__all__ = ["paged_decode_attention", "sparse_decode_attention", "dense_decode_attention", "SharedPrefixPlan",
           "plan_shared_prefix", "shared_prefix_decode_attention"]
