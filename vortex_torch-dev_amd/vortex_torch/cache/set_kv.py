"""Writes new keys and values into the paged K / V pools.

``set_kv_buffer_launcher`` keeps the reference's name and arguments
(vortex_torch/cache/triton_kernels/set_kv.py:45-63): token i's row for kv
head h goes to pool row ``(loc[i] // P) * (P * H) + h * P + loc[i] % P`` of
``k_cache`` / ``v_cache`` ([pages * H, P, D]), the layout the page-finish
reductions and the indexer read.  Kernel: ``vtx_set_kv_buffer``.

``set_kv_buffer_rope`` rotates the queries and keys to their positions on the
way, in the same launch (the reference's runtime rotates before it stores).
Kernel: ``vtx_set_kv_buffer_rope``.
"""
from __future__ import annotations

from typing import Optional

import torch

from .. import _hip


def set_kv_buffer_launcher(k_cache: torch.Tensor, v_cache: torch.Tensor, new_k: torch.Tensor,
                           new_v: torch.Tensor, loc: torch.Tensor, page_size: int) -> None:
    _hip.set_kv_buffer(k_cache, v_cache, new_k, new_v, loc, page_size)


def set_kv_buffer_rope(k_cache: torch.Tensor, v_cache: torch.Tensor, q: Optional[torch.Tensor], new_k: torch.Tensor,
                       new_v: torch.Tensor, loc: torch.Tensor, page_size: int, positions: torch.Tensor,
                       cos_sin_cache: torch.Tensor, interleaved: bool = False,
                       q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Rotates ``q`` [nnz, Hq, D] and ``new_k`` [nnz, H, D] to ``positions``
    (int64), stores the keys and ``new_v`` at the slots ``loc`` of the pools and
    returns the rotated queries (``q_out``, which may be ``q``, or a new tensor;
    None without ``q``).

    ``cos_sin_cache``: fp32 [positions, R], R / 2 cosines and then as many
    sines per position.  Column pairs (j, j + R / 2) of a row's first R columns
    are rotated, or (2j, 2j + 1) with ``interleaved``.  bf16, fp16 or fp32; the
    new tokens' rows may be slices of one projection's output (any token and
    head strides).

    A token with a ``loc`` outside the pool (padding: -1) is not stored; one
    with a position outside the table is skipped, its ``q_out`` rows unwritten.
    Tokens of a call need slots of their own: where two share one, each value
    there is either's."""
    return _hip.set_kv_buffer_rope(k_cache, v_cache, q, new_k, new_v, loc, int(page_size), positions, cos_sin_cache,
                                   bool(interleaved), q_out)


__all__ = ["set_kv_buffer_launcher", "set_kv_buffer_rope"]
