"""The paged cache in 8 bits: half the bytes of a bf16 one to keep and to read.

Pools ``k_cache`` / ``v_cache`` [pages * H, P, D] hold codes, ``torch.float8_e4m3fn``
or ``torch.int8``; ``kv_scales`` [pages * H, P, 2] (uint8, or the same bytes as
``torch.float8_e8m0fnu``) one power of two per token and kv head, the keys' and
the values': a row is ``code * 2 ** (byte - 127)``.  The power is the least by
which the row's largest value fits the codes' (448 or 127), so quantising is
exact but for the one rounding to the nearest code (ties to even): e4m3 keeps 4
significant bits of every value, int8 steps of 1/64 to 1/127 of the row's largest.
A row with an infinity or a NaN is held as not a number.

``set_kv_buffer_quant`` writes new tokens, ``read_kv_buffer_quant`` reads rows
back, ``quantized_pool`` gives the page-finish reductions (and with them the
flows' ``forward_cache``) such a pool, and ``decode_attention`` has the attention
over it.  The reference's pools hold the model's type; it has no counterpart.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import _hip
from ..abs import FORMAT, as_vtensor, vTensor


def set_kv_buffer_quant(k_cache: torch.Tensor, v_cache: torch.Tensor, kv_scales: torch.Tensor, new_k: torch.Tensor,
                        new_v: torch.Tensor, loc: torch.Tensor, page_size: int) -> None:
    """Quantises ``new_k`` and ``new_v`` ([nnz, H, D]; bf16, fp16 or fp32, any
    token and head strides) into the pools at the slots ``loc`` (int64).

    A token with a ``loc`` outside the pool (padding: -1) is not stored.  Tokens
    of a call need slots of their own."""
    _hip.set_kv_buffer_quant(k_cache, v_cache, kv_scales, new_k, new_v, loc, int(page_size))


def read_kv_buffer_quant(k_cache: torch.Tensor, v_cache: torch.Tensor, kv_scales: torch.Tensor, loc: torch.Tensor,
                         page_size: int, num_kv_heads: int, dtype: torch.dtype = torch.bfloat16,
                         k_out: Optional[torch.Tensor] = None,
                         v_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The keys and values at the slots ``loc``, [nnz, H, D] each, rounded to
    ``dtype`` (bf16, which holds every value, of e4m3 from 2^-130 on, fp16 or
    fp32); zeros where a slot lies outside the pool.  ``k_out`` / ``v_out``: tensors to write into, of any
    token and head strides, whose type then counts."""
    return _hip.read_kv_buffer_quant(k_cache, v_cache, kv_scales, loc, int(page_size), int(num_kv_heads), dtype, k_out,
                                     v_out)


def quantized_pool(codes: torch.Tensor, kv_scales: torch.Tensor, values: bool = False) -> vTensor:
    """``codes`` (a pool of keys; of values with ``values``) as a PAGED vTensor
    that ``cache.Mean`` / ``Max`` / ``Min`` / ``L2Norm`` / ``MultiReduce`` (dim 1)
    reduce with its factors: a flow's ``cache["k"]``, for example.  Nothing is
    copied; the results are those of a bf16 pool of the same values, but that a row
    which is no number makes its page's Max and Min NaN as well."""
    wrong = _hip._quant_pools_refusal(_hip._plain(codes), _hip._plain(codes), _hip._plain(kv_scales))
    if wrong:
        raise RuntimeError("vortex_torch: " + wrong.replace("k_cache and v_cache", "codes").replace("k_cache", "codes"))
    codes = _hip._plain(codes)
    pool = as_vtensor(codes, FORMAT.PAGED)
    pool._quantized = (codes, _hip._plain(kv_scales), bool(values))
    return pool


__all__ = ["set_kv_buffer_quant", "read_kv_buffer_quant", "quantized_pool"]
