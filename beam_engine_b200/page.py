"""``append_paged_kv_cache`` with FlashInfer's signature, on the native kernel.

Replaces ``flashinfer.page.append_paged_kv_cache`` as the reference calls it
from ``PageTable.write_blocks_vectorized`` (src/beam_engine/page_table.py:199-209):
entry ``i`` lands in page ``kv_indices[kv_indptr[batch_indices[i]] +
positions[i] // page_size]`` at slot ``positions[i] % page_size``
(``kv_last_page_len`` is accepted and unused, as in FlashInfer's append).

A ``float8_e4m3fn`` cache takes its scales as ``kv_scale`` (float32 [pages, 2, kv_heads],
one per page, K | V and head; zeros before the first write): values = codes * scale.
The rows are rounded to the block's scale, a power of two under which the block's largest
finite value is at most 448.  A call that writes a page's slot 0 begins the page anew; any other
keeps the scale or raises it, and where it raises it the tokens that were there are rounded
to it.  With ``rope_inv_freq`` (float32 [head_dim / 2]) the keys are rotated to
``rope_positions`` (default: ``positions``) on the way, into any cache type.
``read_paged_kv_cache`` gives pages of an 8-bit cache back as values.
"""
from __future__ import annotations

import torch

from ._lib import check, lib
from .page_table import (_DT, _int32, append_rows, check_pool8, dtype_code, is_8bit, on_device,
                         raw_stream, require_cuda, require_same_device, stream_ptr)


def append_paged_kv_cache(append_key: torch.Tensor, append_value: torch.Tensor,
                          batch_indices: torch.Tensor, positions: torch.Tensor,
                          paged_kv_cache: torch.Tensor, kv_indices: torch.Tensor,
                          kv_indptr: torch.Tensor, kv_last_page_len: torch.Tensor = None,
                          kv_layout: str = "NHD", kv_scale: torch.Tensor = None,
                          rope_inv_freq: torch.Tensor = None,
                          rope_positions: torch.Tensor = None) -> None:
    if kv_layout != "NHD":
        raise ValueError("only the NHD layout is supported")
    if paged_kv_cache.dim() != 5 or paged_kv_cache.shape[1] != 2:
        raise ValueError("paged_kv_cache must be [pages, 2, page_size, kv_heads, head_dim]")
    if not paged_kv_cache.is_contiguous():
        raise ValueError("paged_kv_cache must be contiguous")
    if is_8bit(paged_kv_cache.dtype):
        check_pool8(paged_kv_cache, kv_scale)
        return append_rows(append_key, append_value, batch_indices, positions, paged_kv_cache,
                           kv_scale, kv_indices, kv_indptr, rope_inv_freq, rope_positions)
    if kv_scale is not None:
        raise ValueError(f"kv_scale belongs to a float8_e4m3fn cache, this one is "
                         f"{paged_kv_cache.dtype}")
    if rope_inv_freq is not None:
        return append_rows(append_key.to(paged_kv_cache.dtype),
                           append_value.to(paged_kv_cache.dtype), batch_indices, positions,
                           paged_kv_cache, None, kv_indices, kv_indptr, rope_inv_freq,
                           rope_positions)
    require_cuda(append_key, append_value, paged_kv_cache, batch_indices, positions, kv_indices,
                 kv_indptr)
    P, _, ps, H, D = paged_kv_cache.shape
    k = append_key.to(paged_kv_cache.dtype)
    v = append_value.to(paged_kv_cache.dtype)
    if k.stride(-1) != 1 or k.stride(-2) != D:
        k = k.contiguous()
    if v.stride(-1) != 1 or v.stride(-2) != D or v.stride(0) != k.stride(0):
        k, v = k.contiguous(), v.contiguous()
    ints = [t.to(torch.int32) for t in (batch_indices, positions, kv_indices, kv_indptr)]
    rc = lib().be_append_paged_kv(k.data_ptr(), v.data_ptr(), k.stride(0), 0, ints[0].data_ptr(),
                                  ints[1].data_ptr(), ints[2].data_ptr(), ints[3].data_ptr(),
                                  k.shape[0], paged_kv_cache.data_ptr(), 0, 1, P, ps, H, D,
                                  dtype_code(paged_kv_cache.dtype),
                                  stream_ptr(paged_kv_cache.device))
    check(rc, "append_paged_kv_cache")


def read_paged_kv_cache(paged_kv_cache: torch.Tensor, pages: torch.Tensor, kv_scale: torch.Tensor,
                        dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """Pages ``pages`` [n] of an 8-bit cache as values [n, 2, page_size, kv_heads, head_dim]."""
    if not is_8bit(paged_kv_cache.dtype) or paged_kv_cache.dim() != 5 or \
            paged_kv_cache.shape[1] != 2 or not paged_kv_cache.is_contiguous():
        raise ValueError("paged_kv_cache must be contiguous float8_e4m3fn "
                         "[pages, 2, page_size, kv_heads, head_dim]")
    check_pool8(paged_kv_cache, kv_scale)
    if dtype not in _DT:
        raise ValueError(f"unsupported dtype {dtype}")
    if pages.dim() != 1:
        raise ValueError("pages must be [n]")
    require_same_device(paged_kv_cache, kv_scale, pages)
    pages = _int32(pages)
    P, _, ps, H, D = paged_kv_cache.shape
    n, dev = pages.shape[0], paged_kv_cache.device
    out = paged_kv_cache.new_empty((n, 2, ps, H, D), dtype=dtype)
    with on_device(dev.index):
        rc = lib().be_read_paged_kv8(paged_kv_cache.data_ptr(), kv_scale.data_ptr(),
                                     pages.data_ptr(), n, P, ps, H, D, out.data_ptr(), _DT[dtype],
                                     raw_stream(dev.index))
    if rc:
        check(rc, "read_paged_kv_cache")
    return out
