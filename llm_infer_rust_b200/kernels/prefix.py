"""Decode attention of rows that share their first keys: a group's shared keys are read once for all of its rows.

Several answers to one prompt hold the prompt's pages in common.  ``ops.decode_attention`` reads them once for every row;
here the query vectors of a group's rows are the rows of one product with the shared keys, each row's own keys follow, and one
softmax goes over both:

    out[r, h] = sum_j p_j v_j,  p = softmax_j(scale q[r, h] . k_j),  j = 0 .. kv_len[r] - 1

with keys below the group's ``shared`` read through the block table of the group's first row, the others through the row's own.
"""
from __future__ import annotations

import ctypes

import torch

from . import ops
from .build import load_entry_points
from .ops import KernelError

_TILE = 32                    # query vectors of a CTA of the all-sizes kernel
_TC_VECTORS = 128             # of a tile of the tcgen05 kernel; a CTA takes one or two
_KEYS_PER_CTA_AT_LEAST = 64
_MOST_SPLITS = 64             # of the shared keys
_MOST_ENTRIES = 400           # rows and groups of a call that the tensor-core kernels take


def _lib(head_dim: int):
    return load_entry_points("prefix_attention.cu", {"HEAD_DIM": ops.padded_head_dim(head_dim)})


def _on_tcgen05(head_dim: int, vectors: int, most_shared: int) -> bool:
    """Whether a group's shared keys go to the tcgen05 kernel (``vectors``: its query vectors of a KV head)."""
    return head_dim == 128 and vectors > 32 and most_shared >= 256


def _split(most_shared: int, most_own: int, shared_ctas: int, own_ctas: int, room: int, least: int) -> tuple:
    """Into how many splits the shared and the own keys are cut, ``shared_ctas`` and ``own_ctas`` CTAs for each split: about as
    many keys a CTA on both sides, at least ``least``, and about ``room`` CTAs in all."""
    a_cta = max(least, -(-(most_shared * shared_ctas + most_own * own_ctas) // max(1, room)))
    return max(1, min(64, -(-most_shared // a_cta))), max(1, min(64, -(-most_own // a_cta)))


def prefix_attention(q, k_cache, v_cache, out, block_table, cu_q, kv_len, rows, groups, num_heads, num_kv_heads, head_dim, page_size,
                     scale, *, most_rows, most_shared, most_own) -> None:
    """Attention of single decoded tokens behind shared keys; operands as ``ops.decode_attention`` takes them.

    ``rows`` (int32) lists the batch rows to serve group by group; ``groups`` (int32 [groups, 2]) holds for each group the index
    of its first row in ``rows`` (0 for the first group, rising) and how many keys its rows share.  The shared keys need not end
    with a page; a row that sees fewer keys than its group shares sees those.  A row of no keys gets zeros.

    ``most_rows``, ``most_shared`` and ``most_own`` are about how many rows a group has, how many keys it shares and how many keys
    a row has beyond them, at most: they decide how the work is cut up (and what a captured graph is cut up for), not the result's
    meaning.  Page ids outside the pool and rows longer than their block table set the error word (``ops.check_errors``)."""
    ops._cuda(q, k_cache, v_cache, out, block_table, cu_q, kv_len, rows, groups)
    ops._contig(q, k_cache, v_cache, out, block_table, cu_q, kv_len, rows, groups)
    code = ops._code(q)
    if k_cache.dtype != q.dtype or v_cache.dtype != q.dtype or out.dtype != q.dtype:
        raise KernelError("q, cache and output must share a dtype")
    if any(t.dtype != torch.int32 for t in (block_table, cu_q, kv_len, rows, groups)):
        raise KernelError("block table, cu_q, kv_len, rows and groups are int32")
    if num_kv_heads <= 0 or num_heads <= 0 or num_heads % num_kv_heads:
        raise KernelError("num_heads must be a multiple of num_kv_heads")
    if head_dim % 2 or not 2 <= head_dim <= 512:
        raise KernelError(f"head size {head_dim} is refused: the attention kernels take even head sizes up to 512")
    ops._check_cache(k_cache, v_cache, num_kv_heads, page_size, head_dim, head_dim)
    if k_cache.shape != v_cache.shape:
        raise KernelError("keys and values have as many pages")
    if q.shape[-1] != num_heads * head_dim or out.shape != q.shape or q.dim() != 2:
        raise KernelError("q and out are [tokens, num_heads * head_dim]")
    if block_table.dim() != 2 or block_table.shape[1] == 0 or rows.dim() != 1 or groups.dim() != 2 or groups.shape[1] != 2:
        raise KernelError("block_table is [rows, pages], rows [n], groups [groups, 2]")
    if not scale > 0.0:
        raise KernelError("the scale must be positive")
    if min(most_rows, most_shared, most_own) < 0:
        raise KernelError("most_rows, most_shared and most_own must not be negative")
    ops._on_current(q.device)
    n_rows, n_groups = rows.shape[0], groups.shape[0]
    if n_rows == 0:
        return
    per = num_heads // num_kv_heads
    most_rows = max(1, min(most_rows, n_rows))
    lib = _lib(head_dim)
    # (the splits' parts stand between the kernels of the call, in memory of the call's own)
    err, stream, sms = ops.error_word(q.device), ops._stream(), ops._sm_count(q.device)
    common = (block_table, block_table.shape[1], cu_q, kv_len, rows, n_rows, groups, n_groups, num_heads, num_kv_heads, page_size,
              k_cache.shape[0], float(scale))

    if not ops.decode_uses_tensor_cores(q.dtype, num_heads, num_kv_heads, head_dim, page_size) or (q.data_ptr() | out.data_ptr()) % 16 \
            or n_rows + n_groups > _MOST_ENTRIES:
        lib = _lib(head_dim)
        tiles = -(-most_rows * per // _TILE)
        per_sm = max(1, 227 * 1024 // (lib.b200_prefix_attention_smem() + 1024))
        shared, own = _split(most_shared, most_own, n_groups * num_kv_heads * tiles, n_rows * num_kv_heads * -(-per // _TILE), per_sm * sms,
                             _KEYS_PER_CTA_AT_LEAST)
        scratch = ops._empty((n_rows * num_heads * (shared + own) * (ops.padded_head_dim(head_dim) + 2),), torch.float32, q.device)
        rc = lib.b200_prefix_attention(q, k_cache, v_cache, out, scratch, *common, shared, own, tiles, code, head_dim, err, stream)
        ops._ok(rc, "prefix_attention", 2)
        return
    lib = load_entry_points("prefix_mma.cu", {"HEAD_DIM": head_dim})
    covered = shared = 0
    if n_groups and _on_tcgen05(head_dim, most_rows * per, most_shared):
        two = most_rows * per > _TC_VECTORS
        covered = _TC_VECTORS * (2 if two else 1)
        tiles = -(-most_rows * per // covered)
        ctas = max(1, min(-(-most_shared // (128 if two else 256)), sms // (n_groups * num_kv_heads * tiles), _MOST_SPLITS if two else _MOST_SPLITS // 2))
        shared, covered = ctas * (1 if two else 2), covered * tiles
    floats = lib.library.b200_prefix_scratch_floats
    floats.restype = ctypes.c_longlong
    scratch = ops._empty((floats(n_rows, n_groups, num_heads, num_kv_heads, shared, sms),), torch.float32, q.device)
    if covered:
        rc = load_entry_points("prefix_tcgen05.cu").b200_prefix_tcgen05(q, k_cache, v_cache, scratch, *common, shared, tiles, int(two), err, stream)
        ops._ok(rc, "prefix_tcgen05")
    rc = lib.b200_prefix_attention_mma(q, k_cache, v_cache, out, scratch, *common, shared, covered, sms, err, stream)
    ops._ok(rc, "prefix_attention_mma", 2)
