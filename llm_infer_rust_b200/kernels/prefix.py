"""Decode attention of rows that share their first keys: a group's shared keys are read once for all of its rows.

Several answers to one prompt hold the prompt's pages in common.  ``ops.decode_attention`` reads them once for every row;
here the query vectors of a group's rows are the rows of one product with the shared keys, each row's own keys follow, and one
softmax goes over both:

    out[r, h] = sum_j p_j v_j,  p = softmax_j(scale q[r, h] . k_j),  j = 0 .. kv_len[r] - 1

with keys below the group's ``shared`` read through the block table of the group's first row, the others through the row's own.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import ops
from .build import load_call_binding, load_entry_points
from .ops import KernelError

_TILE = 32                    # query vectors of a CTA of the all-sizes kernel
_TC_VECTORS = 128             # of a tile of the tcgen05 kernel; a CTA takes one or two
_KEYS_PER_CTA_AT_LEAST = 32
_MOST_SPLITS = 64
_MOST_ENTRIES = 400           # rows and groups of a call that the tensor-core kernels take
# The tcgen05 kernel takes the shared keys of more vectors of a KV head than the mma.sync kernel has in a tile, from so many blocks on (32 keys
# of a KV head against 16 vectors each), which goes by the steps that a CTA would have.  (mma.sync / tcgen05, us, 8 KV heads of 128, a step: 32
# vectors, 3,000 keys 13.7 / 14.3, 4,096 keys 15.9 / 12.9; 64 vectors, 1,000 keys 12.8 / 14.0, 1,500 keys 14.3 / 14.2, 2,000 keys 16.3 / 14.7; 128
# vectors, 512 keys 13.4 / 14.6, 1,024 keys 16.4 / 15.0; 256 vectors, 512 keys 19.5 / 18.9.  Two: 32 vectors, 5,000 keys 16.7 / 17.9, 6,500 keys 20.2 / 16.4;
# 256 vectors, 8,192 keys 99 / 28.  One KV head, a step: 128 vectors, 4,096 keys 11.5 / 13.4, 8,192 keys 15.4 / 13.9; 512 vectors, 2,048 keys 15.8 /
# 16.2, 4,096 keys 20.8 / 17.3.)  Several groups are as a rule unlike in their rows and keys, and `blocks` counts
# each as the largest, so it has to be more then: of up to 24 vectors six behind up to 3,001 keys (9,024 blocks) 20.8 / 28.8, of up to 80
# three behind 500 (1,920) 14.7 / 15.6 and behind 1,500 (5,640) 19.2 / 18.5, of up to 48 six behind 700 (3,168) 15.4 / 18.0, of up to 64
# twelve behind 1,000 (12,288) 31.0 / 29.4.
_TENSOR_CORE_BLOCKS, _TENSOR_CORE_BLOCKS_A_STEP, _TENSOR_CORE_BLOCKS_OF_GROUPS = 600, 1150, 12288
_MMA_VECTORS = _TENSOR_CORE_VECTORS = 16      # of a tile of the mma.sync kernel; more than which the other takes


def _splits(most_shared: int, most_own: int, shared_ctas: int, own_ctas: int, room: int) -> tuple:
    """Into how many splits the all-sizes kernel cuts the shared and the own keys, ``shared_ctas`` and ``own_ctas`` CTAs for each split:
    about as many keys a CTA on both sides, and about twice ``room`` CTAs in all (a CTA is a chain of waits; groups and rows are often
    smaller than the largest)."""
    a_cta = max(_KEYS_PER_CTA_AT_LEAST, -(-(most_shared * shared_ctas + most_own * own_ctas) // max(1, 2 * room)))
    return max(1, min(_MOST_SPLITS, -(-most_shared // a_cta))), max(1, min(_MOST_SPLITS, -(-most_own // a_cta)))


# What the tcgen05 kernel takes beside its steps, and a step: one tile of vectors (a block of keys for each of two streams), two tiles (a
# block for both).  What the stream kernel takes beside its bytes, bytes that one of few SMs and all of them together take in, and the
# keys that an item costs beside its own (us, bytes a us).
_TC_FIXED, _TC_STEP = (5.0, 12.0), (2.9, 1.8)
_OWN_FIXED, _OWN_BYTES, _OWN_BYTES_ALL, _OWN_KEYS = 5.0, 78000.0, 6.5e6, 64


def _most_ctas(steps: int, tiles: int, sms: int) -> int:
    return max(1, min(steps, sms // tiles, _MOST_SPLITS))


def _share_sms(steps: int, two: int, tiles: int, items: int, most_own: int, key_bytes: int, sms: int) -> tuple:
    """How many CTAs cut each of ``tiles`` tiles' ``steps``, and the CTAs of the stream kernel for ``items`` of own keys (half of ``most_own``
    each): side by side on SMs of their own, as the registers and shared memory of either leave no room for the other, or one behind the
    other on all.  (64 rows of 32 heads behind 32,768 keys, own keys of 1 to 1,024: 13 CTAs a tile beside 44 SMs 66.6 us, 10 beside 68
    77.2, 15 beside 28 90.8, one behind the other 79.5; 24 rows of 64 heads behind 8,000 keys, 1 to 200: 26.0 and 29.3.)"""
    own_bytes = items * (most_own / 2 + _OWN_KEYS) * key_bytes
    of_tc = lambda ctas: _TC_FIXED[two] + _TC_STEP[two] * -(-steps // ctas)
    most = _most_ctas(steps, tiles, sms)
    best = of_tc(most) + _OWN_FIXED + own_bytes / _OWN_BYTES_ALL, most, sms
    for ctas in range(1, most + 1):
        left = sms - ctas * tiles
        if left >= 1:
            best = min(best, (max(of_tc(ctas), _OWN_FIXED + own_bytes / min(left * _OWN_BYTES, _OWN_BYTES_ALL)), ctas, left))
    return best[1:]


@functools.lru_cache(maxsize=4096)
def _plan(dtype, heads: int, kv_heads: int, dim: int, page: int, n_rows: int, n_groups: int, most_rows: int, most_shared: int, most_own: int,
          sharing: int, taken: bool, sms: int) -> tuple:
    """The entry points that a call goes to (all sizes, tcgen05, mma.sync; None: not this one), its sizes as the binding takes them, and
    its launches.  ``taken``: its tensors are aligned and counted as the tensor-core kernels take them."""
    per = heads // kv_heads
    most_rows = max(1, min(most_rows, n_rows))
    vectors = most_rows * per
    sharing = max(1, min(sharing, n_groups))
    # (pages of any size: powers of two in what decode attention asks for and the tcgen05 kernel fetches, not here)
    if not taken or not on_tensor_cores(dtype, heads, kv_heads, dim, n_rows, n_groups):
        lib = load_entry_points("prefix_attention.cu", {"HEAD_DIM": ops.padded_head_dim(dim)})
        tiles = -(-vectors // _TILE)
        per_sm = max(1, 227 * 1024 // (lib.b200_prefix_attention_smem() + 1024))
        shared, own = _splits(most_shared, most_own, sharing * kv_heads * tiles, n_rows * kv_heads * -(-per // _TILE), per_sm * sms)
        floats = n_rows * heads * (shared + own) * (ops.padded_head_dim(dim) + 2)
        return lib.b200_prefix_attention, None, None, (floats, shared, own, tiles, 0, 0, 0, sms), 2
    tcgen05, tiles, two, shared, covered, stream, served = None, 1, 0, 0, 0, sms, 0
    blocks = -(-vectors // _MMA_VECTORS) * -(-most_shared // 32) * kv_heads * sharing
    if n_groups and dim == 128 and page & (page - 1) == 0 and vectors > _TENSOR_CORE_VECTORS:
        # one or two tiles a CTA, none without a block of keys for each of its streams
        two = int(vectors > _TC_VECTORS)
        tiles = -(-vectors // (_TC_VECTORS << two))
        steps, all_tiles = max(1, -(-most_shared // (256 >> two))), sharing * kv_heads * tiles
        least = _TENSOR_CORE_BLOCKS_OF_GROUPS if sharing > 1 else \
            _TENSOR_CORE_BLOCKS + _TENSOR_CORE_BLOCKS_A_STEP * -(-steps // _most_ctas(steps, all_tiles, sms))
        if blocks >= least:
            ctas, stream = _share_sms(steps, two, all_tiles, n_rows * kv_heads, most_own, 4 * dim, sms)
            shared, covered, served = ctas << (1 - two), tiles * (_TC_VECTORS << two), sharing
            tcgen05 = load_entry_points("prefix_tcgen05.cu").b200_prefix_tcgen05
    lib = load_entry_points("prefix_mma.cu", {"HEAD_DIM": dim})
    count = lib.library.b200_prefix_scratch_floats
    count.restype = ctypes.c_longlong
    floats = count(n_rows, n_groups, heads, kv_heads, shared, stream)
    return None, tcgen05, lib.b200_prefix_attention_mma, (floats, shared, served, tiles, two, covered, stream, sms), 2 + (tcgen05 is not None)


def on_tensor_cores(dtype, num_heads: int, num_kv_heads: int, head_dim: int, n_rows: int, n_groups: int) -> bool:
    """Whether calls of these sizes go to the tensor-core kernels (if their tensors are aligned)."""
    return ops.decode_uses_tensor_cores(dtype, num_heads, num_kv_heads, head_dim, 1) and n_rows + n_groups <= _MOST_ENTRIES


def pays(dtype, num_heads: int, num_kv_heads: int, head_dim: int, page_size: int, n_rows: int, n_groups: int, saved_keys: int, read_keys: int,
         least: int) -> bool:
    """Whether ``prefix_attention`` of ``n_rows`` rows in ``n_groups`` groups is quicker than ``ops.decode_attention`` of the same rows, where it
    reads ``read_keys`` keys in all and ``saved_keys`` less than that.  ``least``: bytes that are to be saved in the usual case.

    On the tensor cores (decode attention / shared, us): what a call takes beside its bytes is made up for by 48 MiB, and by 64 MiB where
    more than two query heads share a KV head and their parts are joined (16 heads on 8 KV heads of 128: 16 rows 39 MiB 10.0 / 10.5, 48 MiB
    11.1 / 10.8; 32 on 8: 16 rows 55 MiB 13.5 / 13.8; 64 on 8: 16 rows 55 MiB 14.6 / 16.2, 64 MiB 15.0 / 14.7; 16 on 1: 16 rows 48 MiB 16.4 / 17.4, 64
    MiB 18.9 / 17.9).  Keys that a row has to itself are read up to a twelfth slower, so a sixth of what is read has to be saved (128 rows
    with 600 of their own, 300 MiB: 32 MiB saved 69.3 / 72.4, 64 74.1 / 62.5; 384 rows, 900 MiB: 48 203 / 221, 120 204 / 180; eight rows beside 60
    of 2,000 that share nothing, 470 MiB: 64 91.6 / 93.5, 128 110 / 96).
    float32 gains from the smallest (two rows 16 MiB 39.2 / 19.9, 450 rows 28 MiB of 2.3 GiB 561 / 353), and so do more than 16 query heads
    on a KV head (32 on 1: 450 rows 14 MiB 200 / 76): two thirds.
    Other bfloat16 calls go to the all-sizes kernel, element by element: never where decode attention has its tensor-core kernel (more rows
    and groups than the others take: 450 rows of 64 keys, 505 MiB saved, 154 / 230), else where eight times as much is saved as
    read (heads of 72: 64 rows of 600 keys, 1.5 times, 136 / 143, 16 of 64, 11 times, 94 / 24; heads of 320: 64 rows, 3 times, 111 / 145, 12
    times, 244 / 210)."""
    saved = 2 * saved_keys * num_kv_heads * head_dim * dtype.itemsize
    group = num_heads // num_kv_heads
    if dtype == torch.bfloat16 and group <= ops.MMA_MAX_GROUP:
        if on_tensor_cores(dtype, num_heads, num_kv_heads, head_dim, n_rows, n_groups):
            return saved >= (least if group <= 2 else least * 4 // 3) and 6 * saved_keys >= read_keys
        if ops.decode_uses_tensor_cores(dtype, num_heads, num_kv_heads, head_dim, page_size) or saved_keys < 8 * read_keys:
            return False
    return saved >= least * 2 // 3


def _counts(k_cache, block_table, n_rows: int, n_groups: int, num_heads: int, num_kv_heads: int, page_size: int) -> bool:
    """Whether the tensor-core kernels, which count a cache's rows and a call's blocks of keys in 32 bits, can count a call's (as
    ``prefix_attention`` of csrc/binding/calls.cpp asks)."""
    places = block_table.shape[1] * page_size
    items = -(-n_rows * (num_heads // num_kv_heads) // 16) + n_groups + n_rows
    return k_cache.shape[0] * num_kv_heads * page_size < 1 << 31 and (places // 32 + 2) * num_kv_heads * items < 1 << 30


def _refuse(q, k_cache, v_cache, out, block_table, cu_q, kv_len, rows, groups, num_heads, num_kv_heads, head_dim, page_size, scale) -> None:
    """Says what is wrong with a call's operands."""
    ops._cuda(q, k_cache, v_cache, out, block_table, cu_q, kv_len, rows, groups)
    ops._contig(q, k_cache, v_cache, out, block_table, cu_q, kv_len, rows, groups)
    ops._code(q)
    if k_cache.dtype != q.dtype or v_cache.dtype != q.dtype or out.dtype != q.dtype:
        raise KernelError("q, cache and output must share a dtype")
    if any(t.dtype != torch.int32 for t in (block_table, cu_q, kv_len, rows, groups)):
        raise KernelError("block table, cu_q, kv_len, rows and groups are int32")
    if any(t.device != q.device for t in (k_cache, v_cache, out, block_table, cu_q, kv_len, rows, groups)):
        raise KernelError("the operands are on several devices")
    ops._check_cache(k_cache, v_cache, num_kv_heads, page_size, head_dim, head_dim)
    if k_cache.shape != v_cache.shape or k_cache.shape[0] < 1 or page_size < 1:
        raise KernelError("keys and values have as many pages")
    if q.dim() != 2 or q.shape[1] != num_heads * head_dim or out.shape != q.shape:
        raise KernelError("q and out are [tokens, num_heads * head_dim]")
    if block_table.dim() != 2 or block_table.shape[1] == 0 or any(t.dim() != 1 for t in (cu_q, kv_len, rows)) or groups.dim() != 2 or groups.shape[1] != 2:
        raise KernelError("block_table is [rows, pages], cu_q, kv_len and rows are [n], groups is [groups, 2]")
    if not scale > 0.0:
        raise KernelError("the scale must be positive")


def prefix_attention(q, k_cache, v_cache, out, block_table, cu_q, kv_len, rows, groups, num_heads, num_kv_heads, head_dim, page_size,
                     scale, *, most_rows, most_shared, most_own, sharing_groups=None) -> None:
    """Attention of single decoded tokens behind shared keys; operands as ``ops.decode_attention`` takes them.

    ``rows`` (int32) lists the batch rows to serve group by group; ``groups`` (int32 [groups, 2]) holds for each group the index
    of its first row in ``rows`` (0 for the first group, rising) and how many keys its rows share.  The shared keys need not end
    with a page; a row that sees fewer keys than its group shares sees those (the others, which its group's longer rows see, have to be
    finite: they are multiplied by weights of zero).  A row of no keys gets zeros.  Each row stands in ``rows`` once; ``out`` may be ``q``.

    ``most_rows``, ``most_shared`` and ``most_own`` are about how many rows a group has, how many keys it shares and how many keys
    a row has beyond them, at most (where one row has far more than the others and the tensor-core kernels serve the call: twice the rows' mean),
    ``sharing_groups`` about how many of the groups, the first ones, share keys (None: all): they decide how the work is
    cut up (and what a captured graph is cut up for), not the result's meaning.  Page ids outside the pool and rows longer than
    their block table (of at most 2^30 places) set the error word (``ops.check_errors``); the other index arrays are taken at their word, as ``ops.decode_attention`` takes them."""
    if num_kv_heads <= 0 or num_heads <= 0 or num_heads % num_kv_heads:
        raise KernelError("num_heads must be a multiple of num_kv_heads")
    if head_dim % 2 or not 2 <= head_dim <= 512:
        raise KernelError(f"head size {head_dim} is refused: the attention kernels take even head sizes up to 512")
    if most_rows < 0 or most_shared < 0 or most_own < 0 or (sharing_groups is not None and sharing_groups < 0):
        raise KernelError("most_rows, most_shared, most_own and sharing_groups must not be negative")
    if ops._held is not None or ops._chain is not None:
        ops.flush_chain()                        # (what waits in the chain may be what is read here)
    operands = (q, k_cache, v_cache, out, block_table, cu_q, kv_len, rows, groups)
    sizes = (num_heads, num_kv_heads, head_dim, page_size)
    if not rows.is_cuda or rows.dim() != 1 or groups.dim() != 2 or page_size < 1:
        _refuse(*operands, *sizes, scale)
    n_rows = rows.shape[0]
    if n_rows == 0:
        _refuse(*operands, *sizes, scale)
        return
    device = rows.device
    ops._on_current(device)
    ends = (ops.error_word(device), ops._stream())
    chosen = (q.dtype, num_heads, num_kv_heads, head_dim, page_size, n_rows, groups.shape[0], most_rows, most_shared, most_own,
              groups.shape[0] if sharing_groups is None else sharing_groups)
    sms, scale = ops._sm_count(device), float(scale)
    all_sizes, tcgen05, mma, plan, kernels = _plan(*chosen, True, sms)
    rc = _binding().prefix_attention(all_sizes, tcgen05, mma, *operands, *sizes, scale, plan, *ends)
    if rc is None:
        # something is not as it should be, the tensor-core kernels cannot take the call, or this thread keeps a layer's calls
        # (ops.LayerCalls), which the entry points take part in
        _refuse(*operands, *sizes, scale)
        taken = (q.data_ptr() | k_cache.data_ptr() | v_cache.data_ptr() | out.data_ptr()) % 16 == 0 and \
            _counts(k_cache, block_table, n_rows, groups.shape[0], num_heads, num_kv_heads, page_size)
        all_sizes, tcgen05, mma, plan, kernels = _plan(*chosen, taken, sms)
        floats, shared, own, tiles, two, covered, stream, _ = plan
        scratch = ops._empty((floats,), torch.float32, device)
        common = (scratch, block_table, block_table.shape[1], cu_q, kv_len, rows, n_rows, groups, groups.shape[0], num_heads, num_kv_heads, page_size,
                  k_cache.shape[0], scale)
        if all_sizes is not None:
            rc = all_sizes(q, k_cache, v_cache, out, *common, shared, own, tiles, ops._code(q), head_dim, sms, *ends)
        else:
            # (`own`: the groups that the tcgen05 kernel serves)
            rc = tcgen05(q, k_cache, v_cache, *common, shared, tiles | own << 16, two, *ends) if tcgen05 is not None else 0
            rc = rc or mma(q, k_cache, v_cache, out, *common, shared, covered | own << 16, stream, sms, *ends)
    ops._ok(rc, "prefix_attention", kernels)


_loaded = None


def _binding():
    global _loaded
    if _loaded is None:
        _loaded = load_call_binding()
    return _loaded
