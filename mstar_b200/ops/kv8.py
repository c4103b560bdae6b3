"""The 8-bit key/value cache: rows quantised as they are written, rows read back, and the attention
of single tokens and of prompt portions over its pages.

A cached row (the key or the value of one token and kv head) is held as e4m3 codes and one byte s
that stands for 2^(s - 127), the smallest power of two with which the row's largest number is at
most 448 codes' units (held in [2^-100, 2^119]).  Codes are rounded to nearest even; reading a row
back rounds nothing, in bfloat16 as in float.  A row with a number that is not finite is held as
NaNs (byte 255), and a query that sees its key or value gives NaNs.

The cache of a layer is two tensors: ``kv_cache`` torch.float8_e4m3fn [pages, 2, kv_heads,
page_size, head_dim] and ``kv_scales`` torch.uint8 [pages, 2, kv_heads, page_size].  Block tables
and index arrays are those of the other paged kernels; a token writes nothing where its table has
no page.  Tensors must lie on the current device; launches go to its current stream.

The reference's caches hold the compute type only (mstar/engine/kv_cache_engine.py:132-136).
"""
from __future__ import annotations

import functools
from struct import Struct

import torch

from . import _DT, _error_ptr, _need_cuda, _stream, lib, num_sms
from .lib import KernelError, check

KV8_DTYPE = torch.float8_e4m3fn
_INT = torch.int32
_F32, _BF16, _BYTE = torch.float32, torch.bfloat16, torch.uint8
_device = torch._C._cuda_getDevice
_FAR = 2 ** 31 - 1          # distances of rows are 32-bit numbers in the kernels
# the entry points' arguments as one string (csrc/kv8.cuh)
_pack_write = Struct("=22q").pack
_pack_read = Struct("=15q").pack
_pack_float = Struct("=24qd4q").pack
_pack_decode = Struct("=18qd3q").pack
_pack_portions = Struct("=21qd6q").pack


_sm_counts: dict = {}


def _sms(device: int) -> int:
    n = _sm_counts.get(device)
    if n is None:
        n = _sm_counts[device] = num_sms(torch.device("cuda", device))
    return n


def kv8_supported(head_dim: int) -> bool:
    """Whether a head size can be held in 8 bits by these kernels."""
    return head_dim % 8 == 0 and 0 < head_dim <= 256


def _refuse(what: str, why: str) -> None:
    raise KernelError(f"{what}: {why}")


def _check_cache(what, kv_cache, kv_scales, num_kv_heads, page_size, head_dim) -> int:
    """The cache's pages."""
    if kv_cache.dtype is not KV8_DTYPE or kv_scales.dtype is not _BYTE:
        _refuse(what, f"the cache holds {KV8_DTYPE} codes and uint8 scales, got {kv_cache.dtype} and {kv_scales.dtype}")
    shape = kv_cache.shape
    pages = shape[0] if shape else 0
    if pages < 1 or shape != (pages, 2, num_kv_heads, page_size, head_dim):
        _refuse(what, f"the cache's shape {tuple(shape)} is not (pages, 2, {num_kv_heads}, {page_size}, {head_dim})")
    if kv_scales.shape != (pages, 2, num_kv_heads, page_size):
        _refuse(what, f"the scales' shape {tuple(kv_scales.shape)} is not the cache's {tuple(shape[:4])}")
    if not (kv_cache.is_contiguous() and kv_scales.is_contiguous()):
        _refuse(what, "the cache and its scales must be contiguous")
    if not kv8_supported(head_dim):
        _refuse(what, f"head_dim {head_dim} is not a multiple of 8 up to 256")
    return pages


def _check_table(what, block_table, read=False) -> tuple:
    """The distance of its rows and their entries."""
    strides = block_table.stride()
    if block_table.dtype is not _INT or len(strides) != 2 or strides[1] != 1 or strides[0] < 1:
        _refuse(what, "the block table is int32 [entries, pages], its rows without gaps")
    entries, width = block_table.shape
    if strides[0] > _FAR and entries > 1:
        _refuse(what, "the block table's rows lie 2^31 entries apart or more")
    if read and width < 1:
        _refuse(what, "the block table has no pages")
    return strides[0], width


def _check_index(what, t, n) -> None:
    if t.dtype is not _INT or not t.is_contiguous() or t.numel() < n:
        _refuse(what, f"index arrays are contiguous int32 [at least {n}], got {t.dtype} {tuple(t.shape)}")


def _refuse_device(what, *tensors) -> None:
    _need_cuda(*tensors)
    _refuse(what, "its tensors lie on " + ", ".join(sorted({str(t.device) for t in tensors}))
            + f", not all on the current device cuda:{_device()}")


def rope_kv8_write(qkv: torch.Tensor, positions, cache_pos, token_req, block_table, inv_freq, kv_cache: torch.Tensor,
                   kv_scales: torch.Tensor, num_heads: int, num_kv_heads: int, head_dim: int, rotary_dim: int,
                   interleaved: bool, page_size: int) -> torch.Tensor:
    """Rotate queries and keys of ``qkv`` [tokens, (num_heads + 2 num_kv_heads) * head_dim], quantise keys
    and values into their pages, and return the rotated queries [tokens, num_heads * head_dim] in a
    tensor of their own (``qkv`` stays as it is).  ``inv_freq``: float [rotary_dim / 2], or None when
    rotary_dim == 0.  The tokens of a call name different places: of two with the same one, what is
    left is a mixture."""
    what = "rope_kv8_write"
    dtype = _DT.get(qkv.dtype)
    if dtype is None:
        _refuse(what, f"dtype {qkv.dtype} is not supported (float32 and bfloat16 are)")
    shape, strides = qkv.shape, qkv.stride()
    if len(shape) != 2 or shape[1] != (num_heads + 2 * num_kv_heads) * head_dim or strides[1] != 1:
        _refuse(what, f"qkv {tuple(shape)} is not [tokens, ({num_heads} + 2 * {num_kv_heads}) * {head_dim}] "
                      "with rows without gaps")
    if strides[0] > _FAR and shape[0] > 1:
        _refuse(what, "qkv's rows lie 2^31 numbers apart or more")
    if num_heads < 1 or num_kv_heads < 1:
        _refuse(what, "there is at least one query head and one kv head")
    if rotary_dim % 2 or not 0 <= rotary_dim <= head_dim:
        _refuse(what, f"rotary_dim {rotary_dim} is not even and in [0, head_dim={head_dim}]")
    pages = _check_cache(what, kv_cache, kv_scales, num_kv_heads, page_size, head_dim)
    n, freq = shape[0], 0
    table = _check_table(what, block_table)
    _check_index(what, positions, n)
    _check_index(what, cache_pos, n)
    _check_index(what, token_req, n)
    device = qkv.get_device()
    if rotary_dim:
        if (inv_freq is None or inv_freq.dtype is not _F32 or inv_freq.numel() != rotary_dim // 2
                or not inv_freq.is_contiguous()):
            _refuse(what, f"inv_freq is float32 [{rotary_dim // 2}]")
        if inv_freq.get_device() != device:
            _refuse_device(what, qkv, inv_freq)
        freq = inv_freq.data_ptr()
    if device < 0 or not (
            device == positions.get_device() == cache_pos.get_device() == token_req.get_device()
            == block_table.get_device() == kv_cache.get_device() == kv_scales.get_device() == _device()):
        _refuse_device(what, qkv, positions, cache_pos, token_req, block_table, kv_cache, kv_scales)
    q = qkv.new_empty(n, num_heads * head_dim)          # (sizes as numbers: 1.4 us, 1.8 as a tuple)
    if n == 0:
        return q
    check(lib.get("kv8_cache").mstar_rope_kv8_write_packed(_pack_write(
        qkv.data_ptr(), dtype, strides[0], q.data_ptr(), positions.data_ptr(), cache_pos.data_ptr(),
        token_req.data_ptr(), block_table.data_ptr(), *table, freq, kv_cache.data_ptr(), kv_scales.data_ptr(), pages, n,
        num_heads, num_kv_heads, head_dim, rotary_dim, bool(interleaved), page_size, _stream())), what)
    return q


def kv8_read_rows(kv_cache: torch.Tensor, kv_scales: torch.Tensor, block_table, token_req, cache_pos,
                  dtype: torch.dtype) -> torch.Tensor:
    """The cached rows of the given tokens as numbers, [tokens, 2, kv_heads, head_dim] (keys, then values) of
    ``dtype``: exactly what the cache holds.  Token t is place ``cache_pos[t]`` of request
    ``token_req[t]``; a place whose page the table does not have gives zeros."""
    what = "kv8_read_rows"
    out_type = _DT.get(dtype)
    if out_type is None:
        _refuse(what, f"rows are read as float32 or bfloat16, not {dtype}")
    if kv_cache.dim() != 5:
        _refuse(what, f"the cache's shape {tuple(kv_cache.shape)} is not (pages, 2, kv_heads, page_size, head_dim)")
    _, _, heads, page_size, head_dim = kv_cache.shape
    pages = _check_cache(what, kv_cache, kv_scales, heads, page_size, head_dim)
    table, n = _check_table(what, block_table), token_req.numel()
    _check_index(what, token_req, n)
    _check_index(what, cache_pos, n)
    device = kv_cache.get_device()
    if device < 0 or not (
            device == kv_scales.get_device() == block_table.get_device() == token_req.get_device()
            == cache_pos.get_device() == _device()):
        _refuse_device(what, kv_cache, kv_scales, block_table, token_req, cache_pos)
    out = kv_scales.new_empty(n, 2, heads, head_dim, dtype=dtype)
    if n:
        check(lib.get("kv8_cache").mstar_kv8_read_rows_packed(_pack_read(
            kv_cache.data_ptr(), kv_scales.data_ptr(), block_table.data_ptr(), *table, token_req.data_ptr(),
            cache_pos.data_ptr(), out.data_ptr(), out_type, n, heads, head_dim, pages, page_size, _stream())), what)
    return out


def _check_attention(what, q, out, rows, num_heads, num_kv_heads, head_dim, window, keep_first, scale) -> int:
    """The distance of q's rows."""
    width = num_heads * head_dim
    if q.dtype is not _BF16 and q.dtype is not _F32:
        _refuse(what, f"dtype {q.dtype} is not supported (float32 and bfloat16 are)")
    if num_kv_heads < 1 or num_heads < 1 or num_heads % num_kv_heads:
        _refuse(what, f"{num_heads} query heads are no multiple of {num_kv_heads} kv heads")
    shape, strides = q.shape, q.stride()
    if len(shape) != 2 or shape[0] < rows or shape[1] < width or strides[1] != 1:
        _refuse(what, f"q {tuple(shape)} is not [at least {rows}, at least {width}] with rows without gaps")
    if strides[0] > _FAR and shape[0] > 1:
        _refuse(what, "q's rows lie 2^31 numbers apart or more")
    shape = out.shape
    if out.dtype is not q.dtype or len(shape) != 2 or shape[0] < rows or shape[1] != width or not out.is_contiguous():
        _refuse(what, f"out is contiguous {q.dtype} [at least {rows}, {width}], got {out.dtype} {tuple(shape)}")
    if out.data_ptr() % 16:
        _refuse(what, "out does not start on a 16-byte boundary")
    if not (0 <= window < 2 ** 31 and 0 <= keep_first < 2 ** 31):
        _refuse(what, f"window {window} and keep_first {keep_first} are not negative, and fit 31 bits")
    if not 2.0 ** -126 <= scale <= 2.0 ** 126:
        _refuse(what, f"the scale {scale} is not positive, or not in [2^-126, 2^126]")
    return strides[0]


def kv8_splits(blocks: int, max_keys: int, sms: int) -> int:
    """Parts that the keys of ``blocks`` row tiles are cut into: two blocks an SM, parts of at least 128
    keys, at most 64."""
    return max(1, min(64, -(-2 * sms // max(blocks, 1)), -(-max_keys // 128)))


def kv8_mma_splits(blocks: int, max_keys: int, sms: int, few: bool) -> int:
    """The same for the kernel of the 32-bit mode.  64 rows: two blocks an SM, parts of at least 256 keys.
    (256 blocks on 220 keys, 152 on 1,000, 512 on 6,500, heads of 64: 16.4, 42.0, 350 us uncut, 20.6, 39.7, 335 in two
    parts.)  16 rows or fewer: a block's four warps leave a part each; three blocks on two SMs, 64 keys a warp
    at least.  (8 pairs of a token and a kv head on 16,384 keys, 64 on 2,048 and 512 on 1,028, heads of 128: 39, 24 and
    76 us so, 41, 37 and 76 with half as many parts, 51, 28 and 81 with twice as many; heads of 64: 30, 21, 37 so, 29, 23,
    37 and 39, 16, 40.)"""
    if few:
        return 4 * max(1, min(64, -(-3 * sms // (2 * max(blocks, 1))), -(-max_keys // 256)))
    return max(1, min(64, -(-2 * sms // max(blocks, 1)), -(-max_keys // 256)))


def _parts(q, tokens, num_heads, head_dim, splits) -> tuple:
    """(the tensor, addresses of the outputs' and of the statistics' parts)."""
    if splits == 1:
        return None, 0, 0
    rows = tokens * num_heads * splits
    t = q.new_empty(rows * (head_dim + 2), dtype=_F32)
    return t, t.data_ptr(), t.data_ptr() + 4 * rows * head_dim


def _float_attention(what, q, q_stride, out, kv_cache, kv_scales, pages, block_table, table, indptr, kv_len, req, pos,
                     first_entry, count, max_q, max_len, num_heads, num_kv_heads, head_dim, page_size, window, keep_first,
                     scale) -> None:
    """The kernel that takes every shape: portions by (indptr, kv_len), single tokens by (req, pos)."""
    group, sms = num_heads // num_kv_heads, _sms(q.get_device())
    rows = max_q * group
    if head_dim in KV8_DECODE_HEAD_DIMS and kv_cache.data_ptr() % 16 == 0:
        few = rows <= 16
        splits = kv8_mma_splits((1 if few else -(-rows // 64)) * num_kv_heads * count,
                                _most_keys(max_len, max_q if few else min(max_q, 63 // group + 2), window, keep_first),
                                sms, few)
    else:
        splits = kv8_splits((1 if rows <= 8 else -(-rows // 64)) * num_kv_heads * count,
                            _most_keys(max_len, max_q, window, keep_first), sms)
    tokens = min(out.shape[0], count * max_q)
    part, part_o, part_ml = _parts(q, tokens, num_heads, head_dim, splits)
    check(lib.get("attention_kv8").mstar_kv8_attention_packed(_pack_float(
        q.data_ptr(), q_stride, out.data_ptr(), _DT[q.dtype], kv_cache.data_ptr(), kv_scales.data_ptr(), pages,
        block_table.data_ptr(), *table, indptr, kv_len, req, pos, first_entry, count, max_q, tokens, num_heads,
        num_kv_heads, head_dim, page_size, window, keep_first, scale, splits, part_o, part_ml, _stream())), what)
    if splits > 1:
        lib.add_launches(1)                     # the kernel that joins the parts


KV8_DECODE_HEAD_DIMS = (64, 128, 256)


@functools.lru_cache(maxsize=4096)
def kv8_decode_shape(pairs: int, max_keys: int, head_dim: int, few: bool, sms: int) -> tuple:
    """(blocks of a cluster, warps of a block) that share the keys of each of ``pairs`` (token, kv head, 8
    query heads; ``few``: 4) in the decode kernel.  All blocks run at once (larger clusters leave SMs free: 5 % of
    them for every block of a cluster beyond two where an SM has one; 16 pairs of heads of 128 and of 256 take 7.9
    and 12.9 us so, 11.1 and 17.6 without), with the smallest share of a pair's keys on the SM that has most; among
    those clusters of two at most where that does, and then as many warps as fit.  Where no shape runs at once:
    single blocks of four.  (2,048 keys, 24 shapes each.  Heads of 128, 3 a kv head: 8, 24, 64, 128, 256, 400, 512
    pairs take 5.9 us with 8 x 8, 7.3 with 4 x 8, 11.5 with 2 x 8, 19.1 with 2 x 6, 28.8 with 1 x 6, 40.2 with 1 x 4,
    51.1 with 1 x 3; the best of all shapes is within 0.1 but for 17.9 (1 x 8) at 128.  8 a kv head, and heads of 64:
    within 0.2, but for 62.4 (1 x 2) against 64.8 at 512 pairs of 128 and 7.6 (4 x 4) against 8.1 at 64 of 64.  Heads
    of 256: within 0.1 while all blocks run at once; 256, 400, 512 pairs take 70.5, 104.8, 137.3 with 1 x 4 where 1 x 3
    or 1 x 2 take 61.3, 90.5, 117.1.)"""
    heads = 4 if few else 8
    # a warp's two tiles of 32 keys and values with their scales; warps that the registers allow an SM
    ring, most = 2 * 64 * (head_dim + 1) + 256, 16 if head_dim == 64 else 12 if few and head_dim == 128 else 8
    tiles = max(1, -(-max_keys // 32))
    best = None
    for blocks in (1, 2, 4, 8):
        if blocks > tiles:
            break
        for warps in ((8, 6, 4, 3) if most == 12 else (8, 4) if head_dim < 256 else (4,)):
            warps = min(warps, -(-tiles // blocks))
            smem = warps * (ring + 128) + (4 * (512 + heads * head_dim) if blocks > 1 else 0) + 1024
            room = min(most // warps, 228 * 1024 // smem)
            if pairs * blocks * max(1.0, 1 + 0.05 * (blocks - 2) / room) > room * sms:
                continue
            key = (-(-pairs * blocks // sms) / blocks, max(blocks, 2), -blocks * warps, blocks)
            if best is None or key < best[0]:
                best = key, (blocks, warps)
    return best[1] if best else (1, min(4, tiles))


KV8_TC_HEAD_DIMS = (64, 128)


def kv8_tc_reaches(rows: int, q_stride: int) -> bool:
    """Whether the tensor-core kernel, which holds a query's place in units of 8 numbers in 32 bits (the last is taken),
    can name all rows."""
    return rows * q_stride < 2 ** 35 - 8


def kv8_tc_splits(blocks: int, max_keys: int, sms: int, one_tile: bool) -> tuple:
    """(parts that the keys of ``blocks`` blocks of row tiles are cut into in the tensor-core kernel, whether a
    block makes two of them): a block an SM, at least two tiles of 128 keys each, at most 64 parts.  With
    one row tile a block takes two key tiles side by side from four tiles on: two portions of 17 tokens on
    20,000 / 10,000 / 5,000 keys took 41.0 / 27.3 / 21.5 us so, and 49.4 / 31.2 / 22.9 one after another; one
    on 5,000 keys (two tiles a block) 20.6 and 19.8."""
    ranges = max(1, min(32, sms // max(blocks, 1), -(-max_keys // 256)))
    pair = one_tile and max_keys >= ranges * 512
    return (2 * ranges if pair else ranges), pair


def _most_keys(max_len, max_q, window, keep_first) -> int:
    """A bound on the keys that a row tile walks."""
    return max(1, min(max_len, window + max_q - 1 + keep_first) if window else max_len)


def paged_decode_attention_kv8(q: torch.Tensor, out: torch.Tensor, kv_cache: torch.Tensor, kv_scales: torch.Tensor,
                               block_table, token_req, cache_pos, tokens: int, num_heads: int, num_kv_heads: int,
                               head_dim: int, page_size: int, window: int, keep_first: int, scale: float,
                               max_len: int) -> None:
    """Attention of ``tokens`` single-query rows (row i of q, out, token_req and cache_pos) over an 8-bit
    cache: the token at place p of its request sees the keys up to p; with ``window`` W > 0 the keys
    p - W + 1 .. p and those below ``keep_first``.  q [tokens, at least num_heads * head_dim], out
    contiguous [tokens, num_heads * head_dim] on a 16-byte boundary, both float32 or bfloat16;
    ``max_len`` bounds the keys of any request (it decides how the work is cut, not what is computed).
    A token at a place below 0 gives zeros."""
    what = "paged_decode_attention_kv8"
    q_stride = _check_attention(what, q, out, tokens, num_heads, num_kv_heads, head_dim, window, keep_first, scale)
    pages = _check_cache(what, kv_cache, kv_scales, num_kv_heads, page_size, head_dim)
    table = _check_table(what, block_table, read=True)
    _check_index(what, token_req, tokens)
    _check_index(what, cache_pos, tokens)
    device = q.get_device()
    if device < 0 or not (
            device == out.get_device() == kv_cache.get_device() == kv_scales.get_device()
            == block_table.get_device() == token_req.get_device() == cache_pos.get_device() == _device()):
        _refuse_device(what, q, out, kv_cache, kv_scales, block_table, token_req, cache_pos)
    if tokens <= 0:
        return
    most = _most_keys(max_len, 1, window, keep_first)
    q_ptr, codes, scales = q.data_ptr(), kv_cache.data_ptr(), kv_scales.data_ptr()
    if (q.dtype is _BF16 and head_dim in KV8_DECODE_HEAD_DIMS and page_size % 8 == 0 and q_stride % 8 == 0
            and (q_ptr | codes) % 16 == 0 and scales % 8 == 0):
        pairs = tokens * num_kv_heads * -(-num_heads // num_kv_heads // 8)
        blocks, warps = kv8_decode_shape(pairs, most, head_dim, num_heads <= 4 * num_kv_heads, _sms(device))
        check(lib.get("attention_kv8_decode").mstar_kv8_decode_packed(_pack_decode(
            q_ptr, q_stride, out.data_ptr(), codes, scales, pages, block_table.data_ptr(), *table, token_req.data_ptr(),
            cache_pos.data_ptr(), tokens, num_heads, num_kv_heads, head_dim, page_size, window, keep_first, scale, blocks,
            warps, _stream())), what)
        return
    _float_attention(what, q, q_stride, out, kv_cache, kv_scales, pages, block_table, table, 0, 0, token_req.data_ptr(),
                     cache_pos.data_ptr(), 0, tokens, 1, max_len, num_heads, num_kv_heads, head_dim, page_size, window,
                     keep_first, scale)


def paged_prefill_attention_kv8(q: torch.Tensor, out: torch.Tensor, kv_cache: torch.Tensor, kv_scales: torch.Tensor,
                                block_table, qo_indptr, kv_len, first_entry: int, entries: int, max_q_len: int,
                                num_heads: int, num_kv_heads: int, head_dim: int, page_size: int, window: int,
                                keep_first: int, scale: float, max_kv_len: int) -> None:
    """Attention of the new tokens of batch entries [first_entry, first_entry + entries) over an 8-bit
    cache; q and out hold all tokens of the step, entry e's are [qo_indptr[e], qo_indptr[e + 1]) and the
    last of its ``kv_len[e]`` keys (the mask is causal and aligned to the end; window and keep_first as in
    ``paged_decode_attention_kv8``).  ``max_q_len`` bounds the new tokens of these entries, ``max_kv_len``
    their keys.  Rows of other entries are left as they are."""
    what = "paged_prefill_attention_kv8"
    q_stride = _check_attention(what, q, out, 0, num_heads, num_kv_heads, head_dim, window, keep_first, scale)
    pages = _check_cache(what, kv_cache, kv_scales, num_kv_heads, page_size, head_dim)
    table, rows = _check_table(what, block_table, read=True), out.shape[0]
    if first_entry < 0 or q.shape[0] < rows:
        _refuse(what, "first_entry is not negative, and q has a row for every row of out")
    last = first_entry + max(entries, 0)
    if block_table.shape[0] < last:
        _refuse(what, f"the block table has {block_table.shape[0]} rows and {last} entries are named")
    _check_index(what, qo_indptr, last + 1)
    _check_index(what, kv_len, last)
    device = q.get_device()
    if device < 0 or not (
            device == out.get_device() == kv_cache.get_device() == kv_scales.get_device()
            == block_table.get_device() == qo_indptr.get_device() == kv_len.get_device() == _device()):
        _refuse_device(what, q, out, kv_cache, kv_scales, block_table, qo_indptr, kv_len)
    if entries <= 0 or max_q_len <= 0 or rows == 0:
        return
    max_q_len = min(max_q_len, rows)
    group = num_heads // num_kv_heads
    most = _most_keys(max_kv_len, max_q_len, window, keep_first)
    q_ptr, out_ptr, codes = q.data_ptr(), out.data_ptr(), kv_cache.data_ptr()
    if (q.dtype is _BF16 and head_dim in KV8_TC_HEAD_DIMS and group <= 128 and q_stride % 8 == 0
            and (q_ptr | codes) % 16 == 0 and kv8_tc_reaches(q.shape[0], q_stride)):
        per_tile = 128 // group
        tiles = -(-max_q_len // (2 * per_tile))
        splits, pair = kv8_tc_splits(tiles * num_kv_heads * entries, most, _sms(device), max_q_len <= per_tile)
        tokens = min(rows, entries * max_q_len)
        part, part_o, part_ml = _parts(q, tokens, num_heads, head_dim, splits)
        check(lib.get("attention_kv8_tc").mstar_kv8_attention_tc_packed(_pack_portions(
            q_ptr, q_stride, out_ptr, codes, kv_scales.data_ptr(), pages, block_table.data_ptr(), *table,
            qo_indptr.data_ptr(), kv_len.data_ptr(), first_entry, entries, max_q_len, tokens, num_heads, num_kv_heads,
            head_dim, page_size, window, keep_first, scale, splits, pair, part_o, part_ml, _error_ptr(q),
            _stream())), what)
        if splits > 1:
            lib.add_launches(1)                 # the kernel that joins the parts
        return
    _float_attention(what, q, q_stride, out, kv_cache, kv_scales, pages, block_table, table, qo_indptr.data_ptr(),
                     kv_len.data_ptr(), 0, 0, first_entry, entries, max_q_len, max_kv_len, num_heads, num_kv_heads,
                     head_dim, page_size, window, keep_first, scale)
