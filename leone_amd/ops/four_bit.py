"""The cache of 4 bits an element: what fills it, what reads it back and what attends it.

A cached key or value vector is kept in blocks of 32 consecutive elements, each a number of the 4-bit floating type e2m1 times
a power of two of the block's own (``csrc/four_bit.h`` says how they are chosen and laid out).  A cache is four byte tensors
(``FourBitPools``); a token and kv head of ``dim`` elements take ``dim + dim / 16`` bytes, key and value together, against
``4 * dim`` in bfloat16.  A block table reaches up to 2^30 tokens.  Queries, masks, block tables and results are those of the attention
over a bfloat16 or float32 cache (``ops.attention_rows`` and its neighbours); a row that sees no key (position -1) gives zeros, a row in
whose sight a place has no page gives NaN.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import (F32, PREFILL_GROUP_TILES, KernelError, _CODES, _code, _dev, _rotation_shape, _stream, call, choose_prefill_splits, compute_units)

# (a tensor on a GPU is there: nothing has to be initialised)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)

BLOCK = 32                   # elements that share a power of two
FOUR_BIT_MAX_DIM = 256
MAX_SHARES = 64


class FourBitPools(NamedTuple):
    """Pages of a cache of 4 bits an element: key codes ``[pages, kv_heads, dim / 32, page_tokens, 16]``, key powers ``[pages, kv_heads,
    page_tokens, dim / 32]``, value codes ``[pages, kv_heads, page_tokens / 4, dim / 8, 4, 4]``, value powers ``[pages, kv_heads,
    page_tokens / 4, dim / 32, 4]``, all uint8.  Any tuple of four such tensors does in its place."""
    k_codes: torch.Tensor
    k_powers: torch.Tensor
    v_codes: torch.Tensor
    v_powers: torch.Tensor


def four_bit_supported(head_dim: int, page_tokens: int) -> bool:
    """Whether a cache of 4 bits an element holds heads of this size in pages of so many tokens."""
    return head_dim % BLOCK == 0 and BLOCK <= head_dim <= FOUR_BIT_MAX_DIM and page_tokens % 8 == 0 and 8 <= page_tokens <= 4096


def four_bit_pools(pages: int, kv_heads: int, head_dim: int, page_tokens: int, device) -> FourBitPools:
    """A cache of zeros."""
    if not four_bit_supported(head_dim, page_tokens):
        raise KernelError(f"a cache of 4 bits an element takes heads of a multiple of {BLOCK} elements up to {FOUR_BIT_MAX_DIM} in pages of a "
                          f"multiple of 8 tokens, not heads of {head_dim} in pages of {page_tokens}")
    shapes = ((pages, kv_heads, head_dim // BLOCK, page_tokens, 16), (pages, kv_heads, page_tokens, head_dim // BLOCK),
              (pages, kv_heads, page_tokens // 4, head_dim // 8, 4, 4), (pages, kv_heads, page_tokens // 4, head_dim // BLOCK, 4))
    return FourBitPools(*(torch.zeros(shape, dtype=torch.uint8, device=device) for shape in shapes))


def four_bit_dims(pools) -> tuple:
    """(pages, kv_heads, page_tokens, head_dim) of a cache of 4 bits an element."""
    try:
        k_codes, k_powers, v_codes, v_powers = pools
        pages, kv_heads, blocks, page_tokens, block_bytes = k_codes.shape
    except (ValueError, AttributeError, TypeError):
        raise KernelError("a cache of 4 bits an element is four tensors: key codes, key powers, value codes, value powers") from None
    dim, runs = blocks * BLOCK, page_tokens // 4
    if (block_bytes != 16 or k_powers.shape != (pages, kv_heads, page_tokens, blocks) or v_codes.shape != (pages, kv_heads, runs, 4 * blocks, 4, 4)
            or v_powers.shape != (pages, kv_heads, runs, blocks, 4) or page_tokens % 8 or not 8 <= page_tokens <= 4096
            or not BLOCK <= dim <= FOUR_BIT_MAX_DIM):
        raise KernelError(f"pools of shapes {tuple(tuple(p.shape) for p in pools)} are no cache of 4 bits an element")
    return pages, kv_heads, page_tokens, dim


# A call's time on the host counts where a step is issued kernel by kernel (and is what a short one waits for), so the checks below
# ask each tensor once and put their messages together only when something is refused.
def _current(what: str, t: torch.Tensor) -> int:
    """The current device, which the tensors have to be on: a launch goes to its stream."""
    device = t.get_device()
    if device < 0:
        raise KernelError(f"{what}: tensor is on {t.device}; the kernels run on the GPU only")
    if device != _current_device():
        raise KernelError(f"{what}: tensors on {t.device}, which is not the current device")
    return device


def _at(what: str, name: str, t: torch.Tensor, device: int, dtype: torch.dtype, shape: tuple) -> int:
    """The address of an operand that is as it has to be."""
    if t is None:
        raise KernelError(f"{what}: {name} is needed")
    if t.dtype is dtype and t.shape == shape and t.get_device() == device and t.is_contiguous():
        return t.data_ptr()
    _dev(t, f"{what}: {name}", dtype, shape)
    raise KernelError(f"{what}: {name} is on {t.device}, the others on cuda:{device}; one device is needed")


def _pair_at(what: str, name: str, a: Optional[torch.Tensor], b: Optional[torch.Tensor], device: int, dtype: Optional[torch.dtype],
             shape: Optional[tuple]) -> tuple:
    """The addresses of two operands that come together or not at all, of one type and shape (None: the first one's)."""
    if a is None or b is None:
        if a is not b:
            raise KernelError(f"{what}: one {name} of two")
        return 0, 0
    dtype, shape = dtype or a.dtype, shape or a.shape
    if (a.dtype is b.dtype is dtype and a.shape == shape and b.shape == shape and a.get_device() == b.get_device() == device and a.is_contiguous()
            and b.is_contiguous()):
        return a.data_ptr(), b.data_ptr()
    return _at(what, f"first {name}", a, device, dtype, shape), _at(what, f"second {name}", b, device, dtype, shape)


def _pools_at(what: str, pools, device: int) -> tuple:
    """Addresses and pages of pools whose shapes ``four_bit_dims`` has seen."""
    kc, kp, vc, vp = pools
    if (kc.dtype is kp.dtype is vc.dtype is vp.dtype is torch.uint8 and kc.get_device() == kp.get_device() == vc.get_device() == vp.get_device() == device
            and kc.is_contiguous() and kp.is_contiguous() and vc.is_contiguous() and vp.is_contiguous()):
        return kc.data_ptr(), kp.data_ptr(), vc.data_ptr(), vp.data_ptr(), len(kc)
    return tuple(_at(what, name, p, device, torch.uint8, p.shape) for p, name in zip(pools, FourBitPools._fields)) + (len(kc),)


def _rows_at(what: str, device: int, rows: int, positions: torch.Tensor, row_entry: torch.Tensor, block_table: torch.Tensor) -> tuple:
    if positions is None or row_entry is None or block_table is None:
        raise KernelError(f"{what}: positions, a row map and a block table are needed")
    int32, wanted = torch.int32, (rows,)
    if (positions.dtype is row_entry.dtype is block_table.dtype is int32 and positions.shape == wanted and row_entry.shape == wanted
            and positions.get_device() == row_entry.get_device() == block_table.get_device() == device and block_table.dim() == 2
            and positions.is_contiguous() and row_entry.is_contiguous() and block_table.is_contiguous()):
        return positions.data_ptr(), row_entry.data_ptr(), block_table.data_ptr(), block_table.shape[1], block_table.shape[0]
    if block_table.dim() != 2:
        raise KernelError(f"{what}: a block table is int32 [entries, blocks]")
    return (_at(what, "positions", positions, device, int32, wanted), _at(what, "row map", row_entry, device, int32, wanted),
            _at(what, "block table", block_table, device, int32, block_table.shape), block_table.shape[1], block_table.shape[0])


def qk_norm_rope_write_4bit(qkv: torch.Tensor, q_heads: int, kv_heads: int, head_dim: int, q_gain: Optional[torch.Tensor],
                            k_gain: Optional[torch.Tensor], eps: float, cos: Optional[torch.Tensor], sin: Optional[torch.Tensor],
                            positions: torch.Tensor, row_entry: torch.Tensor, block_table: torch.Tensor, pools,
                            write_cache: bool = True, out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
                            pairing: str = "half_split") -> torch.Tensor:
    """``qk_norm_rope_write`` for a cache of 4 bits an element: splits the fused projection, normalises and rotates q and k heads, writes
    k and v into the cache and returns q.  ``qkv`` is ``[rows, width]`` of q's type, or float32 (also as planes ``[p, rows, width]``
    whose sum is meant) with ``out_dtype`` naming the type of q.  Queries are rounded once, to that type; keys are computed in 64
    bits up to their codes.  Rows at a position below 0, and rows whose place has no page, write nothing; without ``write_cache`` (a run
    that reads what another one of the layer's wrote) none does.  Of two rows at one place either may be kept, or parts of both."""
    what = "qk_norm_rope_write_4bit"
    planes = qkv.shape[0] if qkv.dim() == 3 else 1
    if qkv.dim() not in (2, 3) or qkv.shape[-1] != (q_heads + 2 * kv_heads) * head_dim or planes < 1:
        raise KernelError(f"{what}: a projection {tuple(qkv.shape)} is not ({q_heads}+2*{kv_heads})*{head_dim} wide")
    rows, width = qkv.shape[-2:]
    kind = out_dtype or qkv.dtype
    if kind not in _CODES or (qkv.dtype != kind and qkv.dtype != torch.float32):
        raise KernelError(f"{what}: input {qkv.dtype} for outputs of {kind}")
    pages, pool_heads, page_tokens, pool_dim = four_bit_dims(pools)
    if (pool_heads, pool_dim) != (kv_heads, head_dim):
        raise KernelError(f"{what}: a cache of {pool_heads} heads of {pool_dim} does not fit {kv_heads} heads of {head_dim}")
    table_positions, rotary_dim, pairing_code = _rotation_shape(what, head_dim, cos, sin, pairing)
    if (q_gain is None) != (k_gain is None) or (q_gain is not None and k_gain.dtype != q_gain.dtype):
        raise KernelError(f"{what}: q and k gains must come together in one type")
    device = _current(what, qkv)
    if out is None:
        out = qkv.new_empty((rows, q_heads * head_dim), dtype=kind)
        out_at = out.data_ptr()
    else:
        out_at = _at(what, "q out", out, device, kind, (rows, q_heads * head_dim))
    args = (_at(what, "qkv", qkv, device, qkv.dtype, qkv.shape), _CODES[qkv.dtype], planes, rows * width, width,
            out_at, _CODES[kind], *_pools_at(what, pools, device),
            *_pair_at(what, "gain", q_gain, k_gain, device, None, (head_dim,)), F32 if q_gain is None else _code(q_gain, "qk_norm_rope_write_4bit: gain"),
            eps, *_pair_at(what, "table", cos, sin, device, torch.float32, None), table_positions, rotary_dim, pairing_code, *_rows_at(what, device, rows, positions, row_entry, block_table), rows, q_heads, kv_heads,
            head_dim, page_tokens, 1 if write_cache else 0)
    if rows:
        call("leone_four_bit_fill", *args, _stream(device))
    return out


def cache_rows_4bit(pools, positions: torch.Tensor, row_entry: torch.Tensor, block_table: torch.Tensor) -> tuple:
    """The keys and values that a cache of 4 bits an element holds at the rows' positions, bfloat16 ``[rows, kv_heads * dim]`` each (a code
    times its power is a bfloat16 as it is, or from 2^128 on an infinity).  Rows without a page give NaN."""
    what = "cache_rows_4bit"
    pages, kv_heads, page_tokens, dim = four_bit_dims(pools)
    if positions is None:
        raise KernelError(f"{what}: positions are needed")
    device = _current(what, positions)
    rows = positions.shape[0]
    k = positions.new_empty((rows, kv_heads * dim), dtype=torch.bfloat16)
    v = torch.empty_like(k)
    args = (*_pools_at(what, pools, device), *_rows_at(what, device, rows, positions, row_entry, block_table), k.data_ptr(), v.data_ptr(), rows,
            kv_heads, dim, page_tokens)
    if rows:
        call("leone_four_bit_rows", *args, _stream(device))
    return k, v


def _attention_shape(what: str, q: torch.Tensor, pools, block_table: torch.Tensor, q_heads: int, window: int) -> tuple:
    pages, kv_heads, page_tokens, dim = four_bit_dims(pools)
    if block_table is None or block_table.dim() != 2:
        raise KernelError(f"{what}: a block table is int32 [entries, blocks]")
    if q.dim() != 2 or q.shape[1] != q_heads * dim or q_heads <= 0 or q_heads % kv_heads:
        raise KernelError(f"{what}: queries {tuple(q.shape)} are not {q_heads} heads of {dim} over {kv_heads} kv heads")
    if window < 0:
        raise KernelError(f"{what}: window {window} must not be negative")
    return kv_heads, page_tokens, dim


def _out_at(what: str, q: torch.Tensor, out: Optional[torch.Tensor], device: int) -> tuple:
    """(the results' tensor, its address); what is made here need not be asked."""
    if out is None:
        out = torch.empty_like(q)
        return out, out.data_ptr()
    return out, _at(what, "out", out, device, q.dtype, q.shape)


def _shares_at(rows: int, q_heads: int, dim: int, splits: int, device) -> tuple:
    """(a tensor to hold on to, partial results of rows whose keys are shared out, their maxima and sums)."""
    if splits == 1:
        return None, 0, 0
    if not 1 <= splits <= MAX_SHARES:
        raise KernelError(f"a row's keys are cut into 1 to {MAX_SHARES} parts, not {splits}")
    shares = rows * q_heads * splits
    held = torch.empty(shares * (dim + 2), dtype=torch.float32, device=device)
    at = held.data_ptr()
    return held, at, at + 4 * shares * dim


def four_bit_row_splits(blocks: int, keys: int, units: int = 256) -> int:
    """How many workgroups share a row's keys in ``attention_rows_4bit``, where ``blocks`` workgroups would have them all: four
    workgroups for each of the chip's units, as many as fit one, but no more than give each of their four waves 64 keys.  us, by splits: 64
    blocks of 8,176 keys 261 (1), 77 (4), 48 (8), 39 (16), 41 (32); 8 of them 63 (4), 24 (16), 19 (32); 256 of 2,000 74 (1), 37 (4), 38 (8),
    56 (16); 512 of 4,000 169 (1), 116 (2), 111 (4), 206 (32); 16 of 501 to 777 21 (3: some waves have two tiles), 14.1 (4), 14.4 (16)."""
    return max(1, min(4 * units // max(1, blocks), -(-keys // 256), MAX_SHARES))


def attention_rows_4bit(q: torch.Tensor, pools, positions: torch.Tensor, row_entry: torch.Tensor, block_table: torch.Tensor, q_heads: int,
                        scale: float, window: int = 0, max_context: int = 0, splits: Optional[int] = None,
                        out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``attention_rows`` over a cache of 4 bits an element: any head size the cache holds, bfloat16 or float32 queries, all arithmetic in
    float.  Each row attends its request's cached keys up to its own position (the last ``window`` of them).  ``max_context`` (0: what
    the block table reaches) only steers into how many parts a row's keys are cut.  So does the number of rows: the last bits of a row's
    result may differ with the rows beside it (a given ``splits`` keeps them)."""
    what = "attention_rows_4bit"
    kv_heads, page_tokens, dim = _attention_shape(what, q, pools, block_table, q_heads, window)
    rows = q.shape[0]
    if splits is None:
        keys = max_context or block_table.shape[1] * page_tokens
        keys = min(keys, window) if window else keys
        splits = four_bit_row_splits(rows * kv_heads * (-(-(q_heads // kv_heads) // 4)), keys, compute_units(q.device))
    device = _current(what, q)
    out, out_at = _out_at(what, q, out, device)
    held, part_acc, part_ml = _shares_at(rows, q_heads, dim, splits, q.device)
    args = (_at(what, "q", q, device, q.dtype, q.shape), out_at, _code(q, what),
            *_pools_at(what, pools, device), *_rows_at(what, device, rows, positions, row_entry, block_table), rows, q_heads, kv_heads, dim, page_tokens,
            scale, window, splits, part_acc, part_ml)
    if rows:
        call("leone_four_bit_attend_rows", *args, _stream(device))
    return out


def four_bit_decode_supported(dtype: torch.dtype, head_dim: int, page_tokens: int) -> bool:
    """Whether ``attention_decode_4bit`` takes this case; otherwise ``attention_rows_4bit`` does."""
    return (dtype == torch.bfloat16 and head_dim in (64, 128, 256) and four_bit_supported(head_dim, page_tokens)
            and page_tokens >= 16 and page_tokens & (page_tokens - 1) == 0)


def four_bit_decode_splits(blocks: int, keys: int, units: int = 256) -> int:
    """How many workgroups share a row's keys in ``attention_decode_4bit``, where ``blocks`` workgroups would have them all: two workgroups
    for each of the chip's units, but at least 256 keys each (two tiles for each of its waves) and at most 32 to a row, whose partial
    results the second launch reads.  us, 128 elements a head, by splits: 64 blocks of 8,192 keys 41.5 (1), 18.2 (4), 17.0 (8), 18.8 (12);
    8 of 32,768 25.5 (8), 17.6 (16), 14.4 (32), 16.5 (64); 512 of 300 to 8,191 72.8 (1), 82.7 (2), 77.2 (4)."""
    return max(1, min(2 * units // max(1, blocks), keys // 256, 32))


def attention_decode_4bit(q: torch.Tensor, pools, positions: torch.Tensor, row_entry: torch.Tensor, block_table: torch.Tensor, q_heads: int,
                          scale: float, window: int = 0, max_context: int = 0, splits: Optional[int] = None,
                          out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``attention_decode`` over a cache of 4 bits an element: split-KV attention of single rows on the matrix cores, bfloat16
    (``four_bit_decode_supported``).  ``max_context`` (0: what the block table reaches) only steers the number of splits.  A score is off by
    less than 2^-10 of the largest product in each eight neighbouring elements, and weights are rounded to bfloat16."""
    what = "attention_decode_4bit"
    kv_heads, page_tokens, dim = _attention_shape(what, q, pools, block_table, q_heads, window)
    if not four_bit_decode_supported(q.dtype, dim, page_tokens):
        raise KernelError(f"{what}: {q.dtype} heads of {dim} in pages of {page_tokens} tokens (attention_rows_4bit takes those)")
    rows, group = q.shape[0], q_heads // kv_heads
    if splits is None:
        keys = max_context or block_table.shape[1] * page_tokens
        splits = four_bit_decode_splits(rows * kv_heads * -(-group // (16 if dim <= 128 else 8)), min(keys, window) if window else keys,
                                        compute_units(q.device))
    device = _current(what, q)
    out, out_at = _out_at(what, q, out, device)
    held, part_acc, part_ml = _shares_at(rows, q_heads, dim, splits, q.device)
    args = (_at(what, "q", q, device, q.dtype, q.shape), out_at, *_pools_at(what, pools, device),
            *_rows_at(what, device, rows, positions, row_entry, block_table), rows, q_heads, kv_heads, dim, page_tokens, scale, window, splits,
            part_acc, part_ml)
    if rows:
        call("leone_four_bit_decode", *args, _stream(device))
    return out


def four_bit_prefill_supported(dtype: torch.dtype, head_dim: int, page_tokens: int) -> bool:
    """Whether ``attention_prefill_4bit`` takes this case; otherwise the portion's rows go through the kernels for single rows."""
    return head_dim <= 128 and four_bit_decode_supported(dtype, head_dim, page_tokens)


def attention_prefill_4bit(q: torch.Tensor, out: torch.Tensor, pools, positions: torch.Tensor, tiles: torch.Tensor, block_table: torch.Tensor,
                           q_heads: int, scale: float, window: int = 0, mean_keys: int = 1, splits: Optional[int] = None,
                           covered_rows: Optional[int] = None) -> torch.Tensor:
    """``attention_prefill`` over a cache of 4 bits an element (``four_bit_prefill_supported``): attention for the rows that ``tiles``
    covers, into ``out``; other rows of ``out``, and rows from ``covered_rows`` on, are left as they are.  ``tiles``, ``mean_keys`` and
    ``covered_rows`` as there; precision as ``attention_decode_4bit``.  A key in sight of a group of tiles whose place has no page makes the group's rows NaN.
    The keys are cut into ranges by the bfloat16 kernel's rule (``choose_prefill_splits``), which holds here too: the best of 1 to 32 in nine
    of twelve shapes of 64 to 2,048 rows behind 0 to 30,720, 2 us off it in two, 8 % in one."""
    what = "attention_prefill_4bit"
    kv_heads, page_tokens, dim = _attention_shape(what, q, pools, block_table, q_heads, window)
    if not four_bit_prefill_supported(q.dtype, dim, page_tokens):
        raise KernelError(f"{what}: {q.dtype} heads of {dim} in pages of {page_tokens} tokens (attention_decode_4bit and attention_rows_4bit take those)")
    if tiles is None or tiles.dim() != 2 or tiles.shape[1] != 3 or tiles.shape[0] % PREFILL_GROUP_TILES:
        raise KernelError(f"{what}: tiles must be int32 [n, 3] with n a multiple of {PREFILL_GROUP_TILES}")
    rows, groups = q.shape[0], tiles.shape[0] // PREFILL_GROUP_TILES
    if splits is None:
        splits = choose_prefill_splits(groups, q_heads, mean_keys, window, compute_units(q.device))
    covered = rows if covered_rows is None else covered_rows
    if not 0 <= covered <= rows:
        raise KernelError(f"{what}: {covered} covered rows of {rows}")
    device = _current(what, q)
    held, part_acc, part_ml = _shares_at(covered, q_heads, dim, splits, q.device)
    args = (_at(what, "q", q, device, q.dtype, q.shape), _at(what, "out", out, device, q.dtype, q.shape), *_pools_at(what, pools, device),
            _at(what, "positions", positions, device, torch.int32, (rows,)), _at(what, "tiles", tiles, device, torch.int32, tiles.shape), groups, covered,
            _at(what, "block table", block_table, device, torch.int32, block_table.shape), block_table.shape[1], block_table.shape[0], q_heads,
            kv_heads, dim, page_tokens, scale, window, splits, part_acc, part_ml)
    if groups and covered:
        call("leone_four_bit_prefill", *args, _stream(device))
    return out
