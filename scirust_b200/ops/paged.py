"""Ops on a paged KV cache whose sequences share pages (csrc/paged_attention_tcgen05.cu): the attention of a batch behind a common
prefix. CPU tensors take the fp32 PyTorch statement of the same arithmetic."""
from __future__ import annotations

import functools
import math

import torch

from . import _lib
from . import gemm as _g

BF = torch.bfloat16
vp, i32, i64, f32, sz = _lib.vp, _lib.i32, _lib.i64, _lib.f32, _lib.sz
_lib.register("sb_shared_prefix_attention", [vp, i64, vp, i32, vp, i32, i32, vp, vp, i32, vp, i32, i32, i32, i32, i32, i64, f32, vp, sz,
                                             vp, i64, i32, vp, vp])

TILE_ROWS, BLOCK = 128, 128          # rows of a tile, positions of a block of keys


def shared_prefix_attention_ref(q, pool, block_table, page, seq_len, prefix_table, prefix_len, H, Hkv, dh, scale=None, cu_q=None):
    """fp32 statement, one sequence at a time; rows of no sequence and rows that see nothing are zero."""
    scale = 1.0 / math.sqrt(dh) if scale is None else scale
    G, n = H // Hkv, q.shape[0]
    whole = int(prefix_len) // page if prefix_table is not None else 0
    out = torch.zeros((n, H * dh), dtype=torch.float32, device=q.device)
    ends = list(range(seq_len.numel() + 1)) if cu_q is None else cu_q.tolist()
    for b, length in enumerate(seq_len.tolist()):
        t0, t1 = ends[b], ends[b + 1]
        if t1 <= t0 or length <= 0:
            continue
        blocks = block_table[b, :(length + page - 1) // page].long().clone()
        m = min(whole, blocks.numel())
        if m:
            blocks[:m] = prefix_table[:m].long()
        kv = pool[blocks].float()                                                     # [pages, 2, Hkv, page, dh]
        k, v = kv.permute(1, 2, 0, 3, 4).reshape(2, Hkv, -1, dh)[:, :, :length]
        qb = q[t0:t1, :H * dh].float().reshape(t1 - t0, Hkv, G, dh)
        limit = torch.arange(length - (t1 - t0) + 1, length + 1, device=q.device)     # positions that each row sees
        s = torch.einsum("tkgd,kjd->tkgj", qb, k) * scale
        hidden = torch.arange(length, device=q.device) >= limit[:, None]
        s = s.masked_fill(hidden[:, None, None], float("-inf"))
        p = torch.nan_to_num(torch.softmax(s, -1), nan=0.0) if int(limit[0]) <= 0 else torch.softmax(s, -1)
        out[t0:t1] = torch.einsum("tkgj,kjd->tkgd", p, v).reshape(t1 - t0, H * dh)
    return out


_ws: dict = {}


def _workspace(n, device, stream):
    """``(buffer, its bytes)`` of at least ``n`` bytes. Calls on one stream follow one another and share one; what is being captured into
    a graph gets its own from the graph's pool, since graphs captured on one stream may be replayed at once on two."""
    if _lib.DEBUG_POISON or torch._C._cuda_isCurrentStreamCapturing():
        return _lib.empty(n, torch.uint8, device), n
    key = (device.index, stream)
    w = _ws.get(key)
    if w is None or w[1] < n:
        w = _ws[key] = (torch.empty(n, dtype=torch.uint8, device=device), n)
    return w


@functools.lru_cache(maxsize=4096)       # a function of the device and the sizes
def _workspace_bytes(device, NT, B, H, Hkv, dh, ragged, prefix):
    fn = _lib.cuda().sb_shared_prefix_attention_bytes
    fn.argtypes, fn.restype = [i32] * 7, sz
    return fn(NT, B, H, Hkv, dh, int(ragged), prefix)


def shared_prefix_attention(q, pool, block_table, page, seq_len, prefix_table, prefix_len, H, Hkv, dh, scale=None, cu_q=None,
                            max_len=None, out=None):
    """GQA attention of a batch over its paged KV, where all sequences begin with the same ``prefix_len`` positions: the pages that
    they share are read, multiplied and softmaxed once for all rows, what is behind them sequence by sequence.

    ``q`` [n, >= H*dh] bf16 holds the query heads (position already rotated in) of the new tokens, whose keys and values are in
    ``pool`` [n_blocks, 2, Hkv, page, dh] already. Without ``cu_q`` each sequence has one row, with it (int32 [B + 1], on the device)
    sequence b has rows cu_q[b] .. cu_q[b + 1] - 1, its last positions in ascending order; a row sees the positions up to its own.
    ``block_table`` [B, *] holds all pages of each sequence and ``prefix_table`` those of the prefix, of which whole pages are shared:
    the positions behind the last whole page come from each sequence's own table. ``seq_len`` [B] counts the new tokens; a length of
    zero (an empty slot) gives zeros, and so does a row in front of position 0. ``max_len`` bounds the lengths (default: the table);
    it is for the size of the launch only. Rows of ``out`` that belong to no sequence stay as they are; without ``out`` they are zero.

    Positions that no row of a sequence sees may hold anything, infinities and NaN included. Among the new tokens of one call that
    holds for keys; a value that is not finite reaches the rows in front of it too, as in ``attention_fwd``."""
    scale = 1.0 / math.sqrt(dh) if scale is None else float(scale)
    (n, width), (B,), (rows, max_blocks) = q.shape, seq_len.shape, block_table.shape
    n_blocks, *layout = pool.shape
    prefix = int(prefix_len) // page * page if prefix_table is not None else 0
    if H <= 0 or H % Hkv or page <= 0 or prefix_len < 0 or not scale > 0.0:
        raise ValueError("shared_prefix_attention: heads must divide by kv heads, page and scale be positive")
    if layout != [2, Hkv, page, dh] or rows != B:
        raise ValueError("shared_prefix_attention: pool must be [n_blocks, 2, Hkv, page, dh] and block_table [B, pages]")
    if width < H * dh or (n != B if cu_q is None else cu_q.shape != (B + 1,)):
        raise ValueError("shared_prefix_attention: q must be [rows, >= H*dh], one row a sequence or rows counted by cu_q [B + 1]")
    if prefix and prefix_table.numel() * page < prefix:
        raise ValueError("shared_prefix_attention: prefix_table is shorter than the prefix")
    if out is not None and out.shape != (n, H * dh):
        raise ValueError("shared_prefix_attention: out must be [rows, H*dh]")
    if not q.is_cuda:
        o = shared_prefix_attention_ref(q, pool, block_table, page, seq_len, prefix_table, prefix_len, H, Hkv, dh, scale, cu_q).to(BF)
        if out is None:
            return o
        if cu_q is None:
            out.copy_(o)
        elif n:
            out[int(cu_q[0]):int(cu_q[-1])] = o[int(cu_q[0]):int(cu_q[-1])]
        return out
    device = q.device
    if device.index != _lib.current_device():
        with torch.cuda.device(device):
            return shared_prefix_attention(q, pool, block_table, page, seq_len, prefix_table, prefix_len, H, Hkv, dh, scale, cu_q,
                                           max_len, out)
    if q.dtype is not BF or pool.dtype is not BF or (out is not None and out.dtype is not BF):
        raise ValueError("shared_prefix_attention: q, pool and out must be bf16")
    if (dh != 128 and dh != 64) or H > TILE_ROWS * Hkv or page % 8:
        raise ValueError("shared_prefix_attention: head dimension 64 or 128, up to 128 query heads per kv head, pages of a multiple of 8")
    # a pointer to anything but 32-bit integers on this device would be read as what it is not
    i = torch.int32
    if not (block_table.dtype is i and seq_len.dtype is i and (not prefix or prefix_table.dtype is i) and (cu_q is None or cu_q.dtype is i)
            and block_table.is_contiguous() and seq_len.is_contiguous() and (not prefix or prefix_table.is_contiguous())
            and (cu_q is None or cu_q.is_contiguous())):
        raise ValueError("shared_prefix_attention: tables, lengths and offsets must be contiguous and int32")
    if not (block_table.device == seq_len.device == pool.device == device and (not prefix or prefix_table.device == device)
            and (cu_q is None or cu_q.device == device) and (out is None or out.device == device)):
        raise ValueError("shared_prefix_attention: all tensors must be on the device of q")
    (ldq, unit), q_at = q.stride(), q.data_ptr()
    if unit != 1 or ldq % 8 or q_at % 16 or not pool.is_contiguous():
        raise ValueError("shared_prefix_attention: pool must be contiguous, rows of q contiguous and 16-byte aligned")
    if out is None:
        fill, ldo = 1, H * dh
        out = _lib.empty((n, ldo), BF, device)
    else:
        fill, (ldo, unit) = 0, out.stride()
        if unit != 1 or ldo % 8 or out.data_ptr() % 16:
            raise ValueError("shared_prefix_attention: rows of out must be contiguous and 16-byte aligned")
    if n == 0:
        return out
    if B == 0 or max_blocks == 0:
        return out.zero_() if fill or cu_q is None else out
    per_tile = TILE_ROWS // (H // Hkv)
    if cu_q is not None and n >= B * per_tile:
        prefix = 0                                  # the sequences fill tiles by themselves: nothing to gain from a part in common
    L = max_blocks * page if max_len is None else min(int(max_len), max_blocks * page)
    pairs = B if cu_q is None else B + n // per_tile
    units = Hkv * (-(-n // per_tile) * -(-prefix // BLOCK) + pairs * max(0, -(-(L - prefix) // BLOCK)))
    stream = _lib.stream()
    ws, ws_bytes = _workspace(_workspace_bytes(device.index, n, B, H, Hkv, dh, cu_q is not None, prefix), device, stream)
    _lib.call("sb_shared_prefix_attention", q_at, ldq, pool.data_ptr(), n_blocks, block_table.data_ptr(), max_blocks, page,
              seq_len.data_ptr(), prefix_table.data_ptr() if prefix else None, prefix, cu_q.data_ptr() if cu_q is not None else None,
              B, n, H, Hkv, dh, units, scale, ws.data_ptr(), ws_bytes, out.data_ptr(), ldo, fill,
              _lib.status_word(device).data_ptr(), stream)
    _g.launch_count += 2 if cu_q is None else 3
    return out
