"""Paged KV cache in 8 bits (csrc/quantized_kv.cu, csrc/quantized_kv_attention.cu): keys and values quantised as they are written, attention
of single tokens over the codes, and pages read back in bf16. CPU tensors take the PyTorch statement of the same arithmetic.

A pool is codes ``[n_blocks, 2, Hkv, page, dh]`` (int8 or float8_e4m3fn; keys, then values) with scales ``[n_blocks, 2, Hkv, page / block]``
(fp32): ``block`` consecutive positions of a head share one scale, and a value is code * scale. What is written gets the smallest power of
two that the block's largest magnitude needs: 2^(k-6) for int8 where that lies in [2^k, 2^(k+1)), for e4m3 the least with 448 * scale no
smaller (k is at least -90). A block that holds positions already keeps the larger of its scale and the new one, and what it holds is
rounded to the new steps; a code stays within one step of its value, e4m3 loses nothing that way but below its smallest normal value. A block that
is given an infinity or a NaN (e4m3: or what rounds to an infinity) reads as NaN until its first position is written again."""
from __future__ import annotations

import ctypes as C
import functools
import math
import threading
from typing import NamedTuple

import torch

from . import _lib
from . import gemm as _g

BF = torch.bfloat16
vp, i32, i64, f32 = _lib.vp, _lib.i32, _lib.i64, _lib.f32
_lib.register("sb_quant_kv_append", [vp, i64, i32, i32, i32, i32, vp, vp, i32, vp, i32, vp, i32, i32, i32, vp, i32, vp, vp, i32, i32, vp])
_lib.register("sb_quant_kv_read", [vp, i32, vp, i32, i32, i32, i32, i32, vp, i32, vp, vp])
_lib.register("sb_quant_kv_attention", [vp, i64, vp, i32, vp, i32, i32, i32, vp, i32, vp, i32, i32, i32, i32, i64, f32, vp, vp, vp, i64, vp, vp])
_lib.register("sb_stream_capture_id", [vp, vp])

CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
LARGEST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
BLOCKS = (8, 16, 32, 64)


class QuantPool(NamedTuple):
    """Codes and scales of a cache's pages; every function here takes one, or a pair of the two tensors."""
    codes: torch.Tensor
    scales: torch.Tensor

    @classmethod
    def zeros(cls, n_blocks, Hkv, page, dh, codes="int8", block=None, device="cuda"):
        """A pool of empty pages. ``block`` (8, 16, 32 or 64, dividing the page; default: 16, or the whole of a smaller page): in a
        smaller one a token of large keys or values makes the steps of fewer others coarse, for 4 bytes of scale per block * dh codes."""
        block = min(page, 16) if block is None else block
        if codes not in CODES:
            raise ValueError(f"QuantPool: codes must be one of {', '.join(CODES)}")
        if block not in BLOCKS or page % block:
            raise ValueError("QuantPool: a block of 8, 16, 32 or 64 positions that divides the page")
        return cls(torch.zeros((n_blocks, 2, Hkv, page, dh), dtype=torch.int8, device=device).view(CODES[codes]),
                   torch.zeros((n_blocks, 2, Hkv, page // block), dtype=torch.float32, device=device))

    @property
    def block(self) -> int:
        return self.codes.shape[3] // self.scales.shape[3]

    def nbytes(self) -> int:
        return self.codes.numel() + 4 * self.scales.numel()


def _layout(what, pool, Hkv=None, dh=None):
    """(codes, scales, n_blocks, Hkv, page, dh, block) of a pool, or ValueError."""
    codes, scales = pool
    if codes.dim() != 5 or scales.dim() != 4:
        raise ValueError(f"{what}: pool must be codes [n_blocks, 2, Hkv, page, dh] and scales [n_blocks, 2, Hkv, page / block]")
    n_blocks, two, heads, page, width = codes.shape
    sn, s2, sh, per_page = scales.shape
    if two != 2 or s2 != 2 or sn != n_blocks or sh != heads or (Hkv is not None and (heads != Hkv or width != dh)):
        raise ValueError(f"{what}: pool must be codes [n_blocks, 2, Hkv, page, dh] and scales [n_blocks, 2, Hkv, page / block]")
    block = page // per_page if per_page else 0
    if block not in BLOCKS or block * per_page != page:
        raise ValueError(f"{what}: a scale for each 8, 16, 32 or 64 positions, which divide the page")
    if codes.dtype not in LARGEST or scales.dtype is not torch.float32:
        raise ValueError(f"{what}: codes must be int8 or float8_e4m3fn, scales fp32")
    if codes.device != scales.device:
        raise ValueError(f"{what}: codes and scales must be on one device")
    return codes, scales, n_blocks, heads, page, width, block


def _on_device(what, device, codes, scales, dh, tensors):
    """What the kernels ask of a pool and of the int32 tensors beside it, whose addresses they are given."""
    if dh != 64 and dh != 128:
        raise ValueError(f"{what}: head dimension 64 or 128")
    if not codes.is_contiguous() or not scales.is_contiguous() or codes.data_ptr() % 16:
        raise ValueError(f"{what}: codes and scales must be contiguous, codes 16-byte aligned")
    if codes.get_device() != device.index:
        raise ValueError(f"{what}: all tensors must be on one device")
    for t in tensors:
        if t is not None and (t.dtype is not torch.int32 or not t.is_contiguous() or t.get_device() != device.index):
            raise ValueError(f"{what}: tables, lengths, offsets and page ids must be contiguous, int32 and on the pool's device")


def _batch(what, n, seq_len, block_table, cu_q):
    if seq_len.dim() != 1 or block_table.dim() != 2 or block_table.shape[0] != seq_len.shape[0]:
        raise ValueError(f"{what}: seq_len [B] and block_table [B, pages]")
    B = seq_len.shape[0]
    if B and not block_table.shape[1]:
        raise ValueError(f"{what}: block_table has no pages")
    if n != B if cu_q is None else tuple(cu_q.shape) != (B + 1,):
        raise ValueError(f"{what}: one row a sequence, or rows counted by cu_q [B + 1]")
    return B, block_table.shape[1]


# ---------------------------------------------------------------------------------------------------------------- writing
def scale_for(largest: torch.Tensor, dtype) -> torch.Tensor:
    """The scale of a block from its largest magnitude (fp32): the statement of the rule above."""
    k = torch.frexp(largest.clamp_min(2.0 ** -90))[1] - 1
    one = torch.ones_like(largest)
    s = torch.ldexp(one, k - 6) if dtype is torch.int8 else torch.ldexp(one, k - 8 + (largest > torch.ldexp(1.75 * one, k)).int())
    top = math.inf if dtype is torch.int8 else 1.9375 * 2.0 ** 127            # from there on e4m3 rounds to 2^128
    return torch.where(largest < top, s, torch.full_like(s, math.nan))


def to_codes(x: torch.Tensor, dtype) -> torch.Tensor:
    """Values in units of the scale as codes: to nearest, ties to even; NaN becomes 0."""
    x = torch.nan_to_num(x, nan=0.0, posinf=math.inf, neginf=-math.inf).clamp(-LARGEST[dtype], LARGEST[dtype])
    return x.round().to(dtype) if dtype is torch.int8 else x.to(dtype)


def _runs(n, seq_len, cu_q):
    """(sequence, first row, position of it, rows) of every sequence with rows; rows in front of position 0 are left out."""
    ends = list(range(n + 1)) if cu_q is None else cu_q.tolist()
    for b, length in enumerate(seq_len.tolist()):
        t0, t1 = ends[b], min(ends[b + 1], n)
        pos = length - (ends[b + 1] - t0)
        skip = max(0, -pos)
        if length > 0 and t0 + skip < t1:
            yield b, t0 + skip, pos + skip, t1 - t0 - skip


def _append_ref(qkv, H, Hkv, dh, rope, codes, scales, block, block_table, seq_len, cu_q):
    page = codes.shape[3]
    cap = min(block_table.shape[1] * page, rope[0].shape[0] if rope is not None else math.inf)
    for b, t0, pos, rows in _runs(qkv.shape[0], seq_len, cu_q):
        rows = min(rows, cap - pos)
        if rows <= 0:
            continue
        x = qkv[t0:t0 + rows]
        if rope is not None:
            from . import basic
            basic.rope_(x, H + Hkv, dh, 1, rope[0], rope[1], positions=torch.arange(pos, pos + rows, dtype=torch.int32))
        kv = x[:, H * dh:(H + 2 * Hkv) * dh].float().reshape(rows, 2, Hkv, dh)
        at = 0
        while at < rows:
            p = pos + at
            cnt = min(block - p % block, rows - at)
            part, slot, blk, off = kv[at:at + cnt], p % page, int(block_table[b, p // page]), p % block
            at += cnt
            if not 0 <= blk < codes.shape[0]:
                continue
            old = scales[blk, :, :, slot // block].clone()
            s = scale_for(part.abs().amax((0, 3)), codes.dtype)
            if off:
                s = torch.where((old > s) | old.isnan(), old, s)
                again = to_codes(codes[blk, :, :, slot - off:slot].float() * (old / s)[..., None, None], codes.dtype)
                keep = (s.isnan() | (s == old))[..., None, None]
                bits = codes.view(torch.int8)
                bits[blk, :, :, slot - off:slot] = torch.where(keep, bits[blk, :, :, slot - off:slot], again.view(torch.int8))
            scales[blk, :, :, slot // block] = s
            new = to_codes((part / s[..., None]).where(~s.isnan()[..., None], torch.zeros(())), codes.dtype)
            codes.view(torch.int8)[blk, :, :, slot:slot + cnt] = new.permute(1, 2, 0, 3).view(torch.int8)


def _chunk(n, B, block):
    """Rows that a warp looks for blocks in: the whole of a block of sixteen where sequences are long, one row where they are short, so that
    the blocks of a chunk, which one warp writes one after the other, are few."""
    return 1 if n < 4 * B else 4 if n < 64 * B else 16


def _append(what, qkv, H, Hkv, dh, rope, pool, block_table, seq_len, cu_q):
    codes, scales, n_blocks, _, page, _, block = _layout(what, pool, Hkv, dh)
    if qkv.dim() != 2 or H < 0 or qkv.shape[1] < (H + 2 * Hkv) * dh:
        raise ValueError(f"{what}: qkv must be [rows, >= (H + 2 Hkv) * dh]")
    n = qkv.shape[0]
    B, max_blocks = _batch(what, n, seq_len, block_table, cu_q)
    if qkv.dtype is not BF:
        raise ValueError(f"{what}: qkv must be bf16")
    if rope is not None and (rope[0].shape != rope[1].shape or rope[0].dim() != 2 or rope[0].shape[1] * 2 != dh
                             or rope[0].dtype is not torch.float32 or rope[1].dtype is not torch.float32):
        raise ValueError(f"{what}: the rotation's tables must be fp32 [positions, dh / 2]")
    device = qkv.device
    if device.type != "cuda":
        return _append_ref(qkv, H, Hkv, dh, rope, codes, scales, block, block_table, seq_len, cu_q)
    if device.index != _lib.current_device():
        with torch.cuda.device(device):
            return _append(what, qkv, H, Hkv, dh, rope, pool, block_table, seq_len, cu_q)
    _on_device(what, device, codes, scales, dh, (block_table, seq_len, cu_q))
    (ld, unit), at = qkv.stride(), qkv.data_ptr()
    if n == 1:
        ld = (H + 2 * Hkv) * dh                        # a dimension of one has any stride
    if unit != 1 or ld % 8 or at % 16 or ld < (H + 2 * Hkv) * dh:
        raise ValueError(f"{what}: rows of qkv must be contiguous, apart and 16-byte aligned")
    cos = sin = None
    n_pos = 0
    if rope is not None:
        cos, sin = rope
        if not (cos.is_contiguous() and sin.is_contiguous() and cos.get_device() == sin.get_device() == device.index):
            raise ValueError(f"{what}: the rotation's tables must be contiguous and on the device of qkv")
        n_pos, cos, sin = cos.shape[0], cos.data_ptr(), sin.data_ptr()
    if n == 0 or B == 0 or n_blocks == 0:
        return
    _lib.call("sb_quant_kv_append", at, ld, n, H, Hkv, dh, cos, sin, n_pos, codes.data_ptr(), codes.dtype is not torch.int8, scales.data_ptr(),
              n_blocks, page, block, block_table.data_ptr(), max_blocks, seq_len.data_ptr(), cu_q.data_ptr() if cu_q is not None else None,
              B, _chunk(n, B, block), _lib.stream())
    _g.launch_count += 1


def kv_append(qkv, H, Hkv, dh, pool, block_table, seq_len, cu_q=None):
    """Quantises the key and value heads of ``qkv`` [n, >= (H + 2 Hkv) * dh] (bf16, positions rotated in already) into ``pool``.

    Without ``cu_q`` each sequence has one row, with it (int32 [B + 1]) sequence b has rows cu_q[b] .. cu_q[b + 1] - 1; they are its last
    positions of ``seq_len`` [B], which counts them, in ascending order. ``block_table`` [B, pages] holds the pages of each sequence, of
    which no two may share one that is written. Rows of no sequence, in front of position 0 or behind the table are left out, and so are
    page ids outside the pool. A block whose first position is among the rows is begun anew, whatever it held."""
    _append("kv_append", qkv, H, Hkv, dh, None, pool, block_table, seq_len, cu_q)


def rope_kv_append(qkv, H, Hkv, dh, cos_t, sin_t, pool, block_table, seq_len, cu_q=None):
    """``kv_append`` with the rotation of the query and key heads, in place, in front of it. ``cos_t`` and ``sin_t`` (fp32) are ``[positions,
    dh / 2]``; rows behind their last position, as those that ``kv_append`` leaves out, stay as they are."""
    _append("rope_kv_append", qkv, H, Hkv, dh, (cos_t, sin_t), pool, block_table, seq_len, cu_q)


# ---------------------------------------------------------------------------------------------------------------- reading back
def _values(codes, scales, block):
    return codes.float() * scales.repeat_interleave(block, -1)[..., None]


def read_pages(pool, pages, out=None):
    """The pages ``pages`` (a list, or a vector of ids) of ``pool`` in bf16, ``[n, 2, Hkv, page, dh]``: page i of the answer is page
    ``pages[i]``, so that with ``arange(n)`` as table it is a pool for the attention over bf16 pages. The same page may be asked for more
    than once. Ids on the host are checked; of those on the device (int32) one outside the pool reads as zeros."""
    codes, scales, n_blocks, Hkv, page, dh, block = _layout("read_pages", pool)
    device = codes.device
    if not torch.is_tensor(pages) or (pages.device.type != "cuda" and device.type == "cuda"):
        ids = [int(i) for i in (pages.tolist() if torch.is_tensor(pages) else pages)]
        if any(not 0 <= i < n_blocks for i in ids):
            raise ValueError("read_pages: page outside the pool")
        pages = torch.tensor(ids, dtype=torch.int32, device=device)
    if pages.dim() != 1:
        raise ValueError("read_pages: a vector of page ids")
    shape = (pages.shape[0], 2, Hkv, page, dh)
    if out is not None and (tuple(out.shape) != shape or out.dtype is not BF or not out.is_contiguous() or out.device != device):
        raise ValueError("read_pages: out must be contiguous bf16 [pages, 2, Hkv, page, dh] beside the pool")
    if device.type != "cuda":
        if pages.numel() and not 0 <= int(pages.min()) <= int(pages.max()) < n_blocks:
            raise ValueError("read_pages: page outside the pool")
        got = _values(codes[pages.long()] if codes.dtype is torch.int8 else codes.view(torch.int8)[pages.long()].view(codes.dtype),
                      scales[pages.long()], block).to(BF)
        return got if out is None else out.copy_(got)
    if device.index != _lib.current_device():
        with torch.cuda.device(device):
            return read_pages(pool, pages, out)
    _on_device("read_pages", device, codes, scales, dh, (pages,))
    if out is None:
        out = _lib.empty(shape, BF, device)
    elif out.data_ptr() % 16:
        raise ValueError("read_pages: out must be 16-byte aligned")
    if out.numel() == 0:
        return out
    if n_blocks == 0:
        return out.zero_()
    _lib.call("sb_quant_kv_read", codes.data_ptr(), codes.dtype is not torch.int8, scales.data_ptr(), n_blocks, Hkv, page, block, dh,
              pages.data_ptr(), shape[0], out.data_ptr(), _lib.stream())
    _g.launch_count += 1
    return out


# ---------------------------------------------------------------------------------------------------------------- attention
TILE, JOB_HEADS, LAUNCH_SEQUENCES = 64, 16, 1024          # positions of a tile, query heads of a job, sequences of a launch


class _Workspace:
    """Parts of jobs that are cut, and a counter for each job, which every launch leaves at zero."""
    __slots__ = ("part", "counters", "capture")

    def __init__(self, floats, counters, device, capture):
        self.part = _lib.empty(floats, torch.float32, device)
        self.counters = torch.zeros(counters, dtype=torch.int32, device=device)
        self.capture = capture


_ws: dict = {}
_ws_lock = threading.Lock()


@functools.lru_cache(maxsize=64)
def _part_floats(device_index, dh):
    return _lib.cuda().sb_quant_kv_attention_floats(dh)


def _workspace(device, stream, floats, counters):
    """Launches on one stream follow one another and share one. Those of a graph share one of the graph's memory, whose counters it clears
    itself: graphs captured on one stream may be replayed at once on two."""
    capture = 0
    if torch._C._cuda_isCurrentStreamCapturing():
        word = (C.c_ulonglong * 1)()
        _lib.call("sb_stream_capture_id", stream, word)
        capture = word[0]
    key = (device.index, stream, capture != 0)
    w = _ws.get(key)
    if w is None or w.capture != capture or w.counters.shape[0] < counters or w.part.shape[0] < floats or _lib.DEBUG_POISON:
        with _ws_lock:
            w = _ws.get(key)
            if w is None or w.capture != capture or w.counters.shape[0] < counters or w.part.shape[0] < floats or _lib.DEBUG_POISON:
                w = _ws[key] = _Workspace(floats, max(counters, 4096), device, capture)
    return w


def drop_workspace(device, stream):
    """Gives back what calls on ``stream`` (a handle) work in, some 4 MB, where no more of them are to come."""
    for captured in (False, True):
        _ws.pop((device.index, stream, captured), None)


def decode_attention_ref(q, pool, block_table, seq_len, H, Hkv, dh, scale=None):
    """fp32 statement, one sequence at a time; a sequence of no positions gets zeros."""
    codes, scales, _, _, page, _, block = _layout("decode_attention", pool, Hkv, dh)
    scale = 1.0 / math.sqrt(dh) if scale is None else scale
    out = torch.zeros((q.shape[0], H * dh), dtype=torch.float32, device=q.device)
    for b, length in enumerate(seq_len.tolist()):
        length = min(length, block_table.shape[1] * page)
        if length <= 0:
            continue
        ids = block_table[b, :(length + page - 1) // page].long()
        kv = _values(codes.view(torch.int8)[ids].view(codes.dtype), scales[ids], block)
        k, v = kv.permute(1, 2, 0, 3, 4).reshape(2, Hkv, -1, dh)[:, :, :length]
        s = torch.einsum("hgd,hld->hgl", q[b, :H * dh].float().reshape(Hkv, H // Hkv, dh), k) * scale
        out[b] = torch.einsum("hgl,hld->hgd", torch.softmax(s, -1), v).reshape(-1)
    return out


def decode_attention(q, pool, block_table, seq_len, H, Hkv, dh, scale=None, max_len=None, out=None):
    """GQA attention of one new token of each sequence over its paged KV in 8 bits. ``q`` [B, >= H * dh] bf16 holds the query heads (rotated);
    the token's own key and value are in ``pool`` already and counted by ``seq_len`` [B]. ``max_len`` bounds the lengths (default: the table);
    it is for the size of the launch only. A sequence of no positions (an empty slot) gets zeros. Positions behind a sequence's last one
    may hold any code and any scale. Returns bf16 [B, H * dh], ``out`` if that is given; ``out`` may not lie in what the call reads."""
    codes, scales, n_blocks, _, page, _, block = _layout("decode_attention", pool, Hkv, dh)
    scale = 1.0 / math.sqrt(dh) if scale is None else float(scale)
    if q.dim() != 2 or H <= 0 or H % Hkv or q.shape[1] < H * dh or not scale > 0.0:
        raise ValueError("decode_attention: q must be [B, >= H * dh], heads a multiple of kv heads, scale positive")
    B, max_blocks = _batch("decode_attention", q.shape[0], seq_len, block_table, None)
    if q.dtype is not BF or (out is not None and (out.dtype is not BF or tuple(out.shape) != (B, H * dh))):
        raise ValueError("decode_attention: q must be bf16, out bf16 [B, H * dh]")
    device = q.device
    if device.type != "cuda":
        o = decode_attention_ref(q, pool, block_table, seq_len, H, Hkv, dh, scale).to(BF)
        return o if out is None else out.copy_(o)
    if device.index != _lib.current_device():
        with torch.cuda.device(device):
            return decode_attention(q, pool, block_table, seq_len, H, Hkv, dh, scale, max_len, out)
    _on_device("decode_attention", device, codes, scales, dh, (block_table, seq_len))
    (ldq, unit), q_at = q.stride(), q.data_ptr()
    if B == 1:
        ldq = H * dh
    if unit != 1 or ldq % 8 or ldq < H * dh or q_at % 16:
        raise ValueError("decode_attention: rows of q must be contiguous, apart and 16-byte aligned")
    if out is None:
        out, ldo = _lib.empty((B, H * dh), BF, device), H * dh
    else:
        ldo, unit = out.stride()
        ldo = H * dh if B == 1 else ldo
        if unit != 1 or ldo % 8 or ldo < H * dh or out.data_ptr() % 16 or out.get_device() != device.index:
            raise ValueError("decode_attention: rows of out must be contiguous, apart, 16-byte aligned and on the device of q")
    if B == 0:
        return out
    if n_blocks == 0:
        raise ValueError("decode_attention: the pool has no pages")
    if page not in (8, 16, 32) and page % TILE:
        raise ValueError("decode_attention: pages of 8, 16, 32 or a multiple of 64 positions")
    if n_blocks * 2 * Hkv * page >= (1 << 31) - TILE:
        raise ValueError("decode_attention: more rows of codes than 31 bits count")
    tiles = -(-max_blocks * page // TILE)                       # of a sequence, at most
    jobs = Hkv * -(-(H // Hkv) // JOB_HEADS)
    at_once = min(B, LAUNCH_SEQUENCES, ((1 << 31) - 1) // (tiles * jobs))
    if at_once == 0:
        raise ValueError("decode_attention: a table of more tiles and heads than 31 bits count")
    if max_len is not None:
        tiles = min(tiles, max(1, -(-int(max_len) // TILE)))
    stream = _lib.stream()
    ws = _workspace(device, stream, _part_floats(device.index, dh), at_once * jobs)
    part, counters, status = ws.part.data_ptr(), ws.counters.data_ptr(), _lib.status_word(device).data_ptr()
    codes_at, e4m3, scales_at, table_at, lens_at, o_at = (codes.data_ptr(), codes.dtype is not torch.int8, scales.data_ptr(),
                                                          block_table.data_ptr(), seq_len.data_ptr(), out.data_ptr())
    for b in range(0, B, at_once):
        n = min(at_once, B - b)
        _lib.call("sb_quant_kv_attention", q_at + b * ldq * 2, ldq, codes_at, e4m3, scales_at, n_blocks, page, block,
                  table_at + b * max_blocks * 4, max_blocks, lens_at + b * 4, n, H, Hkv, dh, n * jobs * tiles, scale, part, counters,
                  o_at + b * ldo * 2, ldo, status, stream)
        _g.launch_count += 1
    return out
