"""Paged KV cache in 8 bits (csrc/quantized_kv.cu, csrc/quantized_kv_attention.cu): keys and values quantised as they are written, attention
of single tokens over the codes, and pages read back in bf16. CPU tensors take the PyTorch statement of the same arithmetic.

A pool is codes ``[n_blocks, 2, Hkv, page, dh]`` (int8 or float8_e4m3fn; keys, then values) with scales ``[n_blocks, 2, Hkv, page / block]``
(fp32): ``block`` consecutive positions of a head share one scale, and a value is code * scale. What is written gets the smallest power of
two that the block's largest magnitude needs: 2^(k-6) for int8 where that lies in [2^k, 2^(k+1)), for e4m3 the least with 448 * scale no
smaller (k is at least -90). A block that holds positions already keeps the larger of its scale and the new one, and what it holds is
rounded to the new steps; a code stays within one step of its value, e4m3 loses nothing that way but below its smallest normal value. A
block that is given an infinity or a NaN (e4m3: or what rounds to an infinity) reads as NaN until its first position is written again."""
from __future__ import annotations

import ctypes as C
import functools
import math
import threading
from typing import NamedTuple

import torch

from . import _lib
from . import gemm as _g

BF, F32, I32 = torch.bfloat16, torch.float32, torch.int32
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
    shape, per_block = codes.shape, scales.shape
    if (len(shape) != 5 or len(per_block) != 4 or shape[:3] != per_block[:3] or shape[1] != 2 or shape[2] == 0
            or (Hkv is not None and (shape[2] != Hkv or shape[4] != dh))):
        raise ValueError(f"{what}: pool must be codes [n_blocks, 2, Hkv, page, dh] and scales [n_blocks, 2, Hkv, page / block]")
    n_blocks, _, heads, page, width = shape
    block = page // per_block[3] if per_block[3] else 0
    if block not in BLOCKS or block * per_block[3] != page:
        raise ValueError(f"{what}: a scale for each 8, 16, 32 or 64 positions, which divide the page")
    if codes.dtype not in LARGEST or scales.dtype is not F32:
        raise ValueError(f"{what}: codes must be int8 or float8_e4m3fn, scales fp32")
    if codes.get_device() != scales.get_device():
        raise ValueError(f"{what}: codes and scales must be on one device")
    return codes, scales, n_blocks, heads, page, width, block


def _on_device(what, index, codes, scales, dh, tensors):
    """What the kernels ask of a pool and of the int32 tensors beside it, whose addresses they are given: the codes' address."""
    if dh != 64 and dh != 128:
        raise ValueError(f"{what}: head dimension 64 or 128")
    at = codes.data_ptr()
    if not codes.is_contiguous() or not scales.is_contiguous() or at % 16:
        raise ValueError(f"{what}: codes and scales must be contiguous, codes 16-byte aligned")
    if codes.get_device() != index:
        raise ValueError(f"{what}: all tensors must be on one device")
    for t in tensors:
        if t.dtype is not I32 or t.get_device() != index or not t.is_contiguous():
            raise ValueError(f"{what}: tables, lengths, offsets and page ids must be contiguous, int32 and on the pool's device")
    return at


def _on_host(what, *tensors):
    if any(t is not None and t.get_device() >= 0 for t in tensors):
        raise ValueError(f"{what}: all tensors must be on one device")


def _batch(what, n, seq_len, block_table, cu_q):
    lens, table = seq_len.shape, block_table.shape
    if len(lens) != 1 or len(table) != 2 or table[0] != lens[0]:
        raise ValueError(f"{what}: seq_len [B] and block_table [B, pages]")
    B, max_blocks = table
    if B and not max_blocks:
        raise ValueError(f"{what}: block_table has no pages")
    if n != B if cu_q is None else tuple(cu_q.shape) != (B + 1,):
        raise ValueError(f"{what}: one row a sequence, or rows counted by cu_q [B + 1]")
    return B, max_blocks


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
    """Rows that a warp looks for blocks in: a block's worth where sequences are long (two blocks of 8: 16 sequences of 700 rows take 14.2 us so
    and 15.4 us with one), one row where they are short, so that the blocks of a chunk, which one warp writes one after the other, are few.
    us with 1 / 4 / 16, rotation and all, blocks of 16, 32 / 8 heads of 128. 64 sequences of 1.5 rows in the mean 3.7 / 7.8 / 24.0, 3 3.9 / 5.9
    / 14.8, 4.2 4.3 / 5.6 / 14.7, 6 5.3 / 6.1 / 12.9, 11 8.5 / 8.2 / 12.4, 25 16.0 / 12.1 / 12.6, 49 26.1 / 17.4 / 17.8; 16 of 94 14.6 / 11.6 /
    12.1; 4 of 51 5.7 / 6.3 / 6.5, 107 6.8 / 6.3 / 6.8; one of 16 4.6 / 4.5 / 5.3, 300 5.9 / 5.8 / 6.1. 16 / 4 heads of 64: 64 of 3 3.2 / 4.9 / 12.2,
    6 3.4 / 4.7 / 9.7, 25 7.2 / 5.8 / 7.2, 16 of 94 6.7 / 5.3 / 6.5. Next to its borders, of 4 to 10 rows and of 64 to 110, the rule takes a
    way that is slower by up to 40 % and 25 %."""
    return 1 if n < 4 * B else 4 if n < 64 * B else max(block, 16)


def _append(what, qkv, H, Hkv, dh, rope, pool, block_table, seq_len, cu_q):
    codes, scales, n_blocks, _, page, _, block = _layout(what, pool, Hkv, dh)
    if qkv.dim() != 2 or H < 0 or qkv.shape[1] < (H + 2 * Hkv) * dh:
        raise ValueError(f"{what}: qkv must be [rows, >= (H + 2 Hkv) * dh]")
    n = qkv.shape[0]
    B, max_blocks = _batch(what, n, seq_len, block_table, cu_q)
    if qkv.dtype is not BF:
        raise ValueError(f"{what}: qkv must be bf16")
    if n_blocks == 0:
        raise ValueError(f"{what}: the pool has no pages")
    if rope is not None:
        turns = rope[0].shape
        if len(turns) != 2 or turns[1] * 2 != dh or rope[1].shape != turns or rope[0].dtype is not F32 or rope[1].dtype is not F32:
            raise ValueError(f"{what}: the rotation's tables must be fp32 [positions, dh / 2]")
    index = qkv.get_device()
    if index < 0:
        _on_host(what, codes, block_table, seq_len, cu_q, *(rope or ()))
        return _append_ref(qkv, H, Hkv, dh, rope, codes, scales, block, block_table, seq_len, cu_q)
    if index != _lib.current_device():
        with torch.cuda.device(index):
            return _append(what, qkv, H, Hkv, dh, rope, pool, block_table, seq_len, cu_q)
    codes_at = _on_device(what, index, codes, scales, dh, (block_table, seq_len) if cu_q is None else (block_table, seq_len, cu_q))
    (ld, unit), at = qkv.stride(), qkv.data_ptr()
    if n == 1:
        ld = (H + 2 * Hkv) * dh                        # a dimension of one has any stride
    if unit != 1 or ld % 8 or at % 16 or ld < (H + 2 * Hkv) * dh:
        raise ValueError(f"{what}: rows of qkv must be contiguous, apart and 16-byte aligned")
    cos = sin = None
    n_pos = 0
    if rope is not None:
        cos, sin = rope
        if cos.get_device() != index or sin.get_device() != index or not (cos.is_contiguous() and sin.is_contiguous()):
            raise ValueError(f"{what}: the rotation's tables must be contiguous and on the device of qkv")
        n_pos, cos, sin = cos.shape[0], cos.data_ptr(), sin.data_ptr()
        if (cos | sin) % 16:
            raise ValueError(f"{what}: the rotation's tables must be 16-byte aligned")
    if n == 0 or B == 0 or (rope is not None and n_pos == 0):      # the address of tables without positions is null, as where there is no rotation
        return
    _lib.call("sb_quant_kv_append", at, ld, n, H, Hkv, dh, cos, sin, n_pos, codes_at, codes.dtype is not torch.int8, scales.data_ptr(), n_blocks,
              page, block, block_table.data_ptr(), max_blocks, seq_len.data_ptr(), None if cu_q is None else cu_q.data_ptr(), B,
              _chunk(n, B, block), _lib.stream())
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
    index = codes.get_device()
    if not torch.is_tensor(pages) or (index >= 0 and not pages.is_cuda):
        ids = [int(i) for i in (pages.tolist() if torch.is_tensor(pages) else pages)]
        if any(not 0 <= i < n_blocks for i in ids):
            raise ValueError("read_pages: page outside the pool")
        pages = torch.tensor(ids, dtype=I32, device=codes.device)
    if pages.dim() != 1:
        raise ValueError("read_pages: a vector of page ids")
    shape = (pages.shape[0], 2, Hkv, page, dh)
    if out is not None and (tuple(out.shape) != shape or out.dtype is not BF or not out.is_contiguous() or out.device != codes.device):
        raise ValueError("read_pages: out must be contiguous bf16 [pages, 2, Hkv, page, dh] beside the pool")
    if index < 0:
        if pages.numel() and not 0 <= int(pages.min()) <= int(pages.max()) < n_blocks:
            raise ValueError("read_pages: page outside the pool")
        got = _values(codes.view(torch.int8)[pages.long()].view(codes.dtype), scales[pages.long()], block).to(BF)
        return got if out is None else out.copy_(got)
    if index != _lib.current_device():
        with torch.cuda.device(index):
            return read_pages(pool, pages, out)
    codes_at = _on_device("read_pages", index, codes, scales, dh, (pages,))
    if out is None:
        out = _lib.empty(shape, BF, codes.device) if _lib.DEBUG_POISON else codes.new_empty(shape, dtype=BF)      # cheaper than torch.empty
    out_at = out.data_ptr()
    if out_at % 16:
        raise ValueError("read_pages: out must be 16-byte aligned")
    if shape[0] == 0:
        return out
    if n_blocks == 0:
        return out.zero_()
    _lib.call("sb_quant_kv_read", codes_at, codes.dtype is not torch.int8, scales.data_ptr(), n_blocks, Hkv, page, block, dh, pages.data_ptr(),
              shape[0], out_at, _lib.stream())
    _g.launch_count += 1
    return out


# ---------------------------------------------------------------------------------------------------------------- attention
TILE, JOB_HEADS, LAUNCH_SEQUENCES = 64, 24, 1024          # positions of a tile, query heads of a job, sequences of a launch


class _Workspace:
    """Parts of jobs that are cut, and a counter for each job, which every launch leaves at zero."""
    __slots__ = ("part", "counters", "capture", "floats", "jobs", "part_at", "counters_at")

    def __init__(self, floats, jobs, device, capture):
        self.part = _lib.empty(floats, torch.float32, device)
        self.counters = torch.zeros(jobs, dtype=torch.int32, device=device)
        self.capture, self.floats, self.jobs = capture, floats, jobs
        self.part_at, self.counters_at = self.part.data_ptr(), self.counters.data_ptr()


_ws: dict = {}
_ws_lock = threading.Lock()


@functools.lru_cache(maxsize=64)
def _part_floats(index, dh):                      # a function of the device and the head dimension
    return _lib.cuda().sb_quant_kv_attention_floats(dh)


def _workspace(index, stream, floats, jobs):
    """Launches on one stream follow one another and share one. Those of a graph share one of the graph's memory, whose counters it clears
    itself: graphs captured on one stream may be replayed at once on two."""
    capture = 0
    if torch._C._cuda_isCurrentStreamCapturing():
        word = (C.c_ulonglong * 1)()
        _lib.call("sb_stream_capture_id", stream, word)
        capture = word[0]
    key = (index, stream, capture != 0)
    w = _ws.get(key)
    if w is None or w.capture != capture or w.jobs < jobs or w.floats < floats or _lib.DEBUG_POISON:
        with _ws_lock:
            w = _ws.get(key)
            if w is None or w.capture != capture or w.jobs < jobs or w.floats < floats or _lib.DEBUG_POISON:
                w = _ws[key] = _Workspace(floats, max(jobs, 4096), torch.device("cuda", index), capture)
    return w


def drop_workspace(device, stream):
    """Gives back what calls on ``stream`` (a handle) work in, some 4 MB, where no more of them are to come."""
    for captured in (False, True):
        _ws.pop((device.index, stream, captured), None)


def decode_attention_ref(q, pool, block_table, seq_len, H, Hkv, dh, scale=None):
    """fp32 statement, one sequence at a time; a sequence of no positions gets zeros, and pages outside the pool hold zeros."""
    codes, scales, _, _, page, _, block = _layout("decode_attention", pool, Hkv, dh)
    scale = 1.0 / math.sqrt(dh) if scale is None else scale
    out = torch.zeros((q.shape[0], H * dh), dtype=torch.float32, device=q.device)
    for b, length in enumerate(seq_len.tolist()):
        length = min(length, block_table.shape[1] * page)
        if length <= 0:
            continue
        ids = block_table[b, :(length + page - 1) // page].long()
        known = (ids >= 0) & (ids < codes.shape[0])
        ids = ids.where(known, 0)
        kv = _values(codes.view(torch.int8)[ids].view(codes.dtype), scales[ids], block).where(known[:, None, None, None, None], 0.0)
        k, v = kv.permute(1, 2, 0, 3, 4).reshape(2, Hkv, -1, dh)[:, :, :length]
        s = torch.einsum("hgd,hld->hgl", q[b, :H * dh].float().reshape(Hkv, H // Hkv, dh), k) * scale
        out[b] = torch.einsum("hgl,hld->hgd", torch.softmax(s, -1), v).reshape(-1)
    return out


def decode_attention(q, pool, block_table, seq_len, H, Hkv, dh, scale=None, max_len=None, out=None):
    """GQA attention of one new token of each sequence over its paged KV in 8 bits. ``q`` [B, >= H * dh] bf16 holds the query heads (rotated);
    the token's own key and value are in ``pool`` already and counted by ``seq_len`` [B]. ``max_len`` bounds the lengths (default: the table);
    it is for the size of the launch only. A sequence of no positions (an empty slot) gets zeros. Positions behind a sequence's last one
    may hold any code and any scale; page ids outside the pool count as pages of zeros. Scores may lie anywhere between -2^127 and 2^127;
    a sequence's scales of values, positive as those that are written, may be up to 2^100 times one another. A head's query is taken over int8 codes
    as whole numbers of 15 bits, relative to its largest element. Returns bf16 [B, H * dh], ``out`` if that is given; ``out`` may not lie in
    what the call reads."""
    codes, scales, n_blocks, _, page, _, block = _layout("decode_attention", pool, Hkv, dh)
    scale = 1.0 / math.sqrt(dh) if scale is None else float(scale)
    shape = q.shape
    if len(shape) != 2 or H <= 0 or H % Hkv or shape[1] < H * dh or not scale > 0.0:
        raise ValueError("decode_attention: q must be [B, >= H * dh], heads a multiple of kv heads, scale positive")
    B, max_blocks = _batch("decode_attention", shape[0], seq_len, block_table, None)
    if n_blocks == 0:
        raise ValueError("decode_attention: the pool has no pages")
    if q.dtype is not BF or (out is not None and (out.dtype is not BF or tuple(out.shape) != (B, H * dh))):
        raise ValueError("decode_attention: q must be bf16, out bf16 [B, H * dh]")
    index = q.get_device()
    if index < 0:
        _on_host("decode_attention", codes, block_table, seq_len, out)
        o = decode_attention_ref(q, pool, block_table, seq_len, H, Hkv, dh, scale).to(BF)
        return o if out is None else out.copy_(o)
    if index != _lib.current_device():
        with torch.cuda.device(index):
            return decode_attention(q, pool, block_table, seq_len, H, Hkv, dh, scale, max_len, out)
    codes_at = _on_device("decode_attention", index, codes, scales, dh, (block_table, seq_len))
    (ldq, unit), q_at = q.stride(), q.data_ptr()
    if B == 1:
        ldq = H * dh
    if unit != 1 or ldq % 8 or ldq < H * dh or q_at % 16:
        raise ValueError("decode_attention: rows of q must be contiguous, apart and 16-byte aligned")
    if out is None:
        out = _lib.empty((B, H * dh), BF, q.device) if _lib.DEBUG_POISON else q.new_empty((B, H * dh))       # cheaper than torch.empty
        ldo, o_at = H * dh, out.data_ptr()
    else:
        (ldo, unit), o_at = out.stride(), out.data_ptr()
        ldo = H * dh if B == 1 else ldo
        if unit != 1 or ldo % 8 or ldo < H * dh or o_at % 16 or out.get_device() != index:
            raise ValueError("decode_attention: rows of out must be contiguous, apart, 16-byte aligned and on the device of q")
    if B == 0:
        return out
    if page % TILE and page not in (8, 16, 32):
        raise ValueError("decode_attention: pages of 8, 16, 32 or a multiple of 64 positions")
    if scales.numel() >= 1 << 31:
        raise ValueError("decode_attention: more scales than 31 bits count")
    tiles = -(-max_blocks * page // TILE)                       # of a sequence, at most
    jobs = Hkv * -(-(H // Hkv) // JOB_HEADS)
    at_once = min(B, LAUNCH_SEQUENCES, ((1 << 31) - 1) // (tiles * jobs))
    if at_once == 0:
        raise ValueError("decode_attention: a table of more tiles and heads than 31 bits count")
    if max_len is not None:
        tiles = min(tiles, max(1, -(-int(max_len) // TILE)))
    stream = _lib.stream()
    ws = _workspace(index, stream, _part_floats(index, dh), at_once * jobs)
    status, table_at, lens_at = _lib.status_word(q.device).data_ptr(), block_table.data_ptr(), seq_len.data_ptr()
    for b in range(0, B, at_once):
        n = min(at_once, B - b)
        _lib.call("sb_quant_kv_attention", q_at + b * ldq * 2, ldq, codes_at, codes.dtype is not torch.int8, scales.data_ptr(), n_blocks, page, block,
                  table_at + b * max_blocks * 4, max_blocks, lens_at + b * 4, n, H, Hkv, dh, n * jobs * tiles, scale, ws.part_at, ws.counters_at,
                  o_at + b * ldo * 2, ldo, status, stream)
        _g.launch_count += 1
    return out
