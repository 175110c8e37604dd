"""Ops on a paged KV cache whose sequences share pages: the attention of a batch behind a common prefix
(csrc/paged_attention_tcgen05.cu), and copies of pages in all layers' pools (csrc/page_copy.cu). CPU tensors take the PyTorch statement
of the same arithmetic."""
from __future__ import annotations

import ctypes as C
import functools
import math
import threading

import torch

from . import _lib
from . import gemm as _g

BF = torch.bfloat16
vp, i32, i64, f32, sz = _lib.vp, _lib.i32, _lib.i64, _lib.f32, _lib.sz
_lib.register("sb_shared_prefix_attention", [vp, i64, vp, i32, vp, i32, i32, vp, vp, i32, vp, i32, i32, i32, i32, i32, i64, f32, vp, sz,
                                             vp, i64, i32, vp, vp])

_lib.register("sb_copy_pages", [vp, vp, i32, vp, vp, i32, i32, i32, i64, i32, i64, i64, vp])

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


class _Workspace:
    """The workspace of a stream's calls. The launches of a call hand their parts on in it, so ``lock`` is held around them: of two threads
    on one stream one would launch between the other's, whose second launch then read what is not its own."""
    __slots__ = ("lock", "buffer", "bytes")

    def __init__(self):
        self.lock, self.buffer, self.bytes = threading.Lock(), None, 0

    def at_least(self, n, device):
        if self.bytes < n:                  # the buffer before goes back to the stream whose launches use it
            self.buffer, self.bytes = _lib.empty(n, torch.uint8, device), n
        return self.buffer.data_ptr()


_ws: dict = {}


def _workspace(device, stream):
    """Calls on one stream follow one another and share one; what is being captured into a graph gets its own from the graph's pool, since
    graphs captured on one stream may be replayed at once on two."""
    if _lib.DEBUG_POISON or torch._C._cuda_isCurrentStreamCapturing():
        return _Workspace()
    key = (device.index, stream)
    return _ws.get(key) or _ws.setdefault(key, _Workspace())


def drop_workspace(device, stream):
    """Gives back what calls on ``stream`` (a handle) work in, some 40 MB, where no more of them are to come. Launches under way keep it: it
    goes to that stream's next allocations."""
    _ws.pop((device.index, stream), None)


@functools.lru_cache(maxsize=4096)       # a function of the device and the sizes
def _workspace_bytes(device, NT, B, H, Hkv, dh, ragged, prefix):
    fn = _lib.cuda().sb_shared_prefix_attention_bytes
    fn.argtypes, fn.restype = [i32] * 7, sz
    return fn(NT, B, H, Hkv, dh, int(ragged), prefix)


def _in_common(n, B, per_tile, prefix, longest=0) -> bool:
    """Whether the rows of ``B`` sequences, ``n`` tokens in all, ``per_tile`` of which fill a tile, go over the prefix together. That takes as
    many tiles as all rows fill, apart each sequence's last one is partly empty; but parts in common have to be joined. us, apart / in common,
    32 / 8 heads, 32 tokens a tile. 16 sequences behind 4096: of 16 tokens 49.9 / 44.0, 24 51.8 / 50.7, 32 53.4 / 57.1, 48 86.4 / 77.2, 64
    89.9 / 97.3. Behind 8192 and 16384: 33 136 / 93, 261 / 169, 1 to 64 112 / 91, 214 / 163, 64 149 / 156, 265 / 294, 100 267 / 236, 501 / 458, 1
    to 300 286 / 282, 501 / 510; one of 1000 beside 31 of one token 486 / 298. Behind 512: 33 30.4 / 31.8, 64 35.3 / 41.4, 100 50.5 / 63.1; behind
    2048 33 53.6 / 46.6, 64 59.5 / 66.4, 100 96.2 / 101.5; one of 1000 beside 31 behind 1024 73.5 / 73.8. The host knows the tokens' sum and,
    where the caller says how long sequences are, the ``longest`` run: behind a long prefix they go apart only where all fill their tiles or
    the last tiles are few beside the others. A part in common takes 1 KB of workspace a row and head, so batches of more than 8192 tokens do
    not ask for it beyond where they did not fill tiles."""
    full = n == B * longest and longest % per_tile == 0
    return n < B * per_tile or (prefix >= 4096 and n < min(4 * B * per_tile, 8193) and not full)


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
    it is for the size of the launch and how the work is split only. Rows of ``out`` that belong to no sequence stay as they are; without
    ``out`` they are zero.

    Positions that no row of the call sees may hold anything, infinities and NaN included. Among the new tokens of a sequence, and in the
    prefix for a sequence that ends inside it, what a row does not see may be any key; a value that is not finite reaches the row all the
    same, as in ``attention_fwd``. ``out`` may not lie in what the call reads."""
    scale = 1.0 / math.sqrt(dh) if scale is None else float(scale)
    (n, width), (B,), (rows, max_blocks) = q.shape, seq_len.shape, block_table.shape
    n_blocks, *layout = pool.shape
    prefix = int(prefix_len) // page * page if prefix_table is not None else 0
    if H <= 0 or H % Hkv or page <= 0 or prefix_len < 0 or not scale > 0.0:
        raise ValueError("shared_prefix_attention: heads must divide by kv heads, page and scale be positive")
    if layout != [2, Hkv, page, dh] or rows != B or (B and not max_blocks):
        raise ValueError("shared_prefix_attention: pool must be [n_blocks, 2, Hkv, page, dh] and block_table [B, pages >= 1]")
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
    index = q.get_device()
    if not (block_table.get_device() == seq_len.get_device() == pool.get_device() == index
            and (not prefix or prefix_table.get_device() == index) and (cu_q is None or cu_q.get_device() == index)
            and (out is None or out.get_device() == index)):
        raise ValueError("shared_prefix_attention: all tensors must be on the device of q")
    (ldq, unit), q_at = q.stride(), q.data_ptr()
    if n == 1:
        ldq = H * dh                                # a dimension of one has any stride
    if unit != 1 or ldq % 8 or ldq < H * dh or q_at % 16 or not pool.is_contiguous():
        raise ValueError("shared_prefix_attention: pool must be contiguous, rows of q contiguous, apart and 16-byte aligned")
    if out is None:
        fill, ldo = 1, H * dh
        out = _lib.empty((n, ldo), BF, device) if _lib.DEBUG_POISON else q.new_empty((n, ldo))       # two thirds of torch.empty's time
    else:
        fill, (ldo, unit) = 0, out.stride()
        ldo = H * dh if n == 1 else ldo
        if unit != 1 or ldo % 8 or ldo < H * dh or out.data_ptr() % 16:
            raise ValueError("shared_prefix_attention: rows of out must be contiguous, apart and 16-byte aligned")
    if n == 0:
        return out
    if B == 0:
        return out.zero_() if fill else out
    per_tile = TILE_ROWS // (H // Hkv)
    if cu_q is not None and not _in_common(n, B, per_tile, prefix, 0 if max_len is None else max_len - prefix_len):
        prefix = 0
    L = max_blocks * page if max_len is None else min(int(max_len), max_blocks * page)
    pairs = B if cu_q is None else B + n // per_tile
    units = Hkv * (-(-n // per_tile) * -(-prefix // BLOCK) + pairs * max(0, -(-(L - prefix) // BLOCK)))
    stream = _lib.stream()
    need, ws = _workspace_bytes(index, n, B, H, Hkv, dh, cu_q is not None, prefix), _workspace(device, stream)
    with ws.lock:
        at = ws.at_least(need, device)
        _lib.call("sb_shared_prefix_attention", q_at, ldq, pool.data_ptr(), n_blocks, block_table.data_ptr(), max_blocks, page,
                  seq_len.data_ptr(), prefix_table.data_ptr() if prefix else None, prefix, cu_q.data_ptr() if cu_q is not None else None,
                  B, n, H, Hkv, dh, units, scale, at, ws.bytes, out.data_ptr(), ldo, fill, _lib.status_word(device).data_ptr(), stream)
    _g.launch_count += 2 if cu_q is None else 3
    return out


def _overlap(spans) -> bool:
    """Whether one of the address ranges, sorted, reaches into another that does not begin where it does."""
    return any(a[0] != b[0] and b[0] < a[1] for a, b in zip(spans, spans[1:]))


class PagePools:
    """The pools of a cache's layers, checked once: tensors of one shape ``[n_blocks, ..., page, width]``, type and device, each contiguous.
    It holds on to the tensors; one that is replaced in the cache needs a new handle."""

    def __init__(self, pools):
        self.pools = list(pools)
        if not self.pools or self.pools[0].dim() < 3:
            raise ValueError("PagePools: at least one pool of [n_blocks, ..., page, width]")
        p = self.pools[0]
        self.shape, self.dtype, self.device = tuple(p.shape), p.dtype, p.device
        for t in self.pools:
            if tuple(t.shape) != self.shape or t.dtype != self.dtype or t.device != self.device or not t.is_contiguous():
                raise ValueError("PagePools: contiguous pools of one shape, type and device")
        self.n_blocks, self.page = self.shape[0], self.shape[-2]
        self.heads = math.prod(self.shape[1:-2])                      # of K and of V
        self.row_bytes = self.shape[-1] * p.element_size()            # of a position of a head
        self.page_bytes = self.heads * self.page * self.row_bytes
        size = self.n_blocks * self.page_bytes
        self.spans = sorted((t.data_ptr(), t.data_ptr() + size) for t in self.pools)
        if _overlap(self.spans):
            raise ValueError("PagePools: pools reach into one another")
        self._table = (C.c_void_p * len(self.pools))(*[t.data_ptr() for t in self.pools])
        self.table = C.addressof(self._table)

    def __len__(self):
        return len(self.pools)


def _page_ids(ids, n_blocks, what):
    ids = [int(i) for i in (ids.tolist() if torch.is_tensor(ids) else ids)]
    if any(not 0 <= i < n_blocks for i in ids):
        raise ValueError(f"copy_pages: {what} page outside the pool")
    return ids


def copy_pages(pools, src, dst, rows=None, out=None):
    """Copies page ``src[i]`` to page ``dst[i]`` in every layer's pool, or to ``dst[i]`` of the pools ``out``; with ``rows`` only the first
    ``rows`` positions of each page. ``pools`` (and ``out``) is a ``PagePools`` or a list of pools.

    A source may be copied many times; a destination must occur once and, in the same pools, be no source. Pools may not reach into one
    another, nor may one occur twice in ``out``. Ids from the host (a list, a CPU tensor) are checked. Ids on the device (int32) are taken
    as they are, so that a captured call can be replayed with others; ids outside the pools are skipped there, as padding may be."""
    pools = pools if isinstance(pools, PagePools) else PagePools(pools)
    to = pools if out is None else out if isinstance(out, PagePools) else PagePools(out)
    if to is not pools and (len(to) != len(pools) or to.shape[1:] != pools.shape[1:] or to.dtype != pools.dtype or to.device != pools.device):
        raise ValueError("copy_pages: out must be as many pools of the same pages, type and device")
    if to is not pools and (_overlap(sorted(pools.spans + to.spans)) or any(a[0] == b[0] < a[1] for a, b in zip(to.spans, to.spans[1:]))):
        raise ValueError("copy_pages: pools reach into one another, or out has one twice")
    if rows is not None and not 0 <= rows <= pools.page:
        raise ValueError("copy_pages: rows must be between 0 and the positions of a page")
    device = pools.device
    on_device = device.type == "cuda" and torch.is_tensor(src) and torch.is_tensor(dst) and src.is_cuda and dst.is_cuda
    if on_device:
        if (src.dtype is not torch.int32 or dst.dtype is not torch.int32 or src.shape != dst.shape or src.dim() != 1
                or not src.is_contiguous() or not dst.is_contiguous() or src.device != device or dst.device != device):
            raise ValueError("copy_pages: page ids on the device must be two contiguous int32 vectors of one length, beside the pools")
    else:
        src, dst = _page_ids(src, pools.n_blocks, "source"), _page_ids(dst, to.n_blocks, "destination")
        if len(src) != len(dst) or len(set(dst)) != len(dst):
            raise ValueError("copy_pages: as many destinations as sources, each once")
        same = {at for at, _ in pools.spans} & {at for at, _ in to.spans}
        if same and set(src) & set(dst):
            raise ValueError("copy_pages: a page is both source and destination")
    n = len(src)
    if n == 0 or rows == 0 or pools.page_bytes == 0:
        return
    rows = pools.page if rows is None else rows
    if device.type != "cuda":
        a, b = torch.tensor(src, device=device), torch.tensor(dst, device=device)
        for s, d in zip(pools.pools, to.pools):
            d[b, ..., :rows, :] = s[a, ..., :rows, :]
        return
    if device.index != _lib.current_device():
        with torch.cuda.device(device):
            return copy_pages(pools, src, dst, rows, to)
    if not on_device:
        src, dst = torch.tensor([src, dst], dtype=torch.int32).to(device)
    pitch = pools.page * pools.row_bytes
    whole = rows == pools.page
    _lib.call("sb_copy_pages", pools.table, to.table, len(pools), src.data_ptr(), dst.data_ptr(), n, pools.n_blocks, to.n_blocks,
              pools.page_bytes, 1 if whole else pools.heads, pools.page_bytes if whole else rows * pools.row_bytes,
              pools.page_bytes if whole else pitch, _lib.stream())
    _g.launch_count += -(-len(pools) // 64)
