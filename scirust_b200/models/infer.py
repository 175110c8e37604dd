"""Inference engine for the SciAgent / Llama-shaped GQA decoder: batched flash prefill, paged
KV cache in bf16 or 8 bits, split-KV flash-decode, bf16 or int8 per-output-channel weights, device-side greedy
feedback (no per-token device->host copy) and CUDA-graph replay of the decode step.

Counterparts in the reference: ``CudaModel::prefill_cached`` / ``decode_step_cached`` /
``generate_cached`` (scirust-sciagent/src/cuda_model.rs:450-581), the batch-1 latency decoder with
fused QKV and gate/up, fixed-capacity KV and device feedback (scirust-sciagent/src/cuda_decode.rs:
17-470), ``PagedKvCache`` (scirust-core/src/nn/paged_attention.rs:21-147) and per-channel int8
weights (scirust-core/src/quantization.rs:95-190). Differences by design: prefill is one batched
causal pass (the reference's latency decoder feeds the prompt token by token), the cache is paged
and pre-sized (the reference's general path re-allocates the cache every token), any batch size
decodes in one step, and sampling other than greedy uses the shared ``sample_row`` policy on a
logits row copied to the host.
"""
from __future__ import annotations

import os

import ctypes as C
import math

import torch

from .. import ops
from ..generate import SamplingParams
from ..ops.sampling import DeviceSampler
from ..ops import _lib, attention as att, decode as D, gemm as G, paged, quantized_kv as Q
from .sciagent import BF, GQADecoder, SciAgentConfig


class BlockAllocator:
    """Host-side page allocator (native: csrc/rt_alloc.cpp)."""

    def __init__(self, n_blocks: int):
        lib = _lib.rt()
        lib.sbrt_balloc_new.restype = C.c_void_p
        lib.sbrt_balloc_new.argtypes = [C.c_int32]
        lib.sbrt_balloc_delete.argtypes = [C.c_void_p]
        lib.sbrt_balloc_num_free.argtypes = [C.c_void_p]
        lib.sbrt_balloc_num_free.restype = C.c_int32
        lib.sbrt_balloc_alloc.argtypes = [C.c_void_p, C.c_int32, C.c_void_p]
        lib.sbrt_balloc_alloc.restype = C.c_int32
        lib.sbrt_balloc_free.argtypes = [C.c_void_p, C.c_void_p, C.c_int32]
        lib.sbrt_balloc_free.restype = C.c_int32
        lib.sbrt_balloc_share.argtypes = [C.c_void_p, C.c_void_p, C.c_int32]
        lib.sbrt_balloc_share.restype = C.c_int32
        lib.sbrt_balloc_owners.argtypes = [C.c_void_p, C.c_int32]
        lib.sbrt_balloc_owners.restype = C.c_int32
        lib.sbrt_balloc_compact.argtypes = [C.c_void_p, C.c_int32, C.c_void_p]
        lib.sbrt_balloc_compact.restype = C.c_int32
        self._lib = lib
        self._h = lib.sbrt_balloc_new(n_blocks)
        if not self._h:
            raise ValueError("n_blocks must be positive")
        self.n_blocks = n_blocks

    def num_free(self) -> int:
        return int(self._lib.sbrt_balloc_num_free(self._h))

    def alloc(self, n: int) -> list:
        buf = (C.c_int32 * max(n, 1))()
        if self._lib.sbrt_balloc_alloc(self._h, n, buf) != 0:
            raise MemoryError(f"KV cache exhausted: {n} pages requested, {self.num_free()} free")
        return list(buf[:n])

    def share(self, ids) -> None:
        """One more owner for each of these pages, which are in use: ``free`` returns a page when its last owner gives it up."""
        ids = list(ids)
        buf = (C.c_int32 * max(len(ids), 1))(*ids)
        if self._lib.sbrt_balloc_share(self._h, buf, len(ids)) != 0:
            raise ValueError("only pages in use can be shared")

    def owners(self, page: int) -> int:
        """How many own the page; 0 if it is free."""
        n = int(self._lib.sbrt_balloc_owners(self._h, page))
        if n < 0:
            raise ValueError("no such page")
        return n

    def compact(self, n_blocks: int | None = None) -> list:
        """Numbers the pages in use anew from 0 on, in a pool of ``n_blocks`` (default: as many as now): the new id of every page, -1 for a
        free one. The lowest ids stay as they are, the others move into the holes."""
        n = self.n_blocks if n_blocks is None else n_blocks
        to = (C.c_int32 * self.n_blocks)()
        if self._lib.sbrt_balloc_compact(self._h, n, to) < 0:
            raise MemoryError(f"{self.n_blocks - self.num_free()} pages in use do not fit into {n}")
        self.n_blocks = n
        return list(to)

    def free(self, ids) -> None:
        ids = list(ids)
        buf = (C.c_int32 * max(len(ids), 1))(*ids)
        if self._lib.sbrt_balloc_free(self._h, buf, len(ids)) != 0:
            raise ValueError("invalid page ids returned to the allocator")

    def __del__(self):
        try:
            if self._h:
                self._lib.sbrt_balloc_delete(self._h)
                self._h = None
        except Exception:
            pass


class PagedKVCache:
    """Pools ``[n_layers][n_blocks, 2, Hkv, page, dh]`` (bf16, or with ``codes`` 8-bit ``QuantPool``s, whose scales count for ``block`` positions) +
    block table + lengths."""

    def __init__(self, n_layers, n_blocks, Hkv, dh, page, max_batch, max_seq, device, codes=None, block=None):
        self.page, self.max_batch = page, max_batch
        self.max_blocks = (max_seq + page - 1) // page
        self.quantized = codes is not None
        if self.quantized:
            self.pools = [Q.QuantPool.zeros(n_blocks, Hkv, page, dh, codes, block, device) for _ in range(n_layers)]
        else:
            self.pools = [torch.zeros((n_blocks, 2, Hkv, page, dh), dtype=BF, device=device) for _ in range(n_layers)]
        self.alloc = BlockAllocator(n_blocks)
        self.table_host = torch.zeros((max_batch, self.max_blocks), dtype=torch.int32)
        self.block_table = torch.zeros((max_batch, self.max_blocks), dtype=torch.int32, device=device)
        self.seq_len = torch.zeros(max_batch, dtype=torch.int32, device=device)
        self.owned = [[] for _ in range(max_batch)]

    def reserve(self, seq: int, n_tokens: int) -> None:
        """Make sure sequence ``seq`` owns pages for positions < n_tokens."""
        need = (n_tokens + self.page - 1) // self.page
        if need > self.max_blocks:
            raise ValueError("sequence longer than the cache was sized for")
        have = len(self.owned[seq])
        if need > have:
            new = self.alloc.alloc(need - have)
            self.table_host[seq, have:need] = torch.tensor(new, dtype=torch.int32)
            self.owned[seq] += new

    def commit(self) -> None:
        self.block_table.copy_(self.table_host, non_blocking=True)

    def release(self, seq: int) -> None:
        self.alloc.free(self.owned[seq])
        self.owned[seq] = []
        self.table_host[seq].zero_()

    def _copy_pages(self, src, dst, rows=None, pools=None, to=None) -> None:
        """``paged.copy_pages`` in the layers' pools, with 8 bits of codes (their first ``rows``) and of all scales."""
        pools = self.pools if pools is None else pools
        if not self.quantized:
            return paged.copy_pages(paged.PagePools(pools), src, dst, rows=rows, out=paged.PagePools(to) if to is not None else None)
        for part, n in ((0, rows), (1, None)):
            parts = [[p[part].view(torch.uint8) if part == 0 else p[part] for p in side] if side is not None else None for side in (pools, to)]
            paged.copy_pages(paged.PagePools(parts[0]), src, dst, rows=n, out=paged.PagePools(parts[1]) if to is not None else None)

    def fork(self, src: int, seqs, n_tokens: int) -> None:
        """Gives the sequences ``seqs``, which have no pages, the first ``n_tokens`` positions of ``src``. Whole pages are shared: each counts
        its owners and is free again with the last of them. A page that the positions do not fill is copied for every sequence, as far as it is
        filled, since each writes on in its own. ``commit`` makes the tables known to the device, as after ``reserve``."""
        seqs = list(seqs)
        whole, rest = divmod(n_tokens, self.page)
        if not 0 <= src < self.max_batch or n_tokens < 0 or len(self.owned[src]) < whole + bool(rest):
            raise ValueError("fork: the sequence does not hold so many positions")
        if len(set(seqs)) != len(seqs) or any(not 0 <= s < self.max_batch or self.owned[s] for s in seqs):
            raise ValueError("fork: to different sequences of the cache without pages")
        last = self.alloc.alloc(len(seqs)) if rest else []
        self.alloc.share(self.owned[src][:whole] * len(seqs))
        for i, s in enumerate(seqs):
            self.owned[s] = self.owned[src][:whole] + last[i:i + 1]
            self.table_host[s, :len(self.owned[s])] = torch.tensor(self.owned[s], dtype=torch.int32)
        if last:
            self._copy_pages([self.owned[src][whole]] * len(seqs), last, rows=rest)

    def _renumber(self, to) -> None:
        for s, ids in enumerate(self.owned):
            self.owned[s] = [to[i] for i in ids]
            if ids:
                self.table_host[s, :len(ids)] = torch.tensor(self.owned[s], dtype=torch.int32)
        self.commit()

    def compact(self) -> int:
        """Moves pages so that those in use have the lowest ids, and returns how many they are. Tables that the caller has of its own (a copy
        of a row of ``block_table``, the page ids of a shared prefix) have to be read again."""
        to = self.alloc.compact()
        moves = [(a, b) for a, b in enumerate(to) if b not in (-1, a)]
        self._copy_pages([a for a, _ in moves], [b for _, b in moves])
        self._renumber(to)
        return sum(b >= 0 for b in to)

    def resize(self, n_blocks: int) -> None:
        """Pools of ``n_blocks`` pages, more or fewer, with what the sequences hold; MemoryError if that is more. Pages are numbered anew as
        by ``compact``, and the pools are other tensors: what was captured into a graph with the old ones still uses those."""
        old = self.pools
        live = self.alloc.n_blocks - self.alloc.num_free()
        if n_blocks < max(live, 1):
            raise MemoryError(f"{live} pages in use do not fit into {n_blocks}")
        def empty(t):
            return torch.zeros((n_blocks, *t.shape[1:]), dtype=torch.uint8, device=t.device).view(t.dtype) if t.element_size() == 1 else \
                torch.zeros((n_blocks, *t.shape[1:]), dtype=t.dtype, device=t.device)

        new = [Q.QuantPool(empty(p.codes), empty(p.scales)) if self.quantized else empty(p) for p in old]
        to = self.alloc.compact(n_blocks)
        pairs = [(a, b) for a, b in enumerate(to) if b >= 0]
        self._copy_pages([a for a, _ in pairs], [b for _, b in pairs], pools=old, to=new)
        self.pools[:] = new
        self._renumber(to)


class _WidenAhead:
    """The int8 matrices of one prefill in the order of their use. A long prompt's products take them as bf16, and expanding each before
    its product leaves the tensor cores idle for as long as memory takes. Instead the launch of a product also expands the next matrices,
    in warps that it has to spare, up to two codes for each of its own weights: the down product takes the next layer's gate/up
    matrix, the gate/up product down and the next qkv and output matrices. Us at 2048 rows, d 4096, ff 14336, expanded before / beside:
    gate/up with down 383 / 336, down with the next gate/up 224 / 199, qkv with the output matrix 82.8 / 78.4; more gains less than the
    next product would with it (qkv with down, 2.3 codes for one, 12 us, gate/up 47) or loses (output product with gate/up, 7 codes, 108
    / 114). At 1024 rows gate/up with three 219 / 202, down with gate/up 139 / 129; d 1024 at 2048 rows gate/up with three 43.5 / 34.4.
    Up to three matrices more than without it are in memory; where memory runs out, for one of them or for what a layer needs beside
    them (``run``), those expanded ahead are given back and every matrix is expanded before its product again."""

    AHEAD = 3
    # Rows times the elements of gate/up. Below it a layer waits for the host, whom planning costs more (12 us) than the launches that it
    # saves: one layer of d 1024, 2000 rows 311 us without and 321 with it, 8192 rows 389 and 349. Of 64 prefills (d 512 to 4096, one and
    # four layers, 1024 to 12000 rows) the line takes the slower way by up to 6 %, all within a factor of 1.5 of it: four layers of d 1024,
    # 4096 rows (2^34.5) 867 without and 821 with, of d 2048, 1024 rows 887 and 846; one layer of d 2048, 1500 rows (2^35) 325 and 334.
    WORK = 1 << 35

    def __init__(self, layers, rows):
        self.rows = rows
        self.order = []
        if layers and rows >= 1024 and rows * math.prod(layers[0]["wgu"].shape) >= self.WORK:
            self.order = [l[k] for l in layers for k in ("wqkv", "wo", "wgu", "wd")]
        self.at = 0
        self.wide = {}                 # position in the order -> bf16 matrix
        self.taken = 0                 # matrices expanded ahead so far
        self.ran_out = False

    def product(self, w):
        """The next product's matrix (expanded, or as it is) and what its launch is to expand, as keyword arguments."""
        if not self.order:
            return w, {}
        w = self.wide.pop(self.at, w)
        self.at += 1
        K, N = w.shape
        if not G.widens_beside(self.rows, N, K):
            return w, {}
        room, jobs = 2 * K * N, []
        for i in range(self.at, min(self.at + self.AHEAD, len(self.order))):
            q = self.order[i]
            if i in self.wide:
                continue
            if type(q) is not D.QuantWeight or not q.widenable() or q.q.numel() > room:      # a subclass may expand in its own way
                break
            try:
                out = torch.empty(q.shape, dtype=torch.bfloat16, device=q.q.device)
            except torch.OutOfMemoryError:
                break
            room -= q.q.numel()
            self.wide[i] = out
            self.taken += 1
            jobs.append((q.q, q.scale, out))
        return w, {"widen": jobs} if jobs else {}

    def run(self, part, *args):
        """``part(*args)``, a piece of a layer that can be run again; if memory runs out in it, once more with nothing expanded ahead. The
        second run is outside the handler, whose exception holds on to what the first one had allocated."""
        try:
            return part(*args)
        except torch.OutOfMemoryError:
            if not self.taken:
                raise
            self.order, self.wide, self.taken = [], {}, 0
            self.ran_out = True
        return part(*args)


class InferenceEngine:
    def __init__(self, model: GQADecoder, quant: str | None = None, max_batch: int = 1, max_seq: int = 4096,
                 page: int = 64, use_graph: bool = True, kv: str | None = None, kv_block: int | None = None):
        """``quant="int8"``: int8 weights. ``kv="int8"`` or ``"e4m3"``: a cache of half the size in 8 bits, one scale for ``kv_block`` positions of
        a head (default: 16); decoding reads half the bytes, and what the cache holds is rounded once more. Large batches gain by it, one
        sequence of a few thousand positions does not (8B model behind 2048 positions, ms a step bf16 / int8: batch of 64 6.9 / 5.6, 16 4.2 / 3.9,
        one 3.24 / 3.27), and many sequences behind a long common prefix (``generate_shared``) lose, since each reads the prefix for itself: 16
        behind 2048 positions 3.8 / 3.8, 16 behind 8192 4.2 / 4.7, 64 behind 1024 4.4 / 4.6, 64 behind 8192 4.9 / 8.6."""
        cfg = model.cfg
        self.cfg, self.quant = cfg, quant
        dev = model.flat.device
        self.dev = dev
        self.max_batch, self.max_seq = max_batch, max_seq
        self.use_graph = use_graph and dev.type == "cuda"

        self.H, self.Hkv = cfg.n_heads, cfg.n_kv_heads      # heads held by this rank
        self._load_weights(model)
        n_blocks = max_batch * ((max_seq + page - 1) // page)
        self.kv = kv
        if kv is not None and dev.type == "cuda" and (page not in (8, 16, 32) and page % 64 or cfg.head_dim not in (64, 128)):
            raise ValueError("a cache in 8 bits has pages of 8, 16, 32 or a multiple of 64 positions and heads of 64 or 128")
        self.cache = PagedKVCache(cfg.n_layers, n_blocks, self.Hkv, cfg.head_dim, page, max_batch, max_seq, dev, kv, kv_block)
        self.cos, self.sin = ops.rope_table(max(cfg.max_seq_len, max_seq), cfg.head_dim, cfg.rope_theta, dev)
        self.tokens = torch.zeros(max_batch, dtype=torch.int64, device=dev)     # device feedback buffer
        self.logits = torch.zeros((max_batch, cfg.vocab_size), dtype=torch.float32, device=dev)
        self._graph = None
        self._graph_batch = None
        self._generated = None
        # greedy decoding of up to 8 rows: the LM-head GEMV does its own arg-max (SB_FUSED_ARGMAX=0: three launches)
        self.fused_argmax = os.environ.get("SB_FUSED_ARGMAX", "1") != "0"

    def _prep(self, w):
        w = w.detach()
        return D.quantize_per_channel(w) if self.quant == "int8" else w

    def _load_weights(self, model: GQADecoder):
        prep = self._prep
        self.embed = model.embed.detach()
        self.layers = []
        for l in model.layers:
            self.layers.append({"rms1": l.rms_attn.detach(), "wqkv": prep(l.wqkv), "wo": prep(l.wo),
                                "rms2": l.rms_ffn.detach(), "wgu": prep(l.wgu), "wd": prep(l.wd)})
        self.rms_final = model.rms_final.detach()
        # LM head as [d, V] so the weight-streaming kernels read it row by row
        self.head_t = prep(model.head_weight().detach().t().contiguous())

    # ------------------------------------------------------------------ linear dispatch
    def _proj_out(self, a, w, x, swiglu=False, site="attn", widen=()):
        """x + f(a) @ w: the attention-output and MLP-down products (row-parallel under tensor
        parallelism, where a subclass adds the all-reduce). ``swiglu``: a is a fused [gate | up]. ``widen``: as in ``_linear``."""
        if a.shape[0] <= D.gemv_max_rows(w):
            return D.gemv(a, w, residual=x, swiglu=swiglu)
        if swiglu:
            a = ops.swiglu_fwd(a)
        return self._linear(a, w, residual=x, **({"widen": widen} if widen else {}))     # a subclass's may not know of it

    def _linear(self, x, w, residual=None, widen=()):
        """``widen``: int8 matrices of later products that this one's launch expands (``_WidenAhead``)."""
        M = x.shape[0]
        if M <= D.gemv_max_rows(w):
            return D.gemv(x, w, residual=residual)
        if D.skinny_ok(x, w):
            # 9..64 rows (batched decoding): still bound by the weight bytes; the weight-streaming tcgen05 kernel
            return D.matmul_skinny(x, w, residual=residual)
        if isinstance(w, D.QuantWeight):
            # few rows: the product is bound by the weight bytes, so the int8 matrix is streamed and
            # dequantised inside the GEMM; many rows (prefill): it is bound by the tensor cores, so the
            # layer's weights are expanded to bf16 once (a few percent of the GEMM's time) and the
            # plain bf16 kernel runs at full rate
            if M < 1024 and w.q.shape[1] % 16 == 0:
                return D.matmul_int8(x, w, residual=residual)
            w = w.dequantize()
        return G.matmul_nn_beside(x, w, residual, widen) if widen else ops.matmul_nn(x, w, residual=residual)

    def _products(self):
        """The functions behind this engine's products. What is done across them (gate/up without ``_linear``, expanding one's matrix in
        another's launch) is done only where they are known to go together: an override of one of them sees every product of its own."""
        return tuple(getattr(getattr(self, name), "__func__", None) for name in ("_linear", "_proj_out", "_gated"))

    def _gated(self, x, w, widen=()):
        """silu(gate) * up of ``[gate | up] = x @ w`` in one launch, or None where that is not how ``_linear`` takes the product (by
        1024 rows int8 weights are expanded whatever their shape)."""
        M, (K, N) = x.shape[0], w.shape
        if not x.is_cuda or not G.swiglu_in_epilogue(M, K, N // 2):
            return None
        if isinstance(w, D.QuantWeight):
            if M < 1024 and N % 16 == 0:
                return None
            w = w.dequantize()
        return ops.matmul_nn_swiglu_act(x, w, widen)

    # ------------------------------------------------------------------ prefill
    _ahead_below = math.inf              # rows of a prefill in which memory ran out for matrices expanded ahead: fewer may still have them

    def prefill(self, tokens: torch.Tensor):
        """tokens [B, P] (all prompts the same length). Fills the cache, leaves the greedy next
        token of every sequence in ``self.tokens`` and returns the last-position logits [B, V]."""
        cfg, cache = self.cfg, self.cache
        B, P = tokens.shape
        H, Hkv, dh = self.H, self.Hkv, cfg.head_dim
        tok = tokens.to(self.dev)
        for b in range(B):
            if cache.owned[b]:
                cache.release(b)
            cache.reserve(b, min(self.max_seq, P + 1))
        cache.commit()
        seq_of = torch.arange(B, dtype=torch.int32, device=self.dev).repeat_interleave(P)
        pos = torch.arange(P, dtype=torch.int32, device=self.dev).repeat(B)
        runs = (torch.full((B,), P, dtype=torch.int32, device=self.dev),
                torch.arange(0, B * P + 1, P, dtype=torch.int32, device=self.dev)) if self.kv is not None else None
        x = self._prompt_layers(tok.reshape(-1), seq_of, pos,
                                lambda li, qkv: att.attention_fwd(qkv, B, P, H, Hkv, dh, causal=True, want_lse=False)[0], runs)
        last = x.view(B, P, -1)[:, -1, :].contiguous()
        logits = self.logits[:B]
        self._head(last, logits, rms_weight=self.rms_final)
        D.argmax_rows(logits, out_tokens=self.tokens[:B])
        cache.seq_len[:B] = P
        return logits

    def _prompt_layers(self, tok, seq_of, pos, attend, runs=None):
        """All layers over prompt tokens: ``tok`` [n], token i at position ``pos[i]`` of sequence ``seq_of[i]``. Keys and values go to the
        cache, then ``attend(layer, qkv)`` is the attention. ``runs``: the same places as each sequence's length with its tokens, and where in
        ``tok`` it begins, [B + 1] (for a cache in 8 bits). Returns the residual stream [n, d]."""
        cfg, cache = self.cfg, self.cache
        H, Hkv, dh, n = self.H, self.Hkv, cfg.head_dim, tok.shape[0]
        x = ops.embed_fwd(self.embed, tok)
        products = self._products()
        gates = products in GATED_PRODUCTS
        ahead = products == _OWN_PRODUCTS and x.is_cuda and n < self._ahead_below
        plan = _WidenAhead(self.layers if ahead else [], n)

        def attention(li, l, x):
            h, _ = ops.rmsnorm_fwd(x, l["rms1"], cfg.eps, want_inv=False)
            w, kw = plan.product(l["wqkv"])
            qkv = self._linear(h, w, **kw)
            if self.kv is None:
                D.rope_kv_append(qkv, H, Hkv, dh, self.cos, self.sin, cache.pools[li], cache.block_table, cache.page, seq_of, pos)
            else:
                Q.rope_kv_append(qkv, H, Hkv, dh, self.cos, self.sin, cache.pools[li], cache.block_table[:runs[0].shape[0]], *runs)
            a = attend(li, qkv)
            w, kw = plan.product(l["wo"])
            return self._proj_out(a, w, x, site="attn", **kw)

        def feed_forward(l, x):
            h, _ = ops.rmsnorm_fwd(x, l["rms2"], cfg.eps, want_inv=False)
            w, kw = plan.product(l["wgu"])
            gu = self._gated(h, w, **kw) if gates else None          # silu(gate) * up
            fused = gu is not None
            if not fused:
                gu = self._linear(h, w, **kw)
            w, kw = plan.product(l["wd"])
            return self._proj_out(gu, w, x, swiglu=not fused, site="mlp", **kw)

        for li, l in enumerate(self.layers):
            x = plan.run(attention, li, l, x)
            x = plan.run(feed_forward, l, x)
        if plan.ran_out:
            self._ahead_below = n
        return x

    def _head(self, hn, logits, rms_weight=None):
        """logits[M, V] (fp32) = norm(hn) @ head; ``rms_weight`` asks for the final RMSNorm to be
        applied here (fused into the weight-streaming kernel when M <= 8)."""
        self._head_local(hn, logits, rms_weight)

    def _head_local(self, hn, logits, rms_weight=None):
        M = hn.shape[0]
        if M <= D.gemv_max_rows(self.head_t):
            D.gemv(hn, self.head_t, out_f32=logits, rms_weight=rms_weight, eps=self.cfg.eps)
            return
        if rms_weight is not None:
            hn, _ = ops.rmsnorm_fwd(hn, rms_weight, self.cfg.eps, want_inv=False)
        if D.skinny_ok(hn, self.head_t):
            logits.copy_(D.matmul_skinny(hn, self.head_t).float())
            return
        if isinstance(self.head_t, D.QuantWeight):
            logits.copy_(D.matmul_int8(hn, self.head_t).float())
        else:
            logits.copy_(ops.matmul_nn(hn, self.head_t).float())

    # ------------------------------------------------------------------ decode
    def _decode_body(self, B: int, max_len: int, greedy: bool = False, stream: bool | None = None):
        cfg, cache = self.cfg, self.cache
        H, Hkv, dh = self.H, self.Hkv, cfg.head_dim
        seq_of = self._seq_of[:B]
        pos = cache.seq_len[:B]
        x = ops.embed_fwd(self.embed, self.tokens[:B])
        # weight-streaming path: norms and SwiGLU are fused into the GEMV loads
        small = B <= D.gemv_max_rows(self.layers[0]["wqkv"])
        for li, l in enumerate(self.layers):
            if small:
                qkv = D.gemv(x, l["wqkv"], rms_weight=l["rms1"], eps=cfg.eps)
            else:
                h, _ = ops.rmsnorm_fwd(x, l["rms1"], cfg.eps, want_inv=False)
                qkv = self._linear(h, l["wqkv"])
            if self.kv is not None:
                table, lens = cache.block_table[:B], self._len_plus1[:B]
                Q.rope_kv_append(qkv, H, Hkv, dh, self.cos, self.sin, cache.pools[li], table, lens)
                a = Q.decode_attention(qkv, cache.pools[li], table, lens, H, Hkv, dh, max_len=max_len)
            else:
                D.rope_kv_append(qkv, H, Hkv, dh, self.cos, self.sin, cache.pools[li], cache.block_table, cache.page,
                                 seq_of, pos)
                if self._shared is not None:
                    a = paged.shared_prefix_attention(qkv, cache.pools[li], cache.block_table[:B], cache.page, self._len_plus1[:B],
                                                      *self._shared, H, Hkv, dh, max_len=max_len)
                else:
                    a = D.decode_attention(qkv, cache.pools[li], cache.block_table, cache.page, self._len_plus1[:B], H, Hkv,
                                           dh, max_len=max_len, stream=stream)
            x = self._proj_out(a, l["wo"], x, site="attn")
            if small:
                gu = D.gemv(x, l["wgu"], rms_weight=l["rms2"], eps=cfg.eps)
            else:
                h, _ = ops.rmsnorm_fwd(x, l["rms2"], cfg.eps, want_inv=False)
                gu = self._linear(h, l["wgu"])
            x = self._proj_out(gu, l["wd"], x, swiglu=True, site="mlp")
        if greedy and self._fused_argmax_ok(B):
            self._head_argmax(x, B)          # LM head and arg-max in one launch; the logits are not written
            return True
        self._head(x, self.logits[:B], rms_weight=self.rms_final)
        return False

    def _fused_argmax_ok(self, B: int) -> bool:
        return (self.dev.type == "cuda" and self.fused_argmax and B <= min(8, D.gemv_max_rows(self.head_t))
                and os.environ.get("SB_GEMV_FMA") != "1")

    def _head_argmax(self, x, B: int, logits=None):
        D.gemv_argmax(x, self.head_t, out_tokens=self.tokens[:B], rms_weight=self.rms_final, eps=self.cfg.eps,
                      logits=logits, generated=self._generated, step=0)

    def _step_eager(self, B, max_len, sampler=None, want_logits=False, stream=None):
        torch.add(self.cache.seq_len[:B], 1, out=self._len_plus1[:B])
        done = self._decode_body(B, max_len, greedy=sampler is None and not want_logits, stream=stream)
        if done:
            pass
        elif sampler is None:
            D.argmax_rows(self.logits[:B], out_tokens=self.tokens[:B], generated=self._generated, step=0)
        else:
            sampler.sample(self.logits[:B], out_tokens=self.tokens[:B])
            sampler.push(self.tokens[:B])
        self.cache.seq_len[:B] += 1

    def _streams(self, B: int, held: int) -> bool:
        """Which of the two decode-attention kernels suits ``B`` sequences of ``held`` positions (the cap that they may grow
        to does not count: the first part of a long generation is short)."""
        return (self.dev.type == "cuda" and self.kv is None
                and D._stream_wins(held, B * self.Hkv, self.H // self.Hkv, self.cache.page, self.dev))

    # A generation that crosses the line between the two kernels captures its step anew (two or three milliseconds for eight
    # layers), unless it ends within this many steps. 64 prompts of 128 tokens, 1800 new ones, eight layers of 4096: 2755 ms
    # so, 2903 with the split kernel to the end.
    RECAPTURE_STEPS = 64

    def generate(self, prompts: torch.Tensor, max_new: int, params: SamplingParams | None = None, seed: int = 0,
                 stop_on_zero: bool = False):
        """Greedy or sampled generation; the token never leaves the device between steps (arg-max or
        the device sampler write the feedback buffer) and the step is replayed from a CUDA graph.
        Sequence ``b`` samples from the stream seeded with ``seed + b``. Returns int64 [B, max_new]."""
        params = params or SamplingParams()
        B, P = prompts.shape
        if B > self.max_batch or P + max_new > self.max_seq:
            raise ValueError("request exceeds the engine's max_batch / max_seq")
        greedy = params.temperature <= 0.0 and params.repetition_penalty <= 1.0
        for b in range(B):
            if self.cache.owned[b]:
                self.cache.release(b)
        logits = self.prefill(prompts)
        if self.dev.type == "cuda":
            # benchmarks time the decode steps from here (prefill and its arg-max are behind this event)
            self.prefill_done = torch.cuda.Event(enable_timing=True)
            self.prefill_done.record()
        for b in range(B):
            self.cache.reserve(b, P + max_new)
        self.cache.commit()
        sampler = None
        if not greedy:
            sampler = DeviceSampler(params, B, self.cfg.vocab_size, [seed + b for b in range(B)], self.dev,
                                    history_len=P + max_new)
            sampler.set_history(prompts)
            sampler.sample(logits[:B], out_tokens=self.tokens[:B])
            sampler.push(self.tokens[:B])
        return self._decode_steps(B, P, max_new, sampler)

    def _decode_steps(self, B: int, P: int, max_new: int, sampler):
        """The tokens [B, max_new] from the first one, which is in ``self.tokens``, on; the longest of the sequences holds ``P``."""
        out = torch.zeros((B, max_new), dtype=torch.int64, device=self.dev)
        self._seq_of = torch.arange(self.max_batch, dtype=torch.int32, device=self.dev)
        self._len_plus1 = torch.zeros(self.max_batch, dtype=torch.int32, device=self.dev)
        self._generated = None
        out[:, 0] = self.tokens[:B]
        max_len = P + max_new
        stream = self._streams(B, P + 1)

        def crosses(i):
            return self._shared is None and max_new - i >= self.RECAPTURE_STEPS and self._streams(B, P + i) != stream

        if self.use_graph and max_new > 2:
            # one eager step on the capture stream warms every workspace (they are kept per stream, and nothing may be
            # allocated or cleared inside the capture), then the step is captured once and replayed
            s = torch.cuda.Stream(device=self.dev)
            graphs = []                        # an earlier one may still be running when the next is captured

            def capture(i):
                g = torch.cuda.CUDAGraph()
                s.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(s):
                    self._step_eager(B, max_len, sampler, stream=stream)
                    out[:, i] = self.tokens[:B]
                    if graphs:                 # in the middle of a generation, without torch.cuda.graph's collection and cache flush
                        g.capture_begin()
                        self._step_eager(B, max_len, sampler, stream=stream)
                        g.capture_end()
                    else:
                        with torch.cuda.graph(g, stream=s):
                            self._step_eager(B, max_len, sampler, stream=stream)
                graphs.append(g)
                torch.cuda.current_stream().wait_stream(s)

            capture(1)
            # capture only records; run the recorded step for positions 2 .. max_new-1
            for i in range(2, max_new):
                if crosses(i):
                    stream = not stream
                    capture(i)
                    continue
                graphs[-1].replay()
                out[:, i] = self.tokens[:B]
            paged.drop_workspace(self.dev, s.cuda_stream)       # of the eager step; the graphs have their own
            Q.drop_workspace(self.dev, s.cuda_stream)
        else:
            for i in range(1, max_new):
                if crosses(i):
                    stream = not stream
                self._step_eager(B, max_len, sampler, stream=stream)
                out[:, i] = self.tokens[:B]
        _lib.check_status(self.dev) if self.dev.type == "cuda" else None
        return out

    # ------------------------------------------------------------------ many sequences from one prefix
    _shared = None                       # (page ids, positions) of the prefix that the sequences of the running generation have in common

    def _shares(self, B: int, P: int) -> bool:
        """Whether the attention that reads a common prefix of ``P`` positions once beats ``decode_attention``, which reads it for each of
        ``B`` sequences (from the cache of the chip, while it fits), but is one launch. us in a graph, 32 positions behind the prefix,
        decode / shared. 32 / 8 heads of 128: 2 x 64 5.3 / 8.3, 2 x 256 9.9 / 8.8, 2 x 2048 11.2 / 11.0, 16 x 64 7.1 / 11.4, 16 x 256 13.4 /
        12.3, 64 x 256 22.8 / 18.3, 16 x 8192 82.1 / 19.7, 64 x 8192 305 / 40.6; 16 / 8 heads: 2 x 256 8.1 / 8.7, 16 x 256 11.2 / 12.0, 2 x
        512 8.9 / 8.9, 16 x 512 14.0 / 12.2; 8 / 1 heads: 2 x 256 13.4 / 11.0, 4 x 8192 13.6 / 14.4, 64 x 8192 48.0 / 24.7. Heads of 64, one
        or three query heads a kv head: 16 / 16 2 x 2048 11.2 / 11.4, 4 x 1024 10.3 / 11.0, 8 x 1024 13.9 / 11.6, 4 x 2048 14.5 / 11.5, 64 x
        512 29.5 / 30.5, 64 x 1024 51.8 / 35.2; 12 / 4 4 x 1024 9.2 / 10.3, 8 x 1024 11.5 / 10.3, 32 x 512 11.0 / 12.2.

        Far behind a short prefix both read about the same, and a generation that grows to there keeps what it began with. Prefix + own
        positions, 32 / 8 heads of 128: 2 x 256 + 2048 11.2 / 12.7, 2 x 1024 + 8192 17.8 / 18.2, 4 x 256 + 8192 28.5 / 31.5, 16 x 256 + 2048
        31.8 / 31.2, 16 x 1024 + 8192 92.7 / 101.9, 64 x 1024 + 8192 345 / 320, 4 x 4096 + 8192 36.2 / 38.2, 16 x 4096 + 8192 120 / 92; 4 / 1
        heads 4 x 1024 + 8192 12.0 / 15.4, 64 x 1024 + 8192 51.7 / 50.0; 16 / 4 heads of 64 4 x 1024 + 8192 21.8 / 19.3, 16 x 1024 + 8192 40.6 /
        51.7, 64 x 1024 + 8192 135 / 98."""
        if self.cache.page % 8:                        # which the kernel does not take
            return False
        if self.cfg.head_dim == 128:
            return B > 1 and P >= (256 if self.H >= 4 * self.Hkv else 512)
        return P >= 1024 and (B - 1) * P >= 4096

    def generate_shared(self, prefix: torch.Tensor, suffixes, max_new: int, params: SamplingParams | None = None, seed: int = 0):
        """Generation for sequences that begin alike. ``prefix`` [P] goes through the model once, and its pages of the cache are shared;
        ``suffixes`` is how many samples of it are wanted, or what each sequence has behind it: a matrix [B, S], or a list of B vectors of
        any lengths, empty ones too. Sequence b samples from the stream seeded with ``seed + b``. Returns int64 [B, max_new].

        The same tokens as ``generate`` on the whole prompts, but for roundings (another kernel reads the prefix)."""
        params = params or SamplingParams()
        if prefix.dim() > 1 and prefix.shape[-1] != prefix.numel():
            raise ValueError("one prefix")
        prefix = prefix.reshape(-1).to(self.dev)
        P = prefix.numel()
        if isinstance(suffixes, int):
            suffixes = [prefix[:0]] * suffixes
        suffixes = [torch.as_tensor(s).reshape(-1).to(self.dev, prefix.dtype) for s in suffixes]
        B, lens = len(suffixes), [s.numel() for s in suffixes]
        if B < 1 or P < 1 or max_new < 1:
            raise ValueError("a prefix, one sequence and one new token at least")
        longest = P + max(lens)
        if B > self.max_batch or longest + max_new > self.max_seq:
            raise ValueError("request exceeds the engine's max_batch / max_seq")
        cache, dev = self.cache, self.dev
        if longest > P and dev.type == "cuda" and cache.page % 8:
            raise ValueError("suffixes need a cache with pages of a multiple of 8")
        for b in range(B):                             # pages that another generation has left
            if cache.owned[b]:
                cache.release(b)
        logits = self.prefill(prefix[None]).clone()
        cache.fork(0, range(1, B), P)
        for b in range(B):
            cache.reserve(b, P + lens[b] + max_new)
        cache.commit()
        greedy = params.temperature <= 0.0 and params.repetition_penalty <= 1.0
        shared = (cache.block_table[0, :P // cache.page].clone(), P)
        logits = self._extend(suffixes, lens, P, shared, logits.expand(B, -1))
        sampler = None
        if greedy:
            D.argmax_rows(logits, out_tokens=self.tokens[:B])
        else:
            sampler = DeviceSampler(params, B, self.cfg.vocab_size, [seed + b for b in range(B)], dev, history_len=longest + max_new)
            sampler.history[:, :P] = prefix
            for b, s in enumerate(suffixes):
                sampler.history[b, P:P + lens[b]] = s
            sampler.n_hist.copy_(torch.tensor([P + n for n in lens], dtype=torch.int32))
            sampler.sample(logits, out_tokens=self.tokens[:B])
            sampler.push(self.tokens[:B])
        cache.seq_len[:B] = torch.tensor([P + n for n in lens], dtype=torch.int32, device=dev)
        # That attention reads pages in bf16; over 8 bits each sequence reads the prefix, from the cache of the chip while it fits. us for the shared
        # attention over bf16 / each sequence over 8 bits, 32 / 8 heads of 128: 2 x 2048 11.0 / 10.7, 16 x 1024 13.2 / 9.5, 16 x 8192 20.1 / 42.9, 64 x
        # 1024 24.4 / 28.0, 64 x 8192 40.3 / 148; 16 / 4 heads of 64: 16 x 1024 10.7 / 6.9, 16 x 8192 14.8 / 17.3, 64 x 1024 16.3 / 11.3, 64 x 8192
        # 26.8 / 48.8.
        self._shared = shared if self.kv is None and self._shares(B, P) else None
        try:
            return self._decode_steps(B, longest, max_new, sampler)
        finally:
            self._shared = None

    def _extend(self, suffixes, lens, P, shared, logits):
        """The layers over what the sequences have behind the prefix, all in one pass; returns their last positions' logits [B, V], those
        given where a sequence has nothing."""
        B, cache, dev = len(lens), self.cache, self.dev
        out = self.logits[:B]
        out.copy_(logits)
        if sum(lens) == 0:
            return out
        tok = torch.cat(suffixes)
        n = torch.tensor(lens, dtype=torch.int32)
        ends = torch.cat([n[:1] * 0, n.cumsum(0, dtype=torch.int32)])
        seq_of = torch.arange(B, dtype=torch.int32).repeat_interleave(n.long())
        pos = torch.arange(tok.numel(), dtype=torch.int32) - ends[:-1].repeat_interleave(n.long()) + P
        seq_of, pos, cu, total = seq_of.to(dev), pos.to(torch.int32).to(dev), ends.to(dev), (n + P).to(dev)
        table, (prefix_table, _), pool = cache.block_table[:B], shared, cache.pools.__getitem__
        if self.kv is not None:
            # the attention over runs of rows reads bf16: a layer's pages of these sequences are read back, under numbers of their own
            pages = [cache.owned[b][:-(-(P + k) // cache.page)] for b, k in enumerate(lens)]
            number = {page: i for i, page in enumerate(dict.fromkeys(sum(pages, [])))}
            rows = torch.zeros((B, cache.max_blocks), dtype=torch.int32)
            for b, ids in enumerate(pages):
                rows[b, :len(ids)] = torch.tensor([number[page] for page in ids], dtype=torch.int32)
            table = rows.to(dev)
            prefix_table = table[0, :P // cache.page].contiguous()
            ids = torch.tensor(list(number), dtype=torch.int32, device=dev)
            back = torch.empty((len(number), 2, self.Hkv, cache.page, self.cfg.head_dim), dtype=BF, device=dev)

            def pool(li):
                return Q.read_pages(cache.pools[li], ids, out=back)
        x = self._prompt_layers(tok, seq_of, pos, lambda li, qkv: paged.shared_prefix_attention(
            qkv, pool(li), table, cache.page, total, prefix_table, P, self.H, self.Hkv, self.cfg.head_dim, cu_q=cu, max_len=P + max(lens)),
            (total, cu))
        some = [b for b in range(B) if lens[b]]
        last = x[torch.tensor([int(ends[b + 1]) - 1 for b in some], device=dev)].contiguous()
        got = torch.empty((len(some), out.shape[1]), dtype=out.dtype, device=dev)
        self._head(last, got, rms_weight=self.rms_final)
        out[torch.tensor(some, device=dev)] = got
        return out


_OWN_PRODUCTS = (InferenceEngine._linear, InferenceEngine._proj_out, InferenceEngine._gated)
# Products whose feed-forward may take gate/up through ``_gated``: a class that replaces one of them enters its own here.
GATED_PRODUCTS = {_OWN_PRODUCTS}


def teacher_forced_logits(engine: "InferenceEngine", prompts: torch.Tensor, tokens: torch.Tensor) -> torch.Tensor:
    """Logits ``[B, n, V]`` (fp32) of ``engine`` when it is FED ``tokens [B, n]`` after ``prompts`` instead of its own
    arg-max: step i sees the prompt and tokens[:, :i+1]. Two engines given the same tokens can then be compared
    step by step, which greedy generation does not allow once one near-tie flips a token (eager steps, no graph)."""
    B, P = prompts.shape
    n = tokens.shape[1]
    for b in range(B):
        if engine.cache.owned[b]:
            engine.cache.release(b)
    engine.prefill(prompts)
    for b in range(B):
        engine.cache.reserve(b, P + n + 1)
    engine.cache.commit()
    engine._seq_of = torch.arange(engine.max_batch, dtype=torch.int32, device=engine.dev)
    engine._len_plus1 = torch.zeros(engine.max_batch, dtype=torch.int32, device=engine.dev)
    engine._generated = None
    out = []
    tok = tokens.to(engine.dev)
    for i in range(n):
        engine.tokens[:B] = tok[:, i]
        engine._step_eager(B, P + n + 1, want_logits=True, stream=engine._streams(B, P + i + 1))
        out.append(engine.logits[:B].float().clone())
    return torch.stack(out, 1)


def reference_generate(model: GQADecoder, prompts: torch.Tensor, max_new: int) -> torch.Tensor:
    """Full-recompute greedy decoding through the training forward (the naive path the cached
    decoder must agree with token for token: scirust-sciagent/tests/cuda_parity.rs:184)."""
    toks = prompts.clone()
    out = []
    with torch.no_grad():
        for _ in range(max_new):
            logits = model(toks)
            nxt = torch.stack([torch.tensor(D._nan_safe_argmax(r.float().cpu())) for r in logits]).to(toks.device)
            out.append(nxt)
            toks = torch.cat([toks, nxt[:, None]], 1)
    return torch.stack(out, 1)
