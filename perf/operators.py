"""Decoding many sequences from one prompt, as timed cases: the attention of a batch whose sequences share a prefix in the paged
cache, and the copies of cache pages behind forking and compacting sequences.

Head counts are those of the configurations of ``models/sciagent.py`` (350m, llama3_8b, and one of eight tensor-parallel shards of the
latter); all inputs are random. ``own`` chooses between the framework's operators and the same mathematics in elementary torch
operations."""
import math

import torch

own = False

BF = torch.bfloat16
F64 = torch.float64
DEV = "cuda"
# query heads, key/value heads, head dimension
HEADS = {"350m": (16, 4, 64), "llama3_8b": (32, 8, 128), "llama3_8b_tp8": (4, 1, 128)}


def listed():
    return [
        # four samples of a short prompt on a small model, at the start of the generation: the smallest call, bound by latency
        dict(name="samples_350m_4", kind="attend", dims="350m", batch=4, prefix=512, own=16, new=1, page=64),
        # one of eight shards of an 8B model, eight samples of a prompt of the benchmark's length
        dict(name="samples_tp8_8", kind="attend", dims="llama3_8b_tp8", batch=8, prefix=2048, own=256, new=1, page=64),
        # 16 samples of a 4k prompt; the prompt does not end with a page
        dict(name="samples_8b_16", kind="attend", dims="llama3_8b", batch=16, prefix=4000, own=256, new=1, page=64),
        # 33 requests behind a document, pages of 16 positions
        dict(name="document_8b_33_page16", kind="attend", dims="llama3_8b", batch=33, prefix=5003, own=512, new=1, page=16),
        # the benchmark's largest batch behind a long document
        dict(name="document_8b_64", kind="attend", dims="llama3_8b", batch=64, prefix=16384, own=512, new=1, page=64),
        # questions of up to 64 tokens, prefilled together behind a document: ragged runs of new tokens
        dict(name="questions_8b_16", kind="attend", dims="llama3_8b", batch=16, prefix=8192, own=64, new=64, page=64),
        # a few long continuations behind a shorter system prompt, on the small model
        dict(name="continuations_350m_4", kind="attend", dims="350m", batch=4, prefix=1000, own=700, new=700, page=64),
        # one forked sequence: a half-filled last page in each layer of the small model
        dict(name="fork_350m_1", kind="pages", dims="350m", layers=24, blocks=64, copies=1, fan=1, rows=17, page=64),
        # 16 forks of one prompt: its half-filled last page goes to 16 pages of each layer
        dict(name="fork_8b_16", kind="pages", dims="llama3_8b", layers=32, blocks=48, copies=16, fan=16, rows=40, page=64),
        # a cache is compacted: a third of its pages move
        dict(name="compact_8b", kind="pages", dims="llama3_8b", layers=8, blocks=384, copies=128, fan=1, rows=0, page=64),
        # the same with small pages of a shard
        dict(name="compact_tp8_page16", kind="pages", dims="llama3_8b_tp8", layers=32, blocks=1024, copies=301, fan=1, rows=0, page=16),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case; what would cost more than the largest listed one is drawn again."""
    largest = max(_cost(c) for c in listed())
    while True:
        case = _draw(rng)
        if _cost(case) <= largest:
            return case


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 6.5e12, w["flops"] / 1.6e15)        # seconds at a B200's memory and tensor-core rates


def _draw(rng):
    dims = rng.choice(["350m", "llama3_8b", "llama3_8b", "llama3_8b_tp8"])
    page = rng.choice([16, 32, 64, 64, 64, 128])
    if rng.random() < 0.7:
        if rng.random() < 0.65:
            return dict(kind="attend", dims=dims, batch=_log_int(rng, 2, 64), prefix=_log_int(rng, 100, 16384),
                        own=_log_int(rng, 1, 512), new=1, page=page)
        new = _log_int(rng, 2, 512)
        return dict(kind="attend", dims=dims, batch=_log_int(rng, 1, max(1, min(64, 1024 // new))), prefix=_log_int(rng, 100, 8192),
                    own=new + rng.choice([0, 0, rng.randint(1, 100)]), new=new, page=page)
    fan = rng.choice([1, 1, _log_int(rng, 2, 32)])
    copies = fan if fan > 1 else _log_int(rng, 1, 128)
    return dict(kind="pages", dims=dims, layers=rng.choice([8, 12, 24, 32]) if copies <= 32 else 8, blocks=2 * copies + rng.randint(1, 64),
                copies=copies, fan=fan, rows=rng.randint(1, page - 1) if fan > 1 or rng.random() < 0.3 else 0, page=page)


# ---------------------------------------------------------------------------------------------- inputs
def _lengths(case, seed):
    """Tokens behind the prefix and new tokens of each sequence: the first one has the most, the others anything below. The new
    tokens are the same for every seed, so that the answers are of one shape."""
    B = case["batch"]
    new = torch.randint(1, case["new"] + 1, (B,), generator=torch.Generator().manual_seed(1000 * B + case["new"]))
    new[0] = case["new"]
    g = torch.Generator().manual_seed(int(seed))
    tail = torch.randint(1, case["own"] + 1, (B,), generator=g)
    tail[0] = case["own"]
    return torch.maximum(tail, new).tolist(), new.tolist()


def _inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    H, Hkv, dh = HEADS[case["dims"]]
    page = case["page"]
    if case["kind"] == "pages":
        shape = (case["blocks"], 2, Hkv, page, dh)
        pools = [torch.randn(shape, generator=g, device=DEV, dtype=BF) for _ in range(case["layers"])]
        order = torch.randperm(case["blocks"], generator=g, device=DEV).int()
        n = case["copies"]
        src = order[:1].repeat(n) if case["fan"] > 1 else order[:n]
        return dict(pools=pools, src=src.contiguous(), dst=order[n:2 * n].contiguous())
    tail, new = _lengths(case, seed)
    B, P = case["batch"], case["prefix"]
    shared = P // page                                          # whole pages; what is behind them each sequence has for itself
    own_pages = [(P + t + page - 1) // page - shared for t in tail]
    total = shared + sum(own_pages) + 3
    order = torch.randperm(total, generator=g, device=DEV).int()
    prefix_table = order[:shared].contiguous()
    width = shared + max(own_pages)
    table = torch.zeros((B, width), dtype=torch.int32, device=DEV)
    at = shared
    for b, n in enumerate(own_pages):
        table[b, :shared] = prefix_table
        table[b, shared:shared + n] = order[at:at + n]
        at += n
    pool = torch.randn((total, 2, Hkv, page, dh), generator=g, device=DEV, dtype=BF)
    ends = torch.tensor([0] + new).cumsum(0)
    # the projection's output, of which attention takes the query heads
    qkv = (torch.randn((int(ends[-1]), (H + 2 * Hkv) * dh), generator=g, device=DEV) * 1.5).to(BF)
    return dict(q=qkv, pool=pool, table=table, prefix_table=prefix_table, tail=tail, new_rows=new,
                seq_len=torch.tensor([P + t for t in tail], dtype=torch.int32, device=DEV),
                cu_q=ends.to(torch.int32).to(DEV) if case["new"] > 1 else None, max_len=P + max(tail))


def prepare(case, seed):
    s = dict(case)
    s.update(_inputs(case, seed))
    if own and case["kind"] == "pages":
        from scirust_b200.ops import paged
        s["pools_handle"] = paged.PagePools(s["pools"])         # made once for a cache
    return s


# ---------------------------------------------------------------------------------------------- passes
def _softmax_part(q, k, v, mask=None):
    """q [heads, rows, dh], k and v [heads, keys, dh] in 32 bits: row maximum, sum of exponentials, weighted values."""
    s = q @ k.transpose(1, 2)
    if mask is not None:
        s = s.masked_fill(mask, float("-inf"))
    m = s.amax(-1, keepdim=True)
    e = torch.exp(s - m)
    return m, e.sum(-1, keepdim=True), e @ v


def _plain_attend(s):
    H, Hkv, dh = HEADS[s["dims"]]
    G, n, page = H // Hkv, s["q"].shape[0], s["page"]
    q = s["q"][:, :H * dh].float().view(n, Hkv, G, dh).transpose(0, 1) / math.sqrt(dh)        # [Hkv, n, G, dh]

    def keys_values(blocks):
        kv = s["pool"][blocks].float()                                                        # [pages, 2, Hkv, page, dh]
        return kv.permute(1, 2, 0, 3, 4).reshape(2, Hkv, -1, dh)

    shared = s["prefix_table"].numel() * page
    if shared:
        k, v = keys_values(s["prefix_table"].long())
        mp, lp, op = _softmax_part(q.reshape(Hkv, n * G, dh), k, v)
    parts, at = [], 0
    for b, (tail, new) in enumerate(zip(s["tail"], s["new_rows"])):
        length = s["prefix"] + tail - shared
        k, v = keys_values(s["table"][b, shared // page:(shared + length + page - 1) // page].long())
        k, v = k[:, :length], v[:, :length]
        last = torch.arange(length - new, length, device=k.device).repeat_interleave(G)       # the row's own position
        mask = torch.arange(length, device=k.device) > last[:, None] if new > 1 else None
        parts.append(_softmax_part(q[:, at:at + new].reshape(Hkv, new * G, dh), k, v, mask))
        at += new
    m, l, o = (torch.cat(p, 1) for p in zip(*parts))
    if shared:
        top = torch.maximum(m, mp)
        w, wp = torch.exp(m - top), torch.exp(mp - top)
        l, o = l * w + lp * wp, o * w + op * wp
    return (o / l).view(Hkv, n, G, dh).transpose(0, 1).reshape(n, H * dh).to(BF)


def run(state):
    s = state
    if own:
        from scirust_b200.ops import paged
        if s["kind"] == "pages":
            paged.copy_pages(s["pools_handle"], s["src"], s["dst"], rows=s["rows"] or None)
            return s["pools"]
        H, Hkv, dh = HEADS[s["dims"]]
        return paged.shared_prefix_attention(s["q"], s["pool"], s["table"], s["page"], s["seq_len"], s["prefix_table"], s["prefix"],
                                             H, Hkv, dh, cu_q=s["cu_q"], max_len=s["max_len"])
    if s["kind"] == "pages":
        rows = s["rows"] or s["page"]
        src, dst = s["src"].long(), s["dst"].long()
        for p in s["pools"]:
            p[dst, :, :, :rows] = p[src, :, :, :rows]
        return s["pools"]
    return _plain_attend(s)


# ---------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    H, Hkv, dh = HEADS[case["dims"]]
    page = case["page"]
    if case["kind"] == "pages":
        size = 2 * Hkv * (case["rows"] or page) * dh * 2
        read = 1 if case["fan"] > 1 else case["copies"]
        return {"bytes": case["layers"] * size * (read + case["copies"]), "flops": 0}
    B, P = case["batch"], case["prefix"]
    shared = P // page * page
    # sequences behind the first have half the longest tail and half the longest run of new tokens in the mean
    new = case["new"] + (B - 1) * (1 + case["new"]) / 2
    tail = case["own"] + (B - 1) * (1 + case["own"]) / 2
    keys = shared + B * (P - shared) + tail
    pairs = new * P + new * tail / B - (new * new / B - new) / 2
    return {"bytes": 4 * Hkv * dh * keys + 4 * new * H * dh, "flops": 4 * H * dh * pairs}


# ---------------------------------------------------------------------------------------------- 64-bit statement
def exact(case, seed):
    s = _inputs(case, seed)
    H, Hkv, dh = HEADS[case["dims"]]
    page = case["page"]
    if case["kind"] == "pages":
        origin = torch.arange(case["blocks"], device=DEV)
        origin[s["dst"].long()] = s["src"].long()
        rows = case["rows"] or page
        taken = (torch.arange(page, device=DEV) < rows)[:, None]
        return [torch.where(taken, p[origin].to(F64), p.to(F64)) for p in s["pools"]]
    out, at = [], 0
    for b, (tail, new) in enumerate(zip(s["tail"], s["new_rows"])):
        length = case["prefix"] + tail
        pos = torch.arange(length, device=DEV)
        kv = s["pool"][s["table"][b].long()[pos // page], :, :, pos % page].to(F64)           # [length, 2, Hkv, dh]
        q = s["q"][at:at + new, :H * dh].to(F64).reshape(new, Hkv, H // Hkv, dh)
        limit = torch.arange(length - new + 1, length + 1, device=DEV)
        score = torch.einsum("tkgd,jkd->tkgj", q, kv[:, 0]) * dh ** -0.5
        score = torch.where(pos < limit[:, None, None, None], score, -math.inf)
        out.append(torch.einsum("tkgj,jkd->tkgd", torch.softmax(score, -1), kv[:, 1]).reshape(new, H * dh))
        at += new
    return torch.cat(out)
