"""A paged KV cache held in 8 bits, as timed cases: keys and values quantised as they are written, attention of single tokens over the
codes, and pages read back in bf16.

A cache is a pair of codes ``[n_blocks, 2, Hkv, page, dh]`` (int8 or float8_e4m3fn; keys, then values) and scales ``[n_blocks, 2, Hkv,
page / block]`` (fp32): ``block`` consecutive positions of a head have one scale, and a value is its code times that. Writing takes as
scale the smallest power of two that the largest magnitude needs (int8: 2^(k-6) where that lies in [2^k, 2^(k+1)); e4m3: the least with
448 times it no smaller); a block that holds positions already keeps the larger of its scale and the new one, and what it holds is
rounded to the new steps.

Head counts are those of the configurations of ``models/sciagent.py`` (350m, llama3_8b, one of eight tensor-parallel shards of the
latter) and two generic ones; all inputs are random. ``own`` chooses between the framework's operators and the same mathematics in
elementary torch operations."""
import math

import torch

own = False

BF = torch.bfloat16
F64 = torch.float64
DEV = "cuda"
# query heads, key/value heads, head dimension
HEADS = {"350m": (16, 4, 64), "llama3_8b": (32, 8, 128), "llama3_8b_tp8": (4, 1, 128), "own_heads": (12, 12, 64), "one_head": (20, 1, 128)}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
LIMIT = {"int8": 127.0, "e4m3": 448.0}
THETA = 500000.0


def listed():
    return [
        # one decoded token of one user of a small model: the smallest call, bound by latency
        dict(name="step_350m_1", kind="write", dims="350m", codes="int8", page=64, block=16, batch=1, held=100, new=1, rope=True),
        # one decoded token of each sequence of the benchmark's largest batch
        dict(name="step_8b_64", kind="write", dims="llama3_8b", codes="int8", page=64, block=16, batch=64, held=2048, new=1, rope=True),
        # a prompt of the benchmark's length
        dict(name="prompt_8b_1", kind="write", dims="llama3_8b", codes="int8", page=64, block=16, batch=1, held=0, new=2048, rope=True),
        # next turns of conversations, prefilled together: ragged runs that begin and end inside a block; keys are rotated already
        dict(name="turns_8b_16", kind="write", dims="llama3_8b", codes="e4m3", page=16, block=8, batch=16, held=300, new=700, rope=False),
        # the attention of one user of a small model at the start of an answer: the smallest call
        dict(name="attend_350m_1", kind="attend", dims="350m", codes="int8", page=64, block=16, batch=1, length=200),
        # a chat of a few users on one of eight shards of an 8B model, larger blocks
        dict(name="attend_tp8_9", kind="attend", dims="llama3_8b_tp8", codes="e4m3", page=128, block=64, batch=9, length=5003),
        # the benchmark's batch of 16, small pages
        dict(name="attend_8b_16_page16", kind="attend", dims="llama3_8b", codes="e4m3", page=16, block=16, batch=16, length=2304),
        # and its largest batch
        dict(name="attend_8b_64", kind="attend", dims="llama3_8b", codes="int8", page=64, block=16, batch=64, length=2048),
        # one very long document
        dict(name="attend_8b_1_long", kind="attend", dims="llama3_8b", codes="int8", page=64, block=16, batch=1, length=131072),
        # twenty query heads over one key/value head: more rows than a tile takes
        dict(name="attend_one_head_32", kind="attend", dims="one_head", codes="int8", page=64, block=32, batch=32, length=4099),
        # a short prompt's pages, for a prefill that goes on behind it
        dict(name="read_350m_3", kind="read", dims="350m", codes="int8", page=64, block=16, pages=3),
        # the pages of a batch of long contexts
        dict(name="read_8b_1000", kind="read", dims="llama3_8b", codes="e4m3", page=64, block=16, pages=1000),
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
    dims = rng.choice(["350m", "llama3_8b", "llama3_8b", "llama3_8b_tp8", "own_heads", "one_head"])
    page = rng.choice([8, 16, 32, 64, 64, 128])
    block = rng.choice([b for b in (8, 16, 32, 64) if b <= page])
    base = dict(dims=dims, codes=rng.choice(["int8", "e4m3"]), page=page, block=block)
    kind = rng.choice(["write", "write", "attend", "attend", "attend", "read"])
    if kind == "write":
        held = rng.choice([0, _log_int(rng, 1, 4096)])
        if rng.random() < 0.4:
            return dict(base, kind=kind, batch=_log_int(rng, 1, 64), held=held, new=1, rope=rng.random() < 0.7)
        new = _log_int(rng, 2, 4096)
        return dict(base, kind=kind, batch=_log_int(rng, 1, max(1, min(64, 8192 // new))), held=held, new=new, rope=rng.random() < 0.5)
    if kind == "attend":
        length = _log_int(rng, 1, 131072)
        return dict(base, kind=kind, batch=_log_int(rng, 1, max(1, min(64, 131072 // length))), length=length)
    return dict(base, kind=kind, pages=_log_int(rng, 1, 1000))


# ---------------------------------------------------------------------------------------------- inputs
def _pool(g, case, n):
    """Codes and scales of n pages as a cache holds them: magnitudes of a block reach its largest code or nearly so."""
    _, Hkv, dh = HEADS[case["dims"]]
    page, block = case["page"], case["block"]
    x = torch.randn((n, 2, Hkv, page, dh), generator=g, device=DEV, dtype=BF)
    exponent = torch.randint(-1, 2, (n, 2, Hkv, page // block), generator=g, device=DEV).float()
    if case["codes"] == "int8":
        return (x * 24).round().clamp_(-127, 127).to(torch.int8), torch.exp2(exponent - 5)
    return (x * 96).clamp_(-448, 448).to(torch.float8_e4m3fn), torch.exp2(exponent - 7)


def _lengths(case, seed):
    """Positions that each sequence holds before, and new tokens. Of a write both are the same for every seed, so that the answers are of
    one shape; the first sequence has the most."""
    B = case["batch"]
    if case["kind"] == "write":
        g = torch.Generator().manual_seed(1000 * B + case["new"] + 7 * case["held"])
        held = torch.randint(case["held"] // 2, case["held"] + 1, (B,), generator=g)
        new = torch.randint((case["new"] + 1) // 2, case["new"] + 1, (B,), generator=g)
        held[0], new[0] = case["held"], case["new"]
        return held.tolist(), new.tolist()
    g = torch.Generator().manual_seed(int(seed))
    length = torch.randint((case["length"] + 1) // 2, case["length"] + 1, (B,), generator=g)
    length[0] = case["length"]
    return length.tolist(), [1] * B


def _inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    H, Hkv, dh = HEADS[case["dims"]]
    page = case["page"]
    if case["kind"] == "read":
        n = case["pages"] + 5
        codes, scales = _pool(g, case, n)
        return dict(codes_of=codes, scales=scales, pages_read=torch.randperm(n, generator=g, device=DEV)[:case["pages"]].int())
    B = case["batch"]
    held, new = _lengths(case, seed)
    total = [h + n for h, n in zip(held, new)] if case["kind"] == "write" else held
    own_pages = [(t + page - 1) // page for t in total]
    n = sum(own_pages) + 3
    order = torch.randperm(n, generator=g, device=DEV).int()
    table = torch.zeros((B, max(own_pages)), dtype=torch.int32, device=DEV)
    at = 0
    touched = []
    for b, k in enumerate(own_pages):
        table[b, :k] = order[at:at + k]
        touched.append(order[at + held[b] // page:at + k])
        at += k
    codes, scales = _pool(g, case, n)
    rows = sum(new)
    # the projection's output; a few channels of the keys are several times as large as the others, as rotary models have them
    qkv = torch.randn((rows, (H + 2 * Hkv) * dh), generator=g, device=DEV)
    qkv[:, H * dh + 3:(H + Hkv) * dh:dh] *= 4
    s = dict(qkv=(qkv * 1.5).to(BF), codes_of=codes, scales=scales, table=table,
             seq_len=torch.tensor(total, dtype=torch.int32, device=DEV), max_len=max(total))
    if case["kind"] == "write":
        s["cu_q"] = torch.tensor([0] + new).cumsum(0).to(torch.int32).to(DEV) if case["new"] > 1 else None
        s["touched"] = torch.cat(touched).contiguous()
        if case["rope"]:
            inverse = THETA ** (-torch.arange(0, dh, 2, dtype=F64) / dh)
            angle = torch.arange(max(total), dtype=F64)[:, None] * inverse
            s["cos"], s["sin"] = angle.cos().float().to(DEV), angle.sin().float().to(DEV)
    return s


def prepare(case, seed):
    s = dict(case)
    s.update(_inputs(case, seed))
    return s


# ---------------------------------------------------------------------------------------------- passes
def _values(codes, scales, block):
    return codes.float() * scales.repeat_interleave(block, -1)[..., None]


def _plain_write(s):
    H, Hkv, dh = HEADS[s["dims"]]
    page, block, codes, scales = s["page"], s["block"], s["codes_of"], s["scales"]
    qkv = s["qkv"]
    n, B = qkv.shape[0], s["batch"]
    row = torch.arange(n, device=DEV)
    if s["cu_q"] is None:
        seq, pos = row, s["seq_len"].long() - 1
    else:
        seq = torch.searchsorted(s["cu_q"][1:].long(), row, right=True)
        pos = s["seq_len"].long()[seq] - s["cu_q"].long()[seq + 1] + row
    if s["rope"]:
        x = qkv[:, :(H + Hkv) * dh].float().view(n, H + Hkv, dh // 2, 2)
        c, sn = s["cos"][pos][:, None], s["sin"][pos][:, None]
        x = torch.stack((x[..., 0] * c - x[..., 1] * sn, x[..., 0] * sn + x[..., 1] * c), -1)
        qkv = torch.cat((x.view(n, -1).to(BF), qkv[:, (H + Hkv) * dh:]), 1)
    kv = qkv[:, H * dh:].float().view(n, 2, Hkv, dh)
    blocks = page // block
    at = s["table"].long()[seq, pos // page]                                          # page of a row
    place = at * blocks + pos % page // block                                         # its block among all pages' blocks
    flat = scales.permute(0, 3, 1, 2).reshape(-1, 2, Hkv)
    largest = torch.zeros_like(flat).index_reduce_(0, place, kv.abs().amax(-1), "amax")
    k = torch.frexp(largest.clamp_min(2.0 ** -90))[1].float() - 1                      # largest lies in [2^k, 2^(k+1))
    if s["codes"] == "int8":
        need = torch.exp2(k - 6)
    else:
        need = torch.exp2(k - 8 + (largest > 1.75 * torch.exp2(k)))
    first = torch.full((flat.shape[0],), block, device=DEV, dtype=torch.long).index_reduce_(0, place, pos % block, "amin")
    kept = first[:, None, None]
    new = torch.where(kept == block, flat, torch.where(kept == 0, need, torch.maximum(flat, need)))
    ratio = (flat / new).view(-1, blocks, 2, Hkv).permute(0, 2, 3, 1)
    scales.copy_(new.view(-1, blocks, 2, Hkv).permute(0, 2, 3, 1))

    def to_codes(x):
        x = x.round() if s["codes"] == "int8" else x
        return x.clamp(-LIMIT[s["codes"]], LIMIT[s["codes"]]).to(codes.dtype)

    t = s["touched"].long()
    old = codes[t]
    before = (torch.arange(page, device=DEV).view(blocks, block) % block < first.view(-1, blocks, 1)[t]) & (first.view(-1, blocks, 1)[t] < block)
    again = to_codes(old.float() * ratio[t].repeat_interleave(block, -1)[..., None])
    bits = torch.where(before.view(-1, 1, 1, page, 1), again.view(torch.int8), old.view(torch.int8))
    codes.view(torch.int8)[t] = bits
    codes.view(torch.int8)[at, :, :, pos % page] = to_codes(kv / new[place][..., None]).view(torch.int8)
    return [qkv, _values(codes[t], scales[t], block).to(BF)]


def _plain_attend(s):
    H, Hkv, dh = HEADS[s["dims"]]
    B = s["batch"]
    kv = _values(s["codes_of"][s["table"].long()], s["scales"][s["table"].long()], s["block"])       # [B, pages, 2, Hkv, page, dh]
    k, v = kv.permute(2, 0, 3, 1, 4, 5).reshape(2, B, Hkv, -1, dh)
    q = s["qkv"][:, :H * dh].float().view(B, Hkv, H // Hkv, dh) / math.sqrt(dh)
    score = q @ k.transpose(2, 3)
    hidden = torch.arange(k.shape[2], device=DEV) >= s["seq_len"][:, None]
    score = score.masked_fill(hidden[:, None, None], float("-inf"))
    e = torch.exp(score - score.amax(-1, keepdim=True))
    return ((e @ v) / e.sum(-1, keepdim=True)).reshape(B, H * dh).to(BF)


def run(state):
    s = state
    if own:
        from scirust_b200.ops import quantized_kv as Q
        pool = Q.QuantPool(s["codes_of"], s["scales"])
        if s["kind"] == "read":
            return Q.read_pages(pool, s["pages_read"])
        H, Hkv, dh = HEADS[s["dims"]]
        if s["kind"] == "attend":
            return Q.decode_attention(s["qkv"], pool, s["table"], s["seq_len"], H, Hkv, dh, max_len=s["max_len"])
        if s["rope"]:
            qkv = s["qkv"].clone()                                                    # it is rotated in place
            Q.rope_kv_append(qkv, H, Hkv, dh, s["cos"], s["sin"], pool, s["table"], s["seq_len"], cu_q=s["cu_q"])
        else:
            qkv = s["qkv"]
            Q.kv_append(qkv, H, Hkv, dh, pool, s["table"], s["seq_len"], cu_q=s["cu_q"])
        return [qkv, Q.read_pages(pool, s["touched"])]
    if s["kind"] == "write":
        return _plain_write(s)
    if s["kind"] == "attend":
        return _plain_attend(s)
    t = s["pages_read"].long()
    return _values(s["codes_of"][t], s["scales"][t], s["block"]).to(BF)


# ---------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    H, Hkv, dh = HEADS[case["dims"]]
    page, block = case["page"], case["block"]
    page_codes, page_scales = 2 * Hkv * page * dh, 2 * Hkv * (page // block) * 4
    if case["kind"] == "read":
        return {"bytes": case["pages"] * (3 * page_codes + page_scales), "flops": case["pages"] * page_codes}
    held, new = _lengths(case, 0)
    if case["kind"] == "write":
        rows = sum(new)
        # k and v are read and their codes written; with the rotation q is read too, and q and k are written, without it rows stay as they
        # are. The pages written to are read back: what was there before as codes (the new ones are at hand), all of it written in bf16.
        pages = sum((h + n + page - 1) // page - h // page for h, n in zip(held, new))
        moved = rows * dh * (2 * Hkv * 3 + (2 * H + 2 * (H + Hkv)) * case["rope"])
        return {"bytes": moved + pages * (2 * page_codes + page_scales) + max(0, pages * page_codes - rows * dh * 2 * Hkv),
                "flops": rows * dh * ((H + Hkv) * 3 * case["rope"] + 2 * Hkv * 4)}
    # sequences behind the first hold three quarters of its length in the mean
    tokens = case["length"] * (1 + 0.75 * (case["batch"] - 1))
    return {"bytes": tokens * (page_codes + page_scales) / page + case["batch"] * 4 * H * dh, "flops": 4 * H * dh * tokens}


# ---------------------------------------------------------------------------------------------- 64-bit statement
def _power(k):
    """2^k for whole numbers, without the error of an exponential."""
    return torch.ldexp(torch.ones_like(k, dtype=F64), k)


def _exact_codes(x, kind):
    """The values nearest to x that a code of this type has, in steps of its exponent (e4m3: three bits behind the leading one, and none
    finer than 2^-9); ties to even."""
    if kind == "int8":
        return torch.round(x).clamp(-127, 127)
    step = _power(torch.frexp(x.abs().clamp_min(2.0 ** -6))[1] - 4)
    return (torch.round(x / step) * step).clamp(-448, 448)


def exact(case, seed):
    s = _inputs(case, seed)
    H, Hkv, dh = HEADS[case["dims"]]
    page, block, kind = case["page"], case["block"], case["codes"]
    if case["kind"] == "read":
        t = s["pages_read"].long()
        return (s["codes_of"][t].to(F64).view(len(t), 2, Hkv, -1, block, dh) * s["scales"][t].to(F64)[..., None, None]).view(-1, 2, Hkv, page, dh)
    if case["kind"] == "attend":
        out = []
        for b, length in enumerate(s["seq_len"].tolist()):
            pos = torch.arange(length, device=DEV)
            at = s["table"][b].long()[pos // page]
            kv = s["codes_of"][at, :, :, pos % page].to(F64) * s["scales"][at, :, :, pos % page // block].to(F64)[..., None]
            q = s["qkv"][b, :H * dh].to(F64).view(Hkv, H // Hkv, dh)
            p = torch.softmax(torch.einsum("kgd,jkd->kgj", q, kv[:, 0]) * dh ** -0.5, -1)
            out.append(torch.einsum("kgj,jkd->kgd", p, kv[:, 1]).reshape(-1))
        return torch.stack(out)
    held, new = _lengths(case, seed)
    qkv = s["qkv"].to(F64)
    pos = torch.cat([torch.arange(h, h + n) for h, n in zip(held, new)]).to(DEV)
    if case["rope"]:
        x = torch.view_as_complex(qkv[:, :(H + Hkv) * dh].reshape(len(pos), H + Hkv, dh // 2, 2))
        turn = torch.complex(s["cos"].to(F64), s["sin"].to(F64))[pos][:, None]
        qkv = torch.cat((torch.view_as_real(x * turn).flatten(1), qkv[:, (H + Hkv) * dh:]), 1)
    kv = qkv[:, H * dh:].to(BF).to(F64).view(-1, 2, Hkv, dh)                          # what the cache is written from is in bf16
    out, at = [], 0
    for b, (h, n) in enumerate(zip(held, new)):
        p0 = h // page
        ids = s["table"][b, p0:(h + n + page - 1) // page].long()
        codes = s["codes_of"][ids].to(F64).permute(1, 2, 0, 3, 4).reshape(2, Hkv, -1, block, dh)       # by blocks of the run of pages
        scale = s["scales"][ids].to(F64).permute(1, 2, 0, 3).reshape(2, Hkv, -1)
        x = torch.zeros((2, Hkv, codes.shape[2] * block, dh), dtype=F64, device=DEV)
        x[:, :, h - p0 * page:h - p0 * page + n] = kv[at:at + n].permute(1, 2, 0, 3)
        place = torch.arange(x.shape[2], device=DEV).view(-1, block) + p0 * page
        fresh, old = ((place >= h) & (place < h + n))[..., None], (place < h)[..., None]
        x = x.view(codes.shape)
        top = x.abs().amax((-1, -2)).clamp_min(2.0 ** -90)
        need = _power(torch.frexp(top)[1] - 7)
        if kind == "e4m3":
            mantissa, power = torch.frexp(top / 448)                                  # the quotient is a power of two or far from one
            need = _power(power - (mantissa == 0.5).int())
        written, holds = fresh.any(1).view(-1), old.any(1).view(-1)
        to = torch.where(written, torch.where(holds, torch.maximum(need, scale), need), scale)
        codes = torch.where(old & written[:, None, None], _exact_codes(codes * (scale / to)[..., None, None], kind), codes)
        codes = torch.where(fresh, _exact_codes(x / to[..., None, None], kind), codes)
        values = (codes * to[..., None, None]).reshape(2, Hkv, -1, page, dh).permute(2, 0, 1, 3, 4)
        out.append(values)
        at += n
    return [qkv, torch.cat(out)]
