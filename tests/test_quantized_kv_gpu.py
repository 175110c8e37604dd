"""Operators on a paged KV cache in 8 bits on the GPU: what is written against the statement, to the bit, attention against 64 bits."""
import math

import pytest
import torch

from scirust_b200 import ops
from scirust_b200.ops import _lib, quantized_kv as Q

pytestmark = pytest.mark.gpu
BF, F64 = torch.bfloat16, torch.float64
DEV = "cuda"
KINDS = ["int8", "e4m3"]
CU = "cu_q"


@pytest.fixture(autouse=True)
def _poisoned(monkeypatch):
    """Workspaces and answers begin as NaN and between fences, so that a part which is read and was not written shows."""
    monkeypatch.setattr(_lib, "DEBUG_POISON", True)
    yield
    torch.cuda.synchronize()
    _lib.check_canaries()


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def bits(t):
    return t.contiguous().view({1: torch.int8, 2: torch.int16, 4: torch.int32}[t.element_size()])


def random_pool(n, Hkv, page, dh, kind, block, seed=0):
    """A pool as earlier writes leave it: codes of all magnitudes, scales that are powers of two."""
    g = gen(seed)
    x = torch.randn((n, 2, Hkv, page, dh), generator=g, device=DEV)
    codes = (x * 40).round().clamp(-127, 127).to(torch.int8) if kind == "int8" else (x * 150).clamp(-448, 448).to(torch.float8_e4m3fn)
    scales = torch.exp2(torch.randint(-8, 0, (n, 2, Hkv, page // block), generator=g, device=DEV).float())
    return Q.QuantPool(codes, scales)


def on_cpu(pool):
    return Q.QuantPool(pool.codes.cpu(), pool.scales.cpu())


def tables(pages, seed=0, spare=3):
    """A table with as many pages a sequence as asked for, every page in one sequence; unused entries name no page."""
    order = torch.randperm(sum(pages) + spare, generator=gen(seed), device=DEV).int()
    table = torch.full((len(pages), max(max(pages), 1)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n]
        at += n
    return table, len(order)


# ---------------------------------------------------------------------------------------------------------------- writing
def write(kind, H, Hkv, dh, page, block, held, new, rope=True, cu=True, chunk=None, monkeypatch=None, seed=0, pad=8, first=0, scale=1.0):
    """One write on the GPU and by the statement on the CPU: rotated rows, codes and scales have to be the same bits."""
    if chunk is not None:
        monkeypatch.setattr(Q, "_chunk", lambda n, B, block: chunk)
    total = [h + n for h, n in zip(held, new)]
    table, n_pages = tables([-(-t // page) for t in total], seed)
    pool = random_pool(n_pages, Hkv, page, dh, kind, block, seed)
    lens = torch.tensor(total, dtype=torch.int32, device=DEV)
    n = first + sum(new) + (2 if cu else 0)                              # rows of no sequence in front and behind
    g = gen(seed + 1)
    x = torch.randn((n, (H + 2 * Hkv) * dh + pad), generator=g, device=DEV)
    x = (x * torch.exp2(torch.randint(-3, 4, (n, 1), generator=g, device=DEV).float()) * scale).to(BF)
    cu_q = (torch.tensor([0] + new).cumsum(0) + first).int().to(DEV) if cu else None
    other, y = on_cpu(pool), x.cpu()
    c = cu_q.cpu() if cu else None
    if rope:
        cos, sin = ops.rope_table(max(total) + 1, dh, 10000.0, DEV)
        Q.rope_kv_append(x, H, Hkv, dh, cos, sin, pool, table, lens, cu_q=cu_q)
        Q.rope_kv_append(y, H, Hkv, dh, cos.cpu(), sin.cpu(), other, table.cpu(), lens.cpu(), cu_q=c)
    else:
        Q.kv_append(x, H, Hkv, dh, pool, table, lens, cu_q=cu_q)
        Q.kv_append(y, H, Hkv, dh, other, table.cpu(), lens.cpu(), cu_q=c)
    assert torch.equal(bits(x.cpu()), bits(y))
    assert torch.equal(bits(pool.scales.cpu()), bits(other.scales))
    assert torch.equal(bits(pool.codes.cpu()), bits(other.codes))
    return pool


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H,Hkv,dh", [(16, 4, 64), (4, 1, 128), (3, 3, 64), (5, 5, 128), (0, 2, 128)])
def test_single_tokens(kind, H, Hkv, dh):
    held = [0, 1, 15, 16, 17, 63, 64, 100, 5]
    write(kind, H, Hkv, dh, 64, 16, held, [1] * len(held), cu=False)
    write(kind, H, Hkv, dh, 64, 16, held, [1] * len(held), cu=False, rope=False, scale=8.0)       # every block's scale grows


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page,block", [(8, 8), (16, 8), (32, 32), (64, 16), (64, 64), (128, 64), (192, 64)])
@pytest.mark.parametrize("chunk", [1, 4, 16])
def test_ragged_runs(kind, page, block, chunk, monkeypatch):
    held, new = [0, 3, 0, 61, 130, 7, 64], [1, 200, 64, 67, 2, 0, 129]
    write(kind, 4, 2, 128, page, block, held, new, chunk=chunk, monkeypatch=monkeypatch, first=3)
    write(kind, 6, 2, 64, page, block, held, new, rope=False, chunk=chunk, monkeypatch=monkeypatch, scale=16.0)


def test_many_sequences():
    """More than one step of the search for a row's sequence: 33 times 32 of them, empty ones among them."""
    g = torch.Generator().manual_seed(4)
    new = torch.randint(0, 4, (1056,), generator=g).tolist()
    held = torch.randint(0, 9, (1056,), generator=g).tolist()
    write("int8", 2, 1, 64, 8, 8, held, new)


def test_long_prompt():
    write("e4m3", 4, 2, 128, 64, 16, [0, 5], [3000, 1111])


@pytest.mark.parametrize("Hkv,dh", [(8, 64), (8, 128)])
def test_more_blocks_than_two_warps_each_would_pay_for(Hkv, dh):
    write("int8", 2, Hkv, dh, 64, 16, [7, 0], [2500, 700])


@pytest.mark.parametrize("kind", KINDS)
def test_writing_in_parts_agrees_where_blocks_are_whole(kind):
    """A prompt in pieces that end with blocks gives the same pool as the whole of it."""
    H, Hkv, dh, page, block = 4, 2, 64, 64, 16
    table, n = tables([4])
    x = torch.randn((200, (H + 2 * Hkv) * dh), generator=gen(0), device=DEV).to(BF)
    one, two = random_pool(n, Hkv, page, dh, kind, block), random_pool(n, Hkv, page, dh, kind, block)
    ends = lambda *e: torch.tensor(e, dtype=torch.int32, device=DEV)
    Q.kv_append(x, H, Hkv, dh, one, table, ends(200), cu_q=ends(0, 200))
    for a, b in ((0, 48), (48, 64), (64, 192), (192, 200)):
        Q.kv_append(x[a:b], H, Hkv, dh, two, table, ends(b), cu_q=ends(0, b - a))
    assert torch.equal(bits(one.codes), bits(two.codes)) and torch.equal(one.scales, two.scales)


@pytest.mark.parametrize("kind", KINDS)
def test_rows_without_a_place_stay(kind):
    """Rows in front of position 0, behind the table or the rotation's tables, of an empty slot, and ids outside the pool."""
    H, Hkv, dh, page, block = 2, 1, 128, 16, 16
    pool = random_pool(4, Hkv, page, dh, kind, block)
    kept = Q.QuantPool(pool.codes.clone(), pool.scales.clone())
    i = lambda *e: torch.tensor(e, dtype=torch.int32, device=DEV)
    x = torch.randn((14, (H + 2 * Hkv) * dh), generator=gen(1), device=DEV).to(BF)
    before = x.clone()
    cos, sin = ops.rope_table(40, dh, 10000.0, DEV)
    # 4 rows for 2 positions; a table of two pages and a length of 34; an empty slot; a page outside; one below; a length behind the rotation
    table = torch.stack([i(0, 1), i(2, 3), i(1, 1), i(4, 4), i(-1, 0), i(3, 3)])
    Q.rope_kv_append(x, H, Hkv, dh, cos, sin, pool, table, i(2, 34, 0, 2, 1, 2 ** 31 - 1), cu_q=i(0, 4, 8, 9, 11, 12, 14))
    turned = (x != before).any(1)
    # row 3 is position 1 and turns; position 0 does not; rows 4 and 5 are positions 30 and 31; row 10 position 1 of a sequence without a page
    assert turned.nonzero().flatten().tolist() == [3, 4, 5, 10]
    changed = (bits(pool.codes) != bits(kept.codes)).flatten(1).any(1)
    assert changed.tolist() == [True, False, False, True]
    assert torch.equal(pool.scales[[1, 2]], kept.scales[[1, 2]])
    assert torch.equal(bits(pool.codes[0, :, :, 2:]), bits(kept.codes[0, :, :, 2:]))


@pytest.mark.parametrize("kind", KINDS)
def test_not_finite(kind):
    H, Hkv, dh, page, block = 1, 2, 64, 32, 16
    table, n = tables([2])
    pool = random_pool(n, Hkv, page, dh, kind, block)
    x = torch.randn((40, (H + 2 * Hkv) * dh), generator=gen(1), device=DEV).to(BF)
    x[3, H * dh + 5] = math.inf
    x[20, -1] = math.nan
    x[33, H * dh + dh] = 3.4e38 if kind == "e4m3" else -math.inf
    i = lambda *e: torch.tensor(e, dtype=torch.int32, device=DEV)
    Q.kv_append(x, H, Hkv, dh, pool, table, i(40), cu_q=i(0, 40))
    bad = pool.scales[table[0].long()].isnan().nonzero().tolist()              # page, k or v, head, block
    assert bad == [[0, 0, 0, 0], [0, 1, 1, 1], [1, 0, 1, 0]]
    back = Q.read_pages(pool, table[0])
    assert torch.equal(back.isnan().view(2, 2, Hkv, 2, block * dh).all(-1), pool.scales[table[0].long()].isnan())
    # in a block that is not begun anew it stays, in one that is it goes
    Q.kv_append(x[:1], H, Hkv, dh, pool, table, i(10))
    assert bool(pool.scales[table[0, 0].long(), 0, 0, 0].isnan())
    Q.kv_append(x[:1], H, Hkv, dh, pool, table, i(1))
    assert not bool(pool.scales[table[0, 0].long(), 0, 0, 0].isnan())


# ---------------------------------------------------------------------------------------------------------------- reading back
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page,block,dh,Hkv", [(8, 8, 64, 1), (64, 16, 128, 8), (128, 64, 64, 3), (48, 16, 128, 5)])
def test_pages_read_back(kind, page, block, dh, Hkv):
    pool = random_pool(9, Hkv, page, dh, kind, block)
    ids = torch.tensor([3, 0, 8, 3, 9, -1, 7], dtype=torch.int32, device=DEV)                    # twice the same; two outside the pool
    want = pool.codes.to(F64) * pool.scales.to(F64).repeat_interleave(block, -1)[..., None]
    got = Q.read_pages(pool, ids)
    assert torch.equal(got[[0, 1, 2, 3, 6]].to(F64), want[[3, 0, 8, 3, 7]])                      # exact: powers of two
    assert not bool(got[4:6].any())
    out = torch.full((2, 2, Hkv, page, dh), math.nan, dtype=BF, device=DEV)
    assert Q.read_pages(pool, [5, 1], out=out) is out and torch.equal(out.to(F64), want[[5, 1]])
    # scales that are no powers of two: one rounding to fp32 and one to bf16
    odd = Q.QuantPool(pool.codes, pool.scales * 1.3)
    want = pool.codes.to(F64) * odd.scales.to(F64).repeat_interleave(block, -1)[..., None]
    assert bool(((Q.read_pages(odd, list(range(9))).to(F64) - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -23)).all())
    assert Q.read_pages(pool, []).shape[0] == 0


@pytest.mark.parametrize("kind", KINDS)
def test_many_pages_read_back(kind):
    pool = random_pool(9, 8, 64, 128, kind, 16)
    ids = torch.randint(-1, 10, (300,), generator=gen(1), device=DEV).int()
    got, known = Q.read_pages(pool, ids), (ids >= 0) & (ids < 9)
    want = (pool.codes.float() * pool.scales.repeat_interleave(16, -1)[..., None]).to(BF)        # exact
    assert torch.equal(got[known], want[ids[known].long()]) and not bool(got[~known].any())


# ---------------------------------------------------------------------------------------------------------------- attention
def batch(kind, H, Hkv, dh, page, block, lens, seed=0, pad=8, dirty=True):
    """A batch of sequences of these lengths. What lies behind a sequence's last position is the largest code, NaN where the type has one,
    and NaN as scale of blocks that hold no position."""
    table, n = tables([-(-t // page) for t in lens], seed)
    pool = random_pool(n, Hkv, page, dh, kind, block, seed)
    if dirty:
        b8 = pool.codes.view(torch.int8)
        used = torch.zeros(n, dtype=torch.bool, device=DEV)
        for b, length in enumerate(lens):
            if length % page:
                at = int(table[b, length // page])
                b8[at, :, :, length % page:] = 127
                pool.scales[at, :, :, -(-(length % page) // block):] = math.nan
            used[table[b, :-(-length // page)].long()] = True
        b8[~used] = 127
        pool.scales[~used] = math.nan
    q = (torch.randn((len(lens), H * dh + pad), generator=gen(seed + 1), device=DEV) * 1.5).to(BF)
    return dict(q=q, pool=pool, block_table=table, seq_len=torch.tensor(lens, dtype=torch.int32, device=DEV), H=H, Hkv=Hkv, dh=dh)


def statement(a, scale=None):
    """(o, bound): 64 bits, and how far an element may be off. A weight is rounded to fp16 (half a step of 2^-11, none finer than 2^-25 of
    2^-9 of the largest) and weighs v, the answer is rounded once to bf16; a score is a sum of dh products in 32 bits, each addition off by
    a step of 2^-23 of the sum of magnitudes, which the exponential passes on as a relative error of a weight and of their sum. With int8 codes
    a query is rounded to whole numbers where its largest element is at least 2^13 of them: half of one, 2^-14 of the largest, for each
    element, times the magnitude of the key's."""
    H, Hkv, dh, pool = a["H"], a["Hkv"], a["dh"], a["pool"]
    page, block = pool.codes.shape[3], pool.block
    scale = dh ** -0.5 if scale is None else scale
    B = a["q"].shape[0]
    o, bound = torch.zeros((B, Hkv, H // Hkv, dh), dtype=F64, device=DEV), torch.zeros((B, Hkv, H // Hkv, dh), dtype=F64, device=DEV)
    for b, length in enumerate(a["seq_len"].tolist()):
        if length <= 0:
            continue
        pos = torch.arange(length, device=DEV)
        at = a["block_table"][b].long()[pos // page]
        kv = pool.codes.view(torch.int8)[at, :, :, pos % page].view(pool.codes.dtype).to(F64) * pool.scales[at, :, :, pos % page // block].to(F64)[..., None]
        q = a["q"][b, :H * dh].to(F64).reshape(Hkv, H // Hkv, dh)
        s = torch.einsum("kgd,jkd->kgj", q, kv[:, 0]) * scale
        size = torch.einsum("kgd,jkd->kgj", q.abs(), kv[:, 0].abs()) * scale
        coarse = q.abs().amax(-1, keepdim=True) * 2.0 ** -14 if pool.codes.dtype is torch.int8 else torch.zeros_like(q[..., :1])
        p = torch.softmax(s, -1)
        o[b] = torch.einsum("kgj,jkd->kgd", p, kv[:, 1])
        mean = torch.einsum("kgj,jkd->kgd", p, kv[:, 1].abs())
        slip = 2 * (dh * 2.0 ** -23 * size + coarse * scale * kv[:, 0].abs().sum(-1).T[:, None]).amax(-1, keepdim=True) + 2.0 ** -11 + 2.0 ** -20
        tiny = 2.0 ** -33 * kv[:, 1].abs().amax(0)[:, None] * length * p.amax(-1, keepdim=True)
        bound[b] = 2.0 ** -8 * o[b].abs() + slip * mean + tiny + 1e-30
    return o.reshape(B, -1), bound.reshape(B, -1)


def check(a, scale=None, **kw):
    out = Q.decode_attention(**a, scale=scale, **kw)
    _lib.check_status(out.device)
    want, bound = statement(a, scale)
    off = (out.to(F64) - want).abs() / bound.clamp_min(1e-30)
    assert bool((off <= 1).all()), f"off by up to {float(off.nan_to_num(9e9).max()):.2f} of the bound"
    return out


HEADS = [(16, 4, 64), (32, 8, 128), (4, 1, 128), (12, 12, 64), (5, 5, 128), (20, 1, 128), (16, 1, 64), (9, 1, 128), (34, 2, 64), (14, 2, 128), (24, 1, 64), (50, 2, 64), (97, 1, 64), (71, 1, 128)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H,Hkv,dh", HEADS)
def test_attention_head_layouts(kind, H, Hkv, dh):
    check(batch(kind, H, Hkv, dh, 64, 16, [1, 200, 0, 64, 65, 15, 130]))
    check(batch(kind, H, Hkv, dh, 64, 32, [777]), scale=0.3, max_len=1000)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page,block", [(8, 8), (16, 8), (16, 16), (32, 8), (64, 8), (64, 64), (128, 64), (192, 32)])
def test_attention_pages_and_blocks(kind, page, block):
    lens = [1, 7, 8, 9, 63, 64, 65, 191, 193, 500, 0, 1025]
    check(batch(kind, 8, 2, 128, page, block, lens))
    check(batch(kind, 8, 2, 64, page, block, lens, seed=3))


@pytest.mark.parametrize("kind", KINDS)
def test_attention_long_and_ragged(kind):
    check(batch(kind, 32, 8, 128, 64, 16, [20000], dirty=False))
    check(batch(kind, 16, 4, 64, 16, 16, [9000, 1, 4321, 2], dirty=False))
    check(batch(kind, 8, 2, 128, 64, 16, [3000, 1, 0, 17, 64, 2900, 640, 1500, 3, 0], dirty=True))


@pytest.mark.parametrize("B", [149, 300, 1025, 2100])
def test_attention_many_sequences(B):
    lens = [(7 * b * b + 3) % 200 for b in range(B)]
    check(batch("int8", 4, 2, 64, 16, 16, lens))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H,Hkv,dh", [(20, 1, 128), (24, 2, 64), (30, 1, 64), (8, 1, 128)])
def test_attention_cut_and_whole_jobs_in_turn(kind, H, Hkv, dh):
    """Long sequences among many short ones and empty slots: a CTA ends one job, has several whole ones and begins another."""
    lens = [(13 * b * b + 5) % 300 if b % 7 else 0 for b in range(200)]
    for at, n in ((0, 4000), (60, 2500), (61, 1), (199, 3333)):
        lens[at] = n
    a = batch(kind, H, Hkv, dh, 16, 8, lens)
    want = check(a)
    for _ in range(4):
        assert torch.equal(Q.decode_attention(**a), want)


@pytest.mark.parametrize("kind", KINDS)
def test_more_bytes_than_32_bits_count(kind):
    """The same three pages at the end of a pool of 4.5 GB as in a small one."""
    H, Hkv, dh, page, block = 8, 8, 128, 64, 16
    n = (9 << 29) // (2 * Hkv * page * dh)
    codes = torch.empty((n, 2, Hkv, page, dh), dtype=torch.int8, device=DEV).view(Q.CODES[kind])
    large = Q.QuantPool(codes, torch.zeros((n, 2, Hkv, page // block), device=DEV))
    small = Q.QuantPool.zeros(3, Hkv, page, dh, kind, block)
    codes[-3:].view(torch.int8).zero_()
    x = torch.randn((150, (H + 2 * Hkv) * dh), generator=gen(0), device=DEV).to(BF)
    lens, cu = torch.tensor([150], dtype=torch.int32, device=DEV), torch.tensor([0, 150], dtype=torch.int32, device=DEV)
    tables_of = [torch.tensor([[n - 1, n - 3, n - 2]], dtype=torch.int32, device=DEV), torch.tensor([[2, 0, 1]], dtype=torch.int32, device=DEV)]
    got = []
    for pool, table in zip((large, small), tables_of):
        Q.kv_append(x, H, Hkv, dh, pool, table, lens, cu_q=cu)
        got.append((Q.decode_attention(x[:1, :H * dh], pool, table, lens, H, Hkv, dh), Q.read_pages(pool, table[0])))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1]) and bool(got[0][0].any())


@pytest.mark.parametrize("kind", KINDS)
def test_attention_wide_scales(kind):
    """Scales of keys and values that differ by many powers of two between blocks, rising, falling and mixed: a small value with a large
    weight beside a large one with a small weight."""
    a = batch(kind, 8, 2, 128, 64, 16, [700, 700, 700], dirty=False)
    n = a["pool"].scales.shape[0]
    e = torch.zeros_like(a["pool"].scales)
    for b in range(3):
        ids = a["block_table"][b].long()
        ramp = torch.arange(len(ids) * 4, device=DEV).view(-1, 1, 1, 4).float()
        e[ids] = {0: ramp, 1: -ramp, 2: torch.randint(-20, 20, (len(ids), 2, 2, 4), generator=gen(7), device=DEV).float()}[b]
    a["pool"].scales.copy_(torch.exp2(-7 + e * torch.tensor([0.1, 1.0], device=DEV).view(1, 2, 1, 1)))
    assert n >= 33
    check(a)
    # and scales that are no powers of two
    a["pool"].scales.mul_(1.37)
    check(a)


@pytest.mark.parametrize("kind", KINDS)
def test_attention_large_scores(kind):
    """Scores in the hundreds, one position far above the others, in the first, a middle and the last place."""
    for at in (0, 333, 699):
        a = batch(kind, 4, 2, 64, 64, 16, [700], dirty=False)
        a["pool"].scales[:, 0] = 2.0 ** -2
        a["pool"].scales[a["block_table"][0, at // 64].long(), 0, :, at % 64 // 16] = 2.0
        check(a)


def test_attention_queries_of_any_size():
    """bf16 has eight bits of exponent, fp16 five: rows of queries near the ends of the range, and one of zeros."""
    a = batch("int8", 4, 1, 128, 64, 16, [300] * 5, dirty=False)
    for row, size in enumerate((2.0 ** 30, 2.0 ** -30, 0.0, 2.0 ** 100, 2.0 ** -120)):
        a["q"][row] *= size
    # at 2^30 and 2^100 one position takes all the weight; the statement's bound of a score would let any other have it
    out = Q.decode_attention(**a)
    want, bound = statement(a)
    for row in (1, 2, 4):
        assert bool(((out[row].to(F64) - want[row]).abs() <= bound[row]).all())
    for row in (0, 3):
        assert bool(((out[row].to(F64) - want[row]).abs() <= 2.0 ** -7 * want[row].abs()).all())


def test_attention_not_finite():
    """A NaN or an infinity in a query spoils that head alone; a NaN scale of a position that is read spoils the kv head's rows of that
    sequence alone."""
    a = batch("int8", 4, 2, 64, 16, 16, [100, 50, 60], dirty=False)
    a["q"][0, 70] = math.nan
    a["q"][1, 0] = math.inf
    a["pool"].scales[a["block_table"][2, 1].long(), 1, 1, 0] = math.nan
    out = Q.decode_attention(**a).view(3, 4, 64)
    bad = torch.zeros((3, 4), dtype=torch.bool, device=DEV)
    bad[0, 1] = bad[1, 0] = bad[2, 2] = bad[2, 3] = True
    assert torch.equal(out.isnan().all(-1), bad) and torch.equal(out.isnan().any(-1), bad)


def test_attention_page_ids_outside_the_pool():
    """They count as zeros: a score of 0 and a value of 0."""
    a = batch("int8", 4, 2, 64, 16, 16, [40, 40], dirty=False)
    zeroed = Q.QuantPool(torch.cat([a["pool"].codes, torch.zeros_like(a["pool"].codes[:1])]), torch.cat([a["pool"].scales, torch.ones_like(a["pool"].scales[:1])]))
    n = a["pool"].codes.shape[0]
    for bad in (n, 2 ** 31 - 1, -1, -2 ** 31):
        t = a["block_table"].clone()
        t[1, 1] = bad
        got = Q.decode_attention(**{**a, "block_table": t})
        t[1, 1] = n
        want = Q.decode_attention(**{**a, "block_table": t, "pool": zeroed})
        assert torch.equal(got, want)


def test_attention_output_rows_and_repeats():
    a = batch("e4m3", 8, 2, 128, 64, 16, [300, 1, 0, 2000])
    want = check(a)
    wide = torch.full((4, 8 * 128 + 24), 7.0, dtype=BF, device=DEV)
    got = Q.decode_attention(**a, out=wide[:, 8:8 + 1024])
    assert torch.equal(got, want) and bool((wide[:, :8] == 7).all()) and bool((wide[:, 1032:] == 7).all())
    for _ in range(5):
        assert torch.equal(Q.decode_attention(**a), want)                   # the same bits every time
    one = {**a, "q": a["q"][3:4], "block_table": a["block_table"][3:4], "seq_len": a["seq_len"][3:4]}
    check(one)
    assert Q.decode_attention(**{**a, "q": a["q"][:0], "block_table": a["block_table"][:0], "seq_len": a["seq_len"][:0]}).shape == (0, 1024)


def test_attention_bits_do_not_depend_on_timing():
    """Which CTA joins a job's pieces, and when it sees the others, is a matter of time; the bits are not. Pieces of two, a few and many CTAs, beside
    a stream that delays some of them."""
    a = batch("int8", 32, 8, 128, 64, 16, [3000, 10, 700, 5000] + [64 * i for i in range(12)], dirty=False)
    long = batch("e4m3", 4, 1, 128, 64, 16, [30000, 17], dirty=False, seed=1)
    twenty = batch("int8", 20, 1, 64, 64, 16, [9000, 4000, 1], dirty=False, seed=2)
    other, x = torch.cuda.Stream(), torch.randn((2048, 2048), device=DEV)
    for args in (a, long, twenty):
        want = Q.decode_attention(**args)
        for i in range(12):
            if i % 2:
                with torch.cuda.stream(other):
                    x @ x
            assert torch.equal(Q.decode_attention(**args), want)
    torch.cuda.synchronize()


def test_lengths_behind_the_table_are_cut():
    a = batch("int8", 4, 2, 64, 16, 16, [48, 32], dirty=False)
    want = Q.decode_attention(**a)
    t = a["block_table"].clone()
    t[1, 2] = t[1, 1]
    want2 = Q.decode_attention(**{**a, "block_table": t, "seq_len": torch.tensor([48, 48], dtype=torch.int32, device=DEV)})
    got = Q.decode_attention(**{**a, "block_table": t, "seq_len": torch.tensor([2 ** 31 - 1, 49], dtype=torch.int32, device=DEV)})
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want2[1])


def test_refusals():
    H, Hkv, dh, page = 4, 2, 64, 16
    pool = random_pool(3, Hkv, page, dh, "int8", 16)
    x = torch.randn((2, (H + 2 * Hkv) * dh), generator=gen(0), device=DEV).to(BF)
    table, lens = torch.zeros((2, 1), dtype=torch.int32, device=DEV), torch.ones(2, dtype=torch.int32, device=DEV)
    good = dict(H=H, Hkv=Hkv, dh=dh, pool=pool, block_table=table, seq_len=lens)
    cos, sin = ops.rope_table(8, dh, 10000.0, DEV)

    def refused(fn, *a, **kw):
        with pytest.raises(ValueError):
            fn(*a, **kw)

    for fn in (Q.kv_append, Q.decode_attention):
        for bad in (dict(block_table=table.long()), dict(seq_len=lens.long()), dict(seq_len=lens.cpu()), dict(block_table=table.cpu()),
                    dict(block_table=torch.zeros((2, 2), dtype=torch.int32, device=DEV)[:, ::2]), dict(pool=on_cpu(pool)),
                    dict(pool=(pool.codes, pool.scales.cpu())), dict(pool=(pool.codes.transpose(0, 1).contiguous().transpose(0, 1), pool.scales))):
            refused(fn, x, **{**good, **bad})
        refused(fn, x[:, 4:], **good)                                        # rows that are not 16-byte aligned, or too short
        refused(fn, x.repeat(1, 2)[:, ::2], **good)
        refused(fn, x[:1].expand(2, -1), **good)
    refused(Q.kv_append, x, **good, cu_q=torch.zeros(3, dtype=torch.int64, device=DEV))
    refused(Q.rope_kv_append, x, H, Hkv, dh, cos.cpu(), sin.cpu(), pool, table, lens)
    refused(Q.rope_kv_append, x, H, Hkv, dh, cos.t().contiguous().t(), sin, pool, table, lens)
    small = random_pool(3, Hkv, page, 32, "int8", 16)
    refused(Q.kv_append, x, H, Hkv, 32, small, table, lens)
    refused(Q.decode_attention, x, small, table, lens, H, Hkv, 32)
    refused(Q.read_pages, small, [0])
    refused(Q.read_pages, pool, [3])
    refused(Q.read_pages, pool, torch.zeros(1, dtype=torch.int64, device=DEV))
    refused(Q.read_pages, pool, torch.zeros(4, dtype=torch.int32, device=DEV)[::2])
    refused(Q.decode_attention, x, **good, out=torch.empty((2, H * dh), dtype=BF))
    refused(Q.decode_attention, x, **good, out=torch.empty((2, H * dh + 4), dtype=BF, device=DEV)[:, 4:])


# ---------------------------------------------------------------------------------------------------------------- ends of the ranges
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("cu", [False, True])
def test_a_rotation_without_positions_leaves_all_rows(kind, cu):
    """Every row lies behind the end of tables that have no positions."""
    H, Hkv, dh, page, block = 4, 2, 64, 16, 16
    pool = random_pool(3, Hkv, page, dh, kind, block)
    kept = Q.QuantPool(pool.codes.clone(), pool.scales.clone())
    i = lambda *e: torch.tensor(e, dtype=torch.int32, device=DEV)
    x = torch.randn((3, (H + 2 * Hkv) * dh), generator=gen(1), device=DEV).to(BF)
    before, none = x.clone(), torch.empty((0, dh // 2), device=DEV)
    table = torch.stack([i(0), i(1), i(2)])
    Q.rope_kv_append(x, H, Hkv, dh, none, none, pool, table, i(1, 3, 1), cu_q=i(0, 1, 2, 3) if cu else None)
    assert torch.equal(x, before)
    assert torch.equal(bits(pool.codes), bits(kept.codes)) and torch.equal(bits(pool.scales), bits(kept.scales))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H,Hkv,dh", [(8, 2, 128), (4, 4, 64), (20, 1, 128), (24, 1, 64)])
def test_attention_scores_near_the_lowest_value(kind, H, Hkv, dh):
    """All scores of a sequence are alike and -2^120 or lower: the answer is the mean of the values, and with one block far less low that of
    its values. Equal keys give equal scores, bit for bit, and so weights of one power of two; what is left are the sums of up to n
    terms in 32 bits, each addition off by a step of 2^-23 at most, and the rounding to bf16."""
    lens = [1, 17, 300, 0, 5000]
    a = batch(kind, H, Hkv, dh, 64, 16, lens, dirty=False)
    pool = a["pool"]
    pool.codes.view(torch.int8)[:, 0] = 1 if kind == "int8" else 0x38            # keys of 1
    pool.scales[:, 0] = 2.0 ** 60
    a["q"][:] = -2.0 ** 60
    for least in (False, True):
        if least:
            for b, length in enumerate(lens):
                if length:
                    pool.scales[a["block_table"][b, length // 2 // 64].long(), 0, :, length // 2 % 64 // 16] = 2.0 ** 59
        out = Q.decode_attention(**a).view(len(lens), Hkv, H // Hkv, dh)
        for b, length in enumerate(lens):
            if not length:
                assert not bool(out[b].any())
                continue
            pos = torch.arange(length, device=DEV)
            if least:
                pos = pos[pos // 16 == length // 2 // 16]
            at = a["block_table"][b].long()[pos // 64]
            v = pool.codes.view(torch.int8)[at, 1, :, pos % 64].view(pool.codes.dtype).to(F64) * pool.scales[at, 1, :, pos % 64 // 16].to(F64)[..., None]
            want, size = v.mean(0)[:, None], v.abs().mean(0)[:, None]
            bound = 2.0 ** -8 * want.abs() + length * 2.0 ** -23 * size
            assert bool(((out[b].to(F64) - want).abs() <= bound).all()), (least, length)


def spread_values(kind, H, Hkv, dh, lens, up, gap, seed=0):
    """Sequences of positive values with a block of them 2^up times as large as the others, whose scores are ``gap`` (base 2) above the others'
    for even query heads and below them for odd ones; in the middle of a sequence."""
    a = batch(kind, H, Hkv, dh, 64, 16, lens, seed=seed, dirty=False)
    pool, one = a["pool"], 1 if kind == "int8" else 0x38
    v = pool.codes.view(torch.int8)[:, 1]
    v.copy_(v.abs() if kind == "int8" else v & 0x7f)
    pool.scales[:, 1] = torch.exp2(torch.randint(-3, 3, pool.scales[:, 1].shape, generator=gen(seed + 5), device=DEV).float())
    pool.scales[:, 0] = 2.0 ** -7
    pool.codes.view(torch.int8)[..., 0][:, 0] = 0
    for b, length in enumerate(lens):
        at, slot = a["block_table"][b, length // 2 // 64].long(), length // 2 % 64 // 16
        pool.scales[at, 1, :, slot] *= 2.0 ** up
        pool.scales[at, 0, :, slot] = 1.0
        keys = pool.codes.view(torch.int8)[at, 0, :, slot * 16:slot * 16 + 16]
        keys[:] = 0
        keys[..., 0] = one
    q = a["q"][:, :H * dh].view(len(lens), H, dh)
    q[:, 0::2, 0] = gap * math.log(2.0) * math.sqrt(dh)
    q[:, 1::2, 0] = -gap * math.log(2.0) * math.sqrt(dh)
    return a


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H,Hkv,dh", [(8, 2, 128), (4, 2, 64), (20, 1, 128)])
@pytest.mark.parametrize("lens", [[40, 700, 512], [3000], [20000, 17]], ids=["whole", "cut", "long"])
@pytest.mark.parametrize("up,gap", [(24, 60), (34, 40), (34, 34), (60, 90), (12, 8), (90, 90), (-40, 60), (60, 150), (100, 160)])
def test_attention_values_of_one_block_far_from_the_others(kind, H, Hkv, dh, up, gap, lens):
    """A weight counts by the value's scale that it has: a scale far above the others' takes nothing from them where its own weight
    is small. As ``statement``, but what a product of a weight and a scale may lose below the numbers of fp16 is half a step of 2^-24 where
    the largest such product of the sequence is 2 at least, times a code of 448 (127) at most: not a share of values without weight. The
    scores here have the magnitudes that ``statement`` takes its slips from."""
    a = spread_values(kind, H, Hkv, dh, lens, up, gap)
    out = Q.decode_attention(**a).to(F64).view(len(lens), Hkv, H // Hkv, dh)
    pool, scale = a["pool"], dh ** -0.5
    largest = Q.LARGEST[pool.codes.dtype]
    for b, length in enumerate(lens):
        pos = torch.arange(length, device=DEV)
        at = a["block_table"][b].long()[pos // 64]
        steps = pool.scales[at, :, :, pos % 64 // 16].to(F64)
        kv = pool.codes.view(torch.int8)[at, :, :, pos % 64].view(pool.codes.dtype).to(F64) * steps[..., None]
        q = a["q"][b, :H * dh].to(F64).reshape(Hkv, H // Hkv, dh)
        p = torch.softmax(torch.einsum("kgd,jkd->kgj", q, kv[:, 0]) * scale, -1)
        size = torch.einsum("kgd,jkd->kgj", q.abs(), kv[:, 0].abs()) * scale
        coarse = q.abs().amax(-1, keepdim=True) * 2.0 ** -14 * (kind == "int8")
        want, mean = torch.einsum("kgj,jkd->kgd", p, kv[:, 1]), torch.einsum("kgj,jkd->kgd", p, kv[:, 1].abs())
        # a score's own slip, before the exponential: of the positions with weight the largest counts
        slip = 2 * (dh * 2.0 ** -23 * size + coarse * scale * kv[:, 0].abs().sum(-1).T[:, None]).amax(-1, keepdim=True) + 2.0 ** -11 + 2.0 ** -20
        tiny = length * largest * 2.0 ** -26 * (p * steps[:, 1].T[:, None]).amax(-1, keepdim=True)
        bound = 2.0 ** -8 * want.abs() + slip * mean + tiny
        off = (out[b] - want).abs() / bound
        assert bool((off <= 1).all()), (length, float(off.nan_to_num(9e9).max()))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H,Hkv,dh", [(8, 2, 128), (20, 1, 64)])
def test_attention_values_near_the_largest_number(kind, H, Hkv, dh):
    """Values of up to 2^127, and down to the smallest scale that is written: 2^-96 (e4m3: 2^-98)."""
    for scale in (2.0 ** (120 if kind == "int8" else 118), 2.0 ** (-96 if kind == "int8" else -98)):
        a = batch(kind, H, Hkv, dh, 64, 16, [1, 16, 300, 2000], dirty=False)
        a["pool"].scales[:, 1] = 2.0
        want, bound = statement(a)
        a["pool"].scales[:, 1] = 2 * scale
        out = Q.decode_attention(**a).to(F64)
        assert bool(((out / scale - want).abs() <= bound).all())


@pytest.mark.parametrize("size", [2.0 ** 30, 2.0 ** -30, 0.0, 2.0 ** 100, 2.0 ** -120, 2.0 ** -126, 2.0 ** 115])
def test_attention_queries_of_any_size_e4m3(size):
    """As whole numbers for int8 keys, queries are brought into fp16's range by a power of two for e4m3: near the ends of bf16's."""
    a = batch("e4m3", 4, 1, 128, 64, 16, [300] * 2, dirty=False)
    a["q"][0] = (a["q"][0].double().clamp(-3.9, 3.9) * size).to(BF)
    out = Q.decode_attention(**a).to(F64)
    want, bound = statement(a)
    # of a large query one position takes all the weight; the statement's bound of a score would let any other have it
    ok = (out - want).abs() <= (2.0 ** -7 * want.abs() if size > 2.0 ** 20 else bound)
    assert bool(ok[0].all()) and bool(((out - want).abs() <= bound)[1].all())


def test_attention_not_finite_e4m3():
    """A NaN or an infinity in a query spoils that head alone; a NaN scale of a position that is read, or a NaN code of a value, the kv head's
    rows of that sequence, the code one dimension of them."""
    a = batch("e4m3", 4, 2, 64, 16, 16, [100, 50, 60, 70], dirty=False)
    a["q"][0, 70] = math.nan
    a["q"][1, 0] = math.inf
    a["pool"].scales[a["block_table"][2, 1].long(), 1, 1, 0] = math.nan
    a["pool"].codes.view(torch.int8)[a["block_table"][3, 4].long(), 1, 0, 5, 9] = 0x7f
    out = Q.decode_attention(**a).view(4, 4, 64)
    bad = torch.zeros((4, 4, 64), dtype=torch.bool, device=DEV)
    bad[0, 1] = bad[1, 0] = bad[2, 2] = bad[2, 3] = True
    bad[3, :2, 9] = True
    assert torch.equal(out.isnan(), bad)


def test_rows_on_the_host_are_refused_beside_a_pool_on_the_device():
    """Before anything is written."""
    H, Hkv, dh, page = 4, 2, 64, 16
    pool = random_pool(3, Hkv, page, dh, "int8", 16)
    kept = pool.codes.clone()
    x = torch.randn((5, (H + 2 * Hkv) * dh), generator=gen(0), device=DEV).to(BF).cpu()
    table, lens, cu = torch.tensor([[1, 2]]).int(), torch.tensor([10]).int(), torch.tensor([0, 5]).int()
    cos, sin = ops.rope_table(16, dh, 10000.0, DEV)
    host = on_cpu(pool)
    for bad in (dict(pool=pool), dict(pool=host, block_table=table.to(DEV)), dict(pool=host, seq_len=lens.to(DEV)), dict(pool=host, cu_q=cu.to(DEV))):
        with pytest.raises(ValueError):
            Q.kv_append(x, H, Hkv, dh, **{**dict(block_table=table, seq_len=lens, cu_q=cu), **bad})
    with pytest.raises(ValueError):
        Q.rope_kv_append(x, H, Hkv, dh, cos, sin, host, table, lens, cu_q=cu)
    for bad in (dict(pool=pool), dict(block_table=table.to(DEV)), dict(seq_len=lens.to(DEV)), dict(out=torch.empty((1, H * dh), dtype=BF, device=DEV))):
        with pytest.raises(ValueError):
            Q.decode_attention(x[:1], **{**dict(pool=host, block_table=table, seq_len=lens, H=H, Hkv=Hkv, dh=dh), **bad})
    assert torch.equal(pool.codes, kept)
