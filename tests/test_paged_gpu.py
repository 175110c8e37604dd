"""Ops on pages that sequences share, against 64-bit statements."""
import math

import pytest
import torch

from scirust_b200.ops import _lib, paged

pytestmark = pytest.mark.gpu
BF, F64 = torch.bfloat16, torch.float64
DEV = "cuda"


def batch(B, H, Hkv, dh, page, prefix, tails, new=None, seed=0, spare=3, q_pad=8):
    """Inputs of a batch: tails[b] positions behind the prefix, of which the last new[b] are rows (default: one each)."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    shared = prefix // page
    own = [max(0, (prefix + t + page - 1) // page - shared) for t in tails]
    total = shared + sum(own) + spare
    order = torch.randperm(total, generator=g, device=DEV).int()
    table = torch.full((B, shared + max(own + [1])), -1, dtype=torch.int32, device=DEV)
    at = shared
    for b, n in enumerate(own):
        table[b, :shared] = order[:shared]
        table[b, shared:shared + n] = order[at:at + n]
        at += n
    pool = torch.randn((total, 2, Hkv, page, dh), generator=g, device=DEV).to(BF)
    rows = [1] * B if new is None else new
    q = (torch.randn((sum(rows), H * dh + q_pad), generator=g, device=DEV) * 1.5).to(BF)
    cu = None if new is None else torch.tensor([0] + list(torch.tensor(new).cumsum(0)), dtype=torch.int32, device=DEV)
    return dict(q=q, pool=pool, block_table=table, page=page, seq_len=torch.tensor([prefix + t for t in tails], dtype=torch.int32, device=DEV),
                prefix_table=order[:shared].contiguous(), prefix_len=prefix, H=H, Hkv=Hkv, dh=dh, cu_q=cu)


def statement(a, scale=None):
    """(o, bound): 64 bits, and how far an element may be off. P is rounded to bf16 (half a step of 2^-8) and weighs v, the answer is
    rounded once more; a score is a sum of dh products in 32 bits, each addition off by a step of 2^-23 of the sum of magnitudes, which
    the exponential passes on as a relative error of a weight and of their sum."""
    H, Hkv, dh, page = a["H"], a["Hkv"], a["dh"], a["page"]
    scale = dh ** -0.5 if scale is None else scale
    n = a["q"].shape[0]
    o, bound = torch.zeros((n, Hkv, H // Hkv, dh), dtype=F64, device=DEV), torch.zeros((n, Hkv, H // Hkv, dh), dtype=F64, device=DEV)
    ends = list(range(n + 1)) if a["cu_q"] is None else a["cu_q"].tolist()
    for b, length in enumerate(a["seq_len"].tolist()):
        t0, t1 = ends[b], ends[b + 1]
        for t in range(t0, t1):
            limit = length - (t1 - t0) + (t - t0) + 1
            if limit <= 0:
                continue
            pos = torch.arange(limit, device=DEV)
            kv = a["pool"][a["block_table"][b].long()[pos // page], :, :, pos % page].to(F64)
            q = a["q"][t, :H * dh].to(F64).reshape(Hkv, H // Hkv, dh)
            s = torch.einsum("kgd,jkd->kgj", q, kv[:, 0]) * scale
            size = torch.einsum("kgd,jkd->kgj", q.abs(), kv[:, 0].abs()) * scale
            p = torch.softmax(s, -1)
            o[t] = torch.einsum("kgj,jkd->kgd", p, kv[:, 1])
            mean = torch.einsum("kgj,jkd->kgd", p, kv[:, 1].abs())
            slip = 2 * dh * 2.0 ** -23 * size.amax(-1, keepdim=True)
            bound[t] = 2.0 ** -8 * (mean + o[t].abs()) + slip * mean + 1e-6
    return o.reshape(n, -1), bound.reshape(n, -1)


@pytest.fixture(autouse=True)
def _poisoned(monkeypatch):
    """Workspaces and answers begin as NaN and between fences, so that a part which is read and was not written shows."""
    monkeypatch.setattr(_lib, "DEBUG_POISON", True)
    yield
    torch.cuda.synchronize()
    _lib.check_canaries()


def check(a, **kw):
    out = paged.shared_prefix_attention(**a, **kw)
    _lib.check_status(out.device)
    want, bound = statement(a, kw.get("scale"))
    off = (out.to(F64) - want).abs() / bound.clamp_min(1e-30)
    assert bool((off <= 1).all()), f"off by up to {float(off.nan_to_num(9e9).max()):.2f} of the bound"
    return out


HEADS = [(16, 4, 64), (32, 8, 128), (4, 1, 128), (8, 8, 64), (6, 2, 128), (20, 1, 64)]


@pytest.mark.parametrize("H,Hkv,dh", HEADS)
@pytest.mark.parametrize("page,prefix,tails", [
    (64, 128, [1, 64, 65, 3]), (64, 1000, [1, 5, 200, 24, 25, 88]), (16, 333, [1, 7, 40]), (8, 80, [9]), (128, 640, [1, 129, 300]),
    (32, 31, [1, 64]), (64, 0, [1, 63, 64, 130]), (192, 400, [20, 700]), (40, 200, [1, 41, 90])])
def test_one_row_each(H, Hkv, dh, page, prefix, tails):
    check(batch(len(tails), H, Hkv, dh, page, prefix, tails))


@pytest.mark.parametrize("H,Hkv,dh", HEADS[:3] + [(6, 2, 128)])
@pytest.mark.parametrize("page,prefix,tails,new", [
    (64, 512, [64, 10, 1, 33], [64, 10, 1, 5]), (64, 1000, [30, 7, 7], [30, 0, 7]), (16, 333, [70, 70], [70, 3]),
    (64, 200, [500], [500]), (64, 0, [150, 1, 64], [150, 1, 64]), (128, 300, [3, 260, 9], [3, 200, 9]), (8, 100, [1, 1, 1], [1, 1, 1])])
def test_ragged_rows(H, Hkv, dh, page, prefix, tails, new):
    check(batch(len(tails), H, Hkv, dh, page, prefix, tails, new))


def test_rows_before_the_first_position_and_empty_sequences():
    a = batch(5, 16, 4, 64, 64, 256, [10, 1, 5, 70, 3])
    a["seq_len"] = torch.tensor([266, 0, 100, 326, 256], dtype=torch.int32, device=DEV)     # empty, inside the prefix, its last position
    out = check(a)
    assert not out[1].any()
    a = batch(3, 16, 4, 64, 64, 128, [40, 6, 4], [40, 6, 4])
    a["seq_len"] = torch.tensor([20, 3, 0], dtype=torch.int32, device=DEV)                  # more rows than positions
    out = check(a)
    assert not out[:20].any() and not out[40:43].any() and not out[46:].any() and bool(out[43].any())
    a = batch(3, 16, 4, 64, 64, 0, [4, 6, 4])
    a["seq_len"] = torch.zeros(3, dtype=torch.int32, device=DEV)
    assert not check(a).any()


@pytest.mark.parametrize("new", [None, [1, 9, 1, 30]])
@pytest.mark.parametrize("junk", [float("nan"), float("inf"), -3.3895e38])
def test_what_no_row_sees_may_hold_anything(new, junk):
    a = batch(4, 8, 2, 128, 16, 100, [1, 9, 50, 30], new)
    page = a["page"]
    table = a["block_table"].cpu()
    seen = torch.zeros(a["pool"].shape[0], page, dtype=torch.bool)
    for b, length in enumerate(a["seq_len"].tolist()):
        pos = torch.arange(length)
        seen[table[b].long()[pos // page], pos % page] = True
    a["pool"].masked_fill_(~seen.to(DEV)[:, None, None, :, None], junk)
    check(a)


@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("G", [1, 2, 3, 5, 7, 8, 9])
def test_rows_of_a_sequence_of_one_token(G, dh):
    """Few rows for each kv head, shared by few or many tokens, blocks that end everywhere, maxima that grow and lie beyond 2^24."""
    for B, prefix, tails in ((1, 0, [1]), (1, 256, [129]), (2, 128, [127, 128]), (3, 0, [500, 1, 256]), (8, 640, [1, 2, 15, 16, 17, 129, 255, 640]),
                             (9, 8, [300 + 60 * b for b in range(9)])):
        a = batch(B, 2 * G, 2, dh, 8, prefix, tails, seed=B)
        check(a, max_len=prefix + max(tails))
        a["pool"][:, 0] *= torch.linspace(0.2, 3.0, a["pool"].shape[0], device=DEV)[:, None, None, None].to(BF)
        check(a)
        a["pool"][:, 0] *= 2.0 ** 14
        a["q"] *= 2.0 ** 14
        check_order(a)


def check_order(a):
    """Scores so far apart that a row's answer is the value of its largest one."""
    out = paged.shared_prefix_attention(**a).to(F64)
    o, _ = statement(a)
    H, Hkv, dh, page = a["H"], a["Hkv"], a["dh"], a["page"]
    for b, length in enumerate(a["seq_len"].tolist()):
        pos = torch.arange(length, device=DEV)
        k = a["pool"][a["block_table"][b].long()[pos // page], 0, :, pos % page].to(F64)
        q = a["q"][b, :H * dh].to(F64).reshape(Hkv, H // Hkv, dh)
        two = torch.einsum("kgd,jkd->kgj", q, k).topk(min(2, length), -1).values
        off = 2 * dh * 2.0 ** -23 * torch.einsum("kgd,jkd->kgj", q.abs(), k.abs()).amax(-1)       # of a score in 32 bits
        clear = two[..., 0] - two[..., -1] > 2 * off if length > 1 else torch.ones_like(off, dtype=torch.bool)
        rows = (out[b] - o[b]).reshape(Hkv, H // Hkv, dh)[clear]
        assert bool((rows.abs() <= 2.0 ** -8 * o[b].reshape(Hkv, H // Hkv, dh)[clear].abs() + 1e-6).all())


def test_scores_far_apart():
    a = batch(6, 16, 4, 64, 64, 320, [1, 9, 50, 30, 77, 128])
    a["q"] *= 20                                   # scores of a few hundred: one position has all the weight
    check(a)
    check(batch(6, 16, 4, 64, 64, 320, [1, 9, 50, 30, 77, 128]), scale=0.01)


def test_weights_of_the_lowest_value_mask():
    """A row whose scores are all near the lowest bf16 value still has weights that sum to one."""
    a = batch(2, 4, 4, 64, 64, 128, [5, 70])
    a["q"].fill_(-3e19)
    a["pool"][:, 0] = 3e18                         # q.k = -9e37 * 64, beyond 32 bits only after 64 products
    a["pool"][:, 0, :, :, 1:] = 0
    out = check(a)
    assert bool(out.any())


@pytest.mark.parametrize("H,Hkv,dh", [(4, 4, 64), (16, 2, 128), (18, 2, 64)])
@pytest.mark.parametrize("new", [None, [5, 60, 1]])
def test_equal_scores_near_the_lowest_value_weigh_all_positions_alike(H, Hkv, dh, new):
    """Scores of -2^127, in units of log 2 -3.387e38, where the type ends at -3.403e38: the answer is the mean of the values that a row sees.
    Weights are 1 and their sum a whole number, both exact; a value's sum is off by a step of 2^-23 of the magnitudes for each addition,
    the division by two steps, and the answer is rounded to bf16."""
    a = batch(3, H, Hkv, dh, 64, 320, [5, 270, 1], new)
    a["q"].zero_()
    a["q"][:, :H * dh:dh] = -2.0 ** 63
    a["pool"][:, 0] = 0
    a["pool"][:, 0, ..., 0] = 2.0 ** 64
    scale = 3.387e38 / 2.0 ** 127 / 1.4426950408889634
    out = paged.shared_prefix_attention(**a, scale=scale).to(F64).view(-1, Hkv, H // Hkv, dh)
    _lib.check_status(out.device)
    t = 0
    for b, length in enumerate(a["seq_len"].tolist()):
        for limit in range(length - (1 if new is None else new[b]) + 1, length + 1):
            pos = torch.arange(limit, device=DEV)
            v = a["pool"][a["block_table"][b].long()[pos // 64], 1, :, pos % 64].to(F64)              # [limit, Hkv, dh]
            mean, size = v.mean(0), v.abs().mean(0)
            bound = 2.0 ** -8 * mean.abs() + (limit + 2) * 2.0 ** -23 * size
            assert bool(((out[t] - mean[:, None]).abs() <= bound[:, None]).all())
            t += 1


def test_rows_of_no_sequence():
    a = batch(3, 16, 4, 64, 64, 256, [9, 5, 20], [9, 5, 20])
    a["q"] = torch.cat([a["q"], a["q"][:7]])
    a["cu_q"] += 3                                 # three rows in front of the first sequence, four behind the last
    a["q"] = a["q"].roll(3, 0).contiguous()
    out = check(a)
    assert not out[:3].any() and not out[-4:].any()
    kept = torch.full_like(out, 7.0)
    assert paged.shared_prefix_attention(**a, out=kept) is kept
    assert torch.equal(kept[3:-4], out[3:-4]) and bool((kept[:3] == 7).all()) and bool((kept[-4:] == 7).all())


def test_offsets_that_make_no_sense_stay_inside():
    a = batch(4, 16, 4, 64, 64, 256, [9, 5, 20, 2], [9, 5, 20, 2])
    a["cu_q"] = torch.tensor([0, 30, 10, 9000, -5], dtype=torch.int32, device=DEV)
    guard = torch.full((a["q"].shape[0] + 8, 1024), 7.0, dtype=BF, device=DEV)
    out = paged.shared_prefix_attention(**a, out=guard[4:-4])
    _lib.check_status(out.device)
    assert bool((guard[:4] == 7).all()) and bool((guard[-4:] == 7).all())


def test_pages_outside_the_pool_read_as_zeros():
    a = batch(3, 16, 4, 64, 64, 128, [70, 5, 300])
    bad = dict(a, block_table=a["block_table"].clone())
    bad["block_table"][0, 2:] = torch.tensor([1 << 30, -7, 5000, 2 ** 31 - 1, 0], device=DEV)[:bad["block_table"].shape[1] - 2].int()
    out = paged.shared_prefix_attention(**bad)
    _lib.check_status(out.device)
    assert torch.equal(out[1:], paged.shared_prefix_attention(**a)[1:]) and bool(out.isfinite().all())


def test_strides_of_rows_and_of_the_answer():
    a = batch(5, 16, 4, 64, 64, 256, [10, 1, 5, 70, 3])
    wide = torch.zeros((5, 4096), dtype=BF, device=DEV)
    wide[:, 8:8 + 1024] = a["q"][:, :1024]
    want = check(a)
    answer = torch.zeros((5, 2048), dtype=BF, device=DEV)
    out = paged.shared_prefix_attention(**dict(a, q=wide[:, 8:]), out=answer[:, 512:1536])
    assert torch.equal(out, want) and not answer[:, :512].any() and not answer[:, 1536:].any()


def test_rows_that_overlap_are_refused_and_one_row_has_any_stride():
    a = batch(3, 8, 2, 64, 16, 100, [5, 9, 1])
    with pytest.raises(ValueError):
        paged.shared_prefix_attention(**{**a, "q": a["q"][:1].expand(3, -1)})
    with pytest.raises(ValueError):
        paged.shared_prefix_attention(**a, out=torch.zeros((1, 512), dtype=BF, device=DEV).expand(3, -1))
    one = batch(1, 8, 2, 64, 16, 100, [5])
    one["q"] = one["q"].as_strided((1, 512), (0, 1))
    check(one, out=torch.zeros(600, dtype=BF, device=DEV).as_strided((1, 512), (7, 1)))


def test_long_prefix_many_sequences():
    check(batch(64, 8, 2, 64, 64, 6000, [1 + 7 * b % 190 for b in range(64)]))
    check(batch(130, 4, 1, 128, 64, 700, [1 + 11 * b % 300 for b in range(130)]))


def test_more_sequences_than_a_cta_plans_for():
    check(batch(1100, 4, 1, 64, 64, 130, [1 + b % 90 for b in range(1100)]))


def test_offsets_beyond_32_bits():
    """Pages whose elements lie past 2^31 of the pool (5.4 GB)."""
    H, Hkv, dh, page = 8, 8, 128, 64
    a = batch(2, H, Hkv, dh, page, 128, [100, 7])
    far = torch.empty((20600, 2, Hkv, page, dh), dtype=BF, device=DEV)
    assert far.numel() > 1 << 31
    n = a["pool"].shape[0]
    far[-n:] = a["pool"]
    move = 20600 - n
    b = dict(a, pool=far, block_table=a["block_table"] + move, prefix_table=a["prefix_table"] + move)
    assert torch.equal(paged.shared_prefix_attention(**b), check(a))


def test_same_bits_again_on_another_stream_and_in_a_graph():
    a = batch(9, 32, 8, 128, 64, 1000, [1 + 30 * b for b in range(9)])
    want = check(a, max_len=1300)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [paged.shared_prefix_attention(**a, max_len=1300) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(o, want) for o in outs)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            o = paged.shared_prefix_attention(**a, max_len=1300)
        graphs.append((g, o))
    a["seq_len"] -= 17                              # lengths and pages are read by the replay
    a["seq_len"].clamp_(min=1000)
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):                              # both graphs at once
        for (g, _), s in zip(graphs, (one, two)):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    want = check(a, max_len=1300)
    assert torch.equal(graphs[0][1], want) and torch.equal(graphs[1][1], want)


def test_two_calls_at_once():
    """On two streams, and graphs captured on one stream and replayed on two: each has a workspace of its own."""
    ab = [batch(16, 32, 8, 128, 64, 4000, [1 + 17 * b for b in range(16)], seed=1),
          batch(7, 32, 8, 128, 64, 2000, [40 + b for b in range(7)], [1 + 5 * b for b in range(7)], seed=2)]
    want = [check(a) for a in ab]
    streams, graphs, outs = [torch.cuda.Stream() for _ in ab], [], [torch.zeros_like(w) for w in want]
    torch.cuda.synchronize()
    for _ in range(10):
        for s, a, o in zip(streams, ab, outs):
            with torch.cuda.stream(s):
                paged.shared_prefix_attention(**a, out=o)
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))
    for a, o in zip(ab, outs):
        o.zero_()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[0]):
            paged.shared_prefix_attention(**a, out=o)
        graphs.append(g)
    for _ in range(10):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    _lib.check_status(torch.device(DEV, 0))
    assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_what_a_bound_of_the_lengths_is_for():
    """max_len sizes the launch; lengths beyond it are still answered."""
    a = batch(3, 16, 4, 64, 64, 256, [300, 5, 700])
    assert torch.allclose(check(a, max_len=1).float(), check(a).float(), atol=0.05)


@pytest.mark.parametrize("B,tail", [(16, 256), (33, 400), (64, 512), (300, 130)])
def test_many_short_pieces_a_cta(B, tail):
    """CTAs that go from piece to piece, of one block and of several, of one tile of rows and of two."""
    g = torch.Generator().manual_seed(B)
    tails = torch.randint(1, tail, (B,), generator=g).tolist()
    check(batch(B, 32, 8, 128, 64, 1000, tails))
    new = [min(t, 1 + b % 70) for b, t in enumerate(tails)]
    check(batch(B, 8, 2, 64, 16, 300, tails, new))


@pytest.mark.parametrize("new", [[300] + [1] * 7, [33] * 6, [64] * 4, [0, 130, 1, 77]])
def test_runs_of_uneven_length_behind_a_long_prefix(new):
    """As many tokens as fill the sequences' tiles, and rows of all of them in a tile of the prefix."""
    a = batch(len(new), 8, 2, 128, 64, 4100, [n + 3 for n in new], new)
    assert sum(new) >= len(new) * 32 and paged._in_common(sum(new), len(new), 32, 4096, max(new) + 3)
    check(a, max_len=4100 + max(new) + 3)
    check(a, max_len=4100 + max(new))               # where all have 64, apart


@pytest.mark.parametrize("H,Hkv,dh,B,prefix,tails,max_len", [
    (32, 32, 128, 8, 512, [257] * 8, None), (32, 32, 128, 8, 512, [2000] * 8, None), (32, 32, 64, 4, 512, [513, 600, 1, 900], None),
    (16, 16, 64, 8, 1024, [2000, 1, 3000, 40, 2500, 7, 129, 1800], None), (32, 8, 128, 2, 256, [8192, 8192], None),
    (32, 8, 128, 2, 256, [12000, 1], None), (32, 8, 128, 2, 128, [300, 300], 1), (32, 8, 128, 2, 128, [1, 1], 1), (16, 4, 64, 1, 128, [9000], 1)])
def test_shared_items_of_few_rows_beside_long_own_parts(H, Hkv, dh, B, prefix, tails, max_len):
    """A CTA has more shared items than it has slots for what is cut."""
    a = batch(B, H, Hkv, dh, 64, prefix, tails)
    check(a, max_len=prefix + max(tails) if max_len is None else max_len)
    check(a)


# ---------------------------------------------------------------------------------------------- copies of pages
def _copied(pools, src, dst, rows, out=None):
    """Each pool as it should be, one copy at a time."""
    want = [(o if out is not None else p).clone() for p, o in zip(pools, out or pools)]
    for w, p in zip(want, pools):
        for a, b in zip(src, dst):
            w[b, ..., :rows, :] = p[a, ..., :rows, :]
    return want


@pytest.mark.parametrize("shape,dtype", [((40, 2, 8, 64, 128), BF), ((33, 2, 3, 16, 64), BF), ((21, 2, 1, 8, 80), torch.float16),
                                         ((17, 2, 2, 5, 7), torch.uint8), ((19, 2, 2, 3, 6), torch.int16), ((9, 4, 1), torch.float32)])
@pytest.mark.parametrize("rows", [None, 1, 3])
def test_copies_of_pages(shape, dtype, rows):
    g = torch.Generator(device=DEV).manual_seed(1)
    pools = [torch.randint(0, 100, shape, generator=g, device=DEV).to(dtype) for _ in range(3)]
    order = torch.randperm(shape[0], generator=torch.Generator().manual_seed(2)).tolist()
    n = shape[0] // 3
    for src, dst in ((order[:n], order[n:2 * n]), ([order[0]] * n, order[n:2 * n]), (order[:1], order[1:2])):
        for ids in (lambda v: v, lambda v: torch.tensor(v), lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)):
            want = _copied(pools, src, dst, rows or shape[-2])
            got = [p.clone() for p in pools]
            paged.copy_pages(paged.PagePools(got), ids(src), ids(dst), rows=rows)
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        other = [torch.zeros((n + 2, *shape[1:]), dtype=dtype, device=DEV) for _ in pools]
        into = list(range(n + 1, n + 1 - len(src), -1))
        want = _copied(pools, src, into, rows or shape[-2], other)
        paged.copy_pages(pools, src, into, rows=rows, out=other)
        assert all(torch.equal(a, b) for a, b in zip(other, want))


def test_copies_skip_what_is_outside_and_take_many_layers():
    pools = [torch.randn(12, 2, 2, 16, 64, device=DEV).to(BF) for _ in range(70)]
    want = _copied(pools, [3, 4], [7, 8], 16)
    src = torch.tensor([3, -1, 12, 5, 4, 2 ** 31 - 1], dtype=torch.int32, device=DEV)
    dst = torch.tensor([7, 0, 1, -5, 8, 2], dtype=torch.int32, device=DEV)
    paged.copy_pages(pools, src, dst)
    assert all(torch.equal(a, b) for a, b in zip(pools, want))


def test_copies_beyond_32_bits():
    pool = torch.empty((20600, 2, 8, 64, 128), dtype=BF, device=DEV)
    pool[-4:] = torch.randn(4, 2, 8, 64, 128, device=DEV)
    pool[3:5] = 0
    paged.copy_pages([pool], [20599, 20597], [3, 20598])
    assert torch.equal(pool[3], pool[20599]) and torch.equal(pool[20598], pool[20597]) and not pool[4].any()


def test_copies_in_a_graph_take_new_ids():
    pools = [torch.randn(12, 2, 2, 16, 64, device=DEV).to(BF) for _ in range(2)]
    src, dst = torch.tensor([1, 2], dtype=torch.int32, device=DEV), torch.tensor([8, 9], dtype=torch.int32, device=DEV)
    handle = paged.PagePools(pools)
    paged.copy_pages(handle, src, dst)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        paged.copy_pages(handle, src, dst)
    src.copy_(torch.tensor([3, 4]))
    dst.copy_(torch.tensor([10, 11]))
    want = _copied(pools, [3, 4], [10, 11], 16)
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(pools, want))


def test_copies_between_pools_that_reach_into_one_another_are_refused_for_ids_on_the_device_too():
    memory = torch.zeros((9, 2, 1, 4, 8), dtype=BF, device=DEV)
    ids = [torch.tensor([i], dtype=torch.int32, device=DEV) for i in (0, 1)]
    for pools, out in (([memory[:5]], [memory[3:]]), ([memory[:3], memory[3:6]], [memory[6:]] * 2)):
        with pytest.raises(ValueError):
            paged.copy_pages(pools, *ids, out=out)
    memory[0] = 1.0
    paged.copy_pages([memory[:5]], *ids, out=[memory[5:]])
    assert [bool(p.any()) for p in memory] == [True] + [False] * 5 + [True] + [False] * 2


def test_many_copies():
    """More copies than a grid has rows."""
    pool = torch.arange(140000, device=DEV, dtype=torch.int32).reshape(-1, 1, 1, 1).repeat(1, 1, 2, 4)
    n = 70000
    paged.copy_pages([pool], torch.arange(n, dtype=torch.int32, device=DEV), torch.arange(n, 2 * n, dtype=torch.int32, device=DEV))
    assert torch.equal(pool[:n], pool[n:])


@pytest.mark.parametrize("P, lens", [(100, (5, 0, 130, 1)), (256, (0, 0, 0)), (9, (3, 40))])
def test_generation_behind_a_shared_prefix(monkeypatch, P, lens):
    """Prefill, fork, attention over the suffixes and decode steps together: each call of the attention against its statement, the graph
    against eager steps, and the first logits against those of whole prompts (about 40 roundings of 2^-9 rms on either side of a
    difference, independent: 2^-9 * sqrt(80) = 0.017 of the logits' size; twice that is allowed)."""
    from scirust_b200.generate import SamplingParams
    from scirust_b200.models.infer import InferenceEngine
    from scirust_b200.models.sciagent import GQADecoder, SciAgentConfig
    model = GQADecoder(SciAgentConfig(256, 256, 2, 4, 2, 384, 512, 10000.0), device=DEV, seed=5, init_std=0.08)
    g = torch.Generator().manual_seed(P)
    prefix = torch.randint(1, 256, (P,), generator=g).to(DEV)
    suffixes = [torch.randint(1, 256, (n,), generator=g).to(DEV) for n in lens]
    B, calls, op = len(lens), [], paged.shared_prefix_attention

    def checked(q, pool, table, page, length, prefix_table, prefix_len, H, Hkv, dh, cu_q=None, max_len=None):
        o = op(q, pool, table, page, length, prefix_table, prefix_len, H, Hkv, dh, cu_q=cu_q, max_len=max_len)
        o64, bound = statement(dict(q=q, pool=pool, block_table=table, page=page, seq_len=length, H=H, Hkv=Hkv, dh=dh, cu_q=cu_q))
        assert bool(((o.to(F64) - o64).abs() <= bound).all())
        calls.append(cu_q is not None)
        return o

    eager = InferenceEngine(model, max_batch=B + 1, max_seq=512, page=16, use_graph=False)
    graph = InferenceEngine(model, max_batch=B + 1, max_seq=512, page=16)
    for e in (eager, graph):
        monkeypatch.setattr(e, "_shares", lambda B, P: True)
    for params in (None, SamplingParams(0.9, 20, 0.95, 1.1)):
        with monkeypatch.context() as m:
            m.setattr(paged, "shared_prefix_attention", checked)
            want = eager.generate_shared(prefix, suffixes, 6, params, seed=2)
        assert sum(calls) == (2 if sum(lens) else 0) and len(calls) - sum(calls) == 2 * 5
        calls.clear()
        for _ in range(2):
            assert torch.equal(graph.generate_shared(prefix, suffixes, 6, params, seed=2), want)
    seen = []
    monkeypatch.setattr(eager, "_decode_steps", lambda *a: seen.append(eager.logits[:B].float().clone()))
    eager.generate_shared(prefix, suffixes, 6)
    for b in range(B):
        whole = graph.prefill(torch.cat([prefix, suffixes[b]])[None])[0].float()
        assert (seen[0][b] - whole).norm() <= 0.034 * whole.norm()
        graph.cache.release(0)


def test_generation_with_pages_that_the_kernel_does_not_take():
    from scirust_b200.models.infer import InferenceEngine
    from scirust_b200.models.sciagent import GQADecoder, SciAgentConfig
    model = GQADecoder(SciAgentConfig(64, 128, 1, 2, 1, 128, 2048, 10000.0), device=DEV, seed=5, init_std=0.08)
    eng = InferenceEngine(model, max_batch=8, max_seq=1600, page=12)
    prefix = torch.arange(1500) % 63 + 1
    out = eng.generate_shared(prefix, 8, 4)
    assert torch.equal(out, out[:1].expand(8, -1))
    with pytest.raises(ValueError):
        eng.generate_shared(prefix, [prefix[:2]], 4)
