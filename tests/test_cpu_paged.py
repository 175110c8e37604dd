"""Ops on shared pages: the CPU statement against dense attention, and what is refused."""
import pytest
import torch

from scirust_b200.ops import paged

BF = torch.bfloat16


def batch(B=3, H=4, Hkv=2, dh=64, page=8, prefix=20, tails=(1, 9, 4), new=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    shared = prefix // page
    own = [(prefix + t + page - 1) // page - shared for t in tails]
    total = shared + sum(own) + 2
    order = torch.randperm(total, generator=g).int()
    table = torch.zeros((B, shared + max(own)), dtype=torch.int32)
    at = shared
    for b, n in enumerate(own):
        table[b, :shared] = order[:shared]
        table[b, shared:shared + n] = order[at:at + n]
        at += n
    rows = [1] * B if new is None else new
    cu = None if new is None else torch.tensor([0] + list(torch.tensor(new).cumsum(0)), dtype=torch.int32)
    return dict(q=torch.randn(sum(rows), H * dh, generator=g).to(BF), pool=torch.randn(total, 2, Hkv, page, dh, generator=g).to(BF),
                block_table=table, page=page, seq_len=torch.tensor([prefix + t for t in tails], dtype=torch.int32),
                prefix_table=order[:shared].contiguous(), prefix_len=prefix, H=H, Hkv=Hkv, dh=dh, cu_q=cu)


@pytest.mark.parametrize("new", [None, [1, 9, 3]])
def test_statement_is_dense_attention(new):
    a = batch(new=new)
    out = paged.shared_prefix_attention(**a)
    at = 0
    for b, n in enumerate(new or [1, 1, 1]):
        L = int(a["seq_len"][b])
        kv = a["pool"][a["block_table"][b].long()].double().permute(1, 2, 0, 3, 4).reshape(2, 2, -1, 64)[:, :, :L]
        for i in range(n):
            limit = L - n + i + 1
            q = a["q"][at].double().view(2, 2, 64)
            p = torch.softmax(q @ kv[0, :, :limit].transpose(1, 2) / 8, -1)
            want = (p @ kv[1, :, :limit]).reshape(-1)
            assert torch.allclose(out[at].double(), want, atol=2 ** -7 * float(want.abs().max()))
            at += 1


def test_empty_sequences_and_rows_of_no_sequence():
    a = batch(new=[1, 9, 3])
    a["seq_len"][1] = 0
    out = paged.shared_prefix_attention(**a)
    assert not out[1:10].any() and bool(out[0].any()) and bool(out[10:].any())
    a = batch(new=[1, 9, 3])
    a["q"] = torch.cat([a["q"], a["q"][:2]])
    out = paged.shared_prefix_attention(**a)
    assert not out[13:].any()
    kept = paged.shared_prefix_attention(**a, out=torch.full_like(out, 3.0))
    assert torch.equal(kept[:13], out[:13]) and bool((kept[13:] == 3).all())


@pytest.mark.parametrize("change", [
    dict(H=3), dict(page=16), dict(dh=32), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(prefix_len=-1),
    dict(prefix_len=30), dict(seq_len=torch.ones(2, dtype=torch.int32)), dict(cu_q=torch.zeros(3, dtype=torch.int32)),
    dict(q=torch.zeros(4, 256, dtype=BF)), dict(q=torch.zeros(3, 255, dtype=BF)), dict(out=torch.zeros(3, 255, dtype=BF)),
    dict(block_table=torch.zeros(3, dtype=torch.int32)), dict(block_table=torch.zeros(3, 0, dtype=torch.int32))])
def test_refusals(change):
    with pytest.raises(ValueError):
        paged.shared_prefix_attention(**{**batch(), **change})


def test_entry_point_refuses():
    """Sizes and pointers are looked at before anything is launched."""
    from scirust_b200.ops import _lib
    ok = dict(q=16, ldq=256, pool=16, n_blocks=4, table=16, max_blocks=4, page=64, seq_len=16, prefix_table=16, prefix=64, cu=None, B=2, NT=2,
              H=4, Hkv=2, dh=64, units=4, scale=0.125, ws=32, ws_bytes=1 << 30, out=16, ldo=256, fill=1, status=16, stream=None)
    for change, what in ((dict(B=0), "bad argument"), (dict(NT=3), "bad argument"), (dict(H=5), "bad argument"), (dict(dh=96), "bad argument"),
                         (dict(page=12), "bad argument"), (dict(page=4), "bad argument"), (dict(prefix=32), "bad argument"),
                         (dict(prefix_table=None), "bad argument"), (dict(scale=0.0), "bad argument"), (dict(scale=float("nan")), "bad argument"),
                         (dict(ws_bytes=100), "bad argument"), (dict(H=260), "bad argument"), (dict(q=24), "misaligned"), (dict(ldq=257), "misaligned"),
                         (dict(out=8), "misaligned"), (dict(ldo=260), "misaligned"), (dict(n_blocks=1 << 24), "size beyond"),
                         (dict(max_blocks=1 << 25), "size beyond"), (dict(B=1 << 22, NT=1 << 22, max_blocks=1 << 12), "size beyond")):
        with pytest.raises(_lib.NativeError, match=what):
            _lib.call("sb_shared_prefix_attention", *{**ok, **change}.values())


@pytest.mark.parametrize("n, B, prefix, longest, want", [
    (511, 16, 512, 0, True), (512, 16, 512, 0, False), (512, 16, 4095, 0, False), (512, 16, 4096, 0, True), (1031, 32, 16384, 1000, True),
    (2047, 16, 8192, 0, True), (2048, 16, 8192, 0, False), (1, 1, 8, 1, True), (32, 1, 64, 32, False), (1024, 16, 8192, 64, False),
    (1024, 16, 8192, 65, True), (768, 16, 8192, 48, True), (8192, 128, 8192, 0, True), (8193, 128, 8192, 0, False), (8193, 300, 8192, 0, True)])
def test_rule_of_which_rows_go_over_the_prefix_together(n, B, prefix, longest, want):
    assert paged._in_common(n, B, 32, prefix, longest) is want


def test_copy_pages_statement():
    pools = [torch.randn(6, 2, 1, 4, 8) for _ in range(2)]
    before = [p.clone() for p in pools]
    paged.copy_pages(pools, [1, 1, 0], [3, 5, 4], rows=3)
    for p, b in zip(pools, before):
        for s, d in ((1, 3), (1, 5), (0, 4)):
            assert torch.equal(p[d, :, :, :3], b[s, :, :, :3]) and torch.equal(p[d, :, :, 3:], b[d, :, :, 3:])
        assert torch.equal(p[:3], b[:3])
    other = [torch.zeros(2, 2, 1, 4, 8) for _ in range(2)]
    paged.copy_pages(pools, [1, 4], [1, 0], out=other)
    assert all(torch.equal(o[1], p[1]) and torch.equal(o[0], p[4]) for o, p in zip(other, pools))
    paged.copy_pages(pools, [], [])


@pytest.mark.parametrize("args,kw", [
    (([0], [6]), {}), (([-1], [2]), {}), (([0, 1], [2, 2]), {}), (([0, 1], [1, 2]), {}), (([0], [1, 2]), {}), (([0], [1]), dict(rows=5)),
    (([0], [1]), dict(rows=-1)), (([0], [1]), dict(out=[torch.zeros(6, 2, 1, 4, 8)])),
    (([0], [1]), dict(out=[torch.zeros(6, 2, 1, 2, 8)] * 2)), (([0], [1]), dict(out=[torch.zeros(6, 2, 1, 4, 8, dtype=BF)] * 2))])
def test_copy_pages_refusals(args, kw):
    with pytest.raises(ValueError):
        paged.copy_pages([torch.zeros(6, 2, 1, 4, 8) for _ in range(2)], *args, **kw)


def test_copies_between_pools_that_reach_into_one_another_are_refused():
    memory = torch.zeros(9, 2, 1, 4, 8)
    pools, other = [memory[:5]], [memory[3:]]
    with pytest.raises(ValueError):
        paged.copy_pages(pools, [0], [1], out=other)
    memory[0] = 1.0
    paged.copy_pages(pools, [0], [3], out=[memory[5:]])             # beside it
    paged.copy_pages(pools, [0], [2], out=[memory[:4]])             # the same pool, by fewer pages
    assert [bool(p.any()) for p in memory] == [True, False, True, False, False, False, False, False, True]


def test_copies_into_one_pool_from_two_are_refused():
    pools, into = [torch.full((6, 2, 1, 4, 8), float(i)) for i in range(2)], torch.zeros(6, 2, 1, 4, 8)
    with pytest.raises(ValueError):
        paged.copy_pages(pools, [0], [1], out=[into, into])
    assert not into.any()
    paged.copy_pages([pools[1], pools[1]], [0], [1], out=[into, pools[0]])         # from one pool to two
    assert bool(into[1].eq(1).all()) and bool(pools[0][1].eq(1).all()) and not pools[0][0].any()
    paged.copy_pages(pools, [], [], out=[into[:0], into[:0]])                      # of nothing


def test_pools_of_a_cache_that_reach_into_one_another_are_refused():
    memory = torch.zeros(9, 2, 1, 4, 8)
    with pytest.raises(ValueError):
        paged.PagePools([memory[:5], memory[3:8]])
    assert len(paged.PagePools([memory[4:8], memory[:4]])) == 2


def test_page_pools_refusals():
    for bad in ([], [torch.zeros(3, 4)], [torch.zeros(3, 2, 4, 8), torch.zeros(3, 2, 4, 7)], [torch.zeros(3, 2, 8, 4).transpose(2, 3)],
                [torch.zeros(3, 2, 4, 8), torch.zeros(3, 2, 4, 8, dtype=BF)]):
        with pytest.raises(ValueError):
            paged.PagePools(bad)


def test_copy_entry_point_refuses():
    import ctypes
    from scirust_b200.ops import _lib
    table = ctypes.addressof((ctypes.c_void_p * 1)(16))
    ok = dict(src=table, dst=table, layers=1, a=16, b=16, n=1, sb=4, db=4, page=1024, segs=1, seg=1024, pitch=1024, stream=None)
    for change, what in ((dict(src=None), "bad argument"), (dict(layers=0), "bad argument"), (dict(n=0), "bad argument"),
                         (dict(sb=0), "bad argument"), (dict(seg=0), "bad argument"), (dict(segs=2, seg=512, pitch=500), "bad argument"),
                         (dict(segs=3, seg=512, pitch=512), "bad argument"), (dict(page=1 << 31, seg=512), "size beyond")):
        with pytest.raises(_lib.NativeError, match=what):
            _lib.call("sb_copy_pages", *{**ok, **change}.values())
