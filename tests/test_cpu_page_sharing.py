"""Pages with several owners: the allocator's counts against a plain model of them, and the cache's fork, release, compact and resize."""
import random

import pytest
import torch

from scirust_b200.models.infer import BlockAllocator, PagedKVCache


def test_a_page_is_free_with_its_last_owner():
    a = BlockAllocator(4)
    x, y = a.alloc(2)
    a.share([x, x, y])
    assert (a.owners(x), a.owners(y), a.num_free()) == (3, 2, 2)
    a.free([x, y, x])
    assert (a.owners(x), a.owners(y), a.num_free()) == (1, 1, 2)
    a.free([y, x])
    assert (a.owners(x), a.owners(y), a.num_free()) == (0, 0, 4)
    assert a.alloc(2) == [x, y]                       # the last returned first
    for ids in ([3], [x, 7], [-1]):
        with pytest.raises(ValueError):
            a.share(ids)
    assert a.owners(x) == 1                            # a refused call changes nothing
    with pytest.raises(ValueError):
        a.free([x, x, x, y, y])
    assert (a.owners(x), a.owners(y), a.num_free()) == (1, 1, 2)
    with pytest.raises(ValueError):
        a.owners(4)


def test_more_owners_than_a_page_has_are_refused():
    a = BlockAllocator(4)
    one, two = a.alloc(2)
    a.share([two])
    for ids in ([one, one], [two, two, two], [one, two, one], [3], [two, 3]):
        with pytest.raises(ValueError):
            a.free(ids)
        assert (a.owners(one), a.owners(two), a.num_free()) == (1, 2, 2)
    a.free([two, one, two])
    assert sorted(a.alloc(4)) == [0, 1, 2, 3]            # each once


def test_random_histories_of_owners():
    rng = random.Random(3)
    for _ in range(20):
        n = rng.randint(1, 30)
        a, count = BlockAllocator(n), {}
        for _ in range(200):
            k = rng.random()
            if k < 0.35:
                want = rng.randint(0, 4)
                if want <= n - len(count):
                    for i in a.alloc(want):
                        assert i not in count and 0 <= i < n
                        count[i] = 1
                else:
                    with pytest.raises(MemoryError):
                        a.alloc(want)
            elif k < 0.6 and count:
                ids = rng.choices(list(count), k=rng.randint(1, 5))
                a.share(ids)
                for i in ids:
                    count[i] += 1
            elif k < 0.95 and count:
                ids = [i for i in rng.choices(list(count), k=rng.randint(1, 5))]
                ids = [i for j, i in enumerate(ids) if ids[:j + 1].count(i) <= count[i]]
                a.free(ids)
                for i in ids:
                    count[i] -= 1
                count = {i: c for i, c in count.items() if c}
            else:
                m = rng.choice([n, rng.randint(1, n + 5)])
                if len(count) > m:
                    with pytest.raises(MemoryError):
                        a.compact(m)
                    continue
                to = a.compact(m)
                assert [to[i] >= 0 for i in range(n)] == [i in count for i in range(n)]
                assert sorted(to[i] for i in count) == list(range(len(count)))
                assert all(to[i] == i for i in count if i < len(count))
                count, n = {to[i]: c for i, c in count.items()}, m
            assert a.num_free() == n - len(count)
            assert all(a.owners(i) == count.get(i, 0) for i in range(n))


def cache(max_batch=5, max_seq=40, page=8, n_blocks=20):
    c = PagedKVCache(2, n_blocks, 2, 4, page, max_batch, max_seq, "cpu")
    for p in c.pools:
        p.copy_(torch.randn(p.shape))
    return c


def held(c, seq, n):
    """What sequence seq holds: [layers][2, Hkv, n, dh]."""
    pos = torch.arange(n)
    return [p[c.table_host[seq].long()[pos // c.page], :, :, pos % c.page].clone() for p in c.pools]


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("n", [0, 1, 7, 8, 20, 24])
def test_fork(n):
    c = cache()
    c.reserve(0, 24)
    before, free = held(c, 0, n), c.alloc.num_free()
    c.fork(0, [1, 3], n)
    c.commit()
    assert c.alloc.num_free() == free - (2 if n % 8 else 0)
    assert torch.equal(c.block_table, c.table_host)
    for s in (1, 3):
        assert same(held(c, s, n), before) and len(c.owned[s]) == (n + 7) // 8
        c.reserve(s, 30)
    assert c.table_host[1, n // 8] != c.table_host[3, n // 8] != c.table_host[0, n // 8]       # each writes on in its own
    for p in c.pools:
        p[c.table_host[1, n // 8]] = 9
    assert same(held(c, 0, n), before) and same(held(c, 3, n), before)
    c.release(0)
    assert same(held(c, 3, n), before)
    c.release(3)
    c.release(1)
    assert c.alloc.num_free() == 20


def test_fork_refusals_change_nothing():
    c = cache(n_blocks=4)
    c.reserve(0, 20)
    for src, seqs, n in ((0, [1], 33), (0, [0], 4), (0, [1, 1], 4), (0, [5], 4), (-1, [1], 4), (0, [1], -1), (2, [1], 1)):
        with pytest.raises(ValueError):
            c.fork(src, seqs, n)
    with pytest.raises(MemoryError):
        c.fork(0, [1, 2], 20)                          # one page is left
    assert c.alloc.num_free() == 1 and not c.owned[1] and not c.owned[2]
    c.fork(0, [1], 20)
    with pytest.raises(ValueError):
        c.fork(0, [1], 4)                              # has pages


@pytest.mark.parametrize("size", [None, 10, 50])
def test_compact_and_resize_keep_what_sequences_hold(size):
    c = cache()
    for s, n in ((0, 20), (1, 33), (2, 9)):
        c.reserve(s, n)
    c.fork(1, [3], 27)
    c.release(0)
    c.reserve(3, 40)
    c.commit()
    before = {s: held(c, s, n) for s, n in ((1, 33), (2, 9), (3, 27))}
    live = 20 - c.alloc.num_free()
    if size is None:
        assert c.compact() == live
    else:
        pools = c.pools
        c.resize(size)
        assert c.pools is pools and all(p.shape[0] == size for p in pools) and c.alloc.num_free() == size - live
    assert max(max(o) for o in c.owned if o) == live - 1
    assert torch.equal(c.block_table, c.table_host)
    assert all(same(held(c, s, b[0].shape[0]), b) for s, b in before.items())
    assert c.alloc.owners(c.owned[1][0]) == 2
    with pytest.raises(MemoryError):
        c.resize(live - 1)
    for s in (1, 2, 3):
        c.release(s)
    assert c.alloc.num_free() == (size or 20)
    assert c.compact() == 0
