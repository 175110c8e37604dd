"""The statements of the operators on a paged KV cache in 8 bits, against 64 bits, and what they refuse."""
import math
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from scirust_b200.generate import SamplingParams
from scirust_b200.models.infer import InferenceEngine, PagedKVCache, teacher_forced_logits
from scirust_b200.models.sciagent import GQADecoder, SciAgentConfig
from scirust_b200.ops import decode as D, quantized_kv as Q

BF, F64 = torch.bfloat16, torch.float64
KINDS = ["int8", "e4m3"]


def half_steps(x, scale, kind):
    """How far the nearest code may be from x (64 bits): half a step of the scale for int8, half a step of a three-bit mantissa, or of
    the smallest exponent's, for e4m3."""
    if kind == "int8":
        return scale / 2
    return torch.maximum(x.abs() * 2.0 ** -4, scale * 2.0 ** -10)


def values(pool):
    codes, scales = pool
    return codes.to(F64) * scales.to(F64).repeat_interleave(pool.block, -1)[..., None]


def rows(n, H, Hkv, dh, seed=0, spread=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((n, (H + 2 * Hkv) * dh), generator=g)
    if spread:
        x *= torch.exp2(torch.randint(-12, 13, (n, 1), generator=g).float())
    return x.to(BF)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page,block", [(8, 8), (16, 8), (64, 16), (64, 64)])
def test_prompts_are_within_half_a_step(kind, page, block):
    H, Hkv, dh = 3, 2, 16
    lens = [1, 2 * page + 3, page, 0, 5]
    n = sum(lens)
    x = rows(n, H, Hkv, dh)
    pool = Q.QuantPool.zeros(16, Hkv, page, dh, kind, block, "cpu")
    table = torch.arange(15).view(5, 3).int()
    cu = torch.tensor([0] + lens).cumsum(0).int()
    before = x.clone()
    Q.kv_append(x, H, Hkv, dh, pool, table, torch.tensor(lens).int(), cu_q=cu)
    assert torch.equal(x, before)
    got = values(pool)
    for b, length in enumerate(lens):
        for p in range(length):
            want = x[int(cu[b]) + p, H * dh:].to(F64).view(2, Hkv, dh)
            scale = pool.scales[table[b, p // page], :, :, p % page // block].to(F64)[..., None]
            off = (got[table[b, p // page], :, :, p % page] - want).abs()
            assert bool((off <= half_steps(want, scale, kind)).all())
            assert bool((torch.frexp(scale)[0] == 0.5).all())                                        # a power of two
            first = p // block * block
            top = x[int(cu[b]) + first:int(cu[b]) + min(first + block, length), H * dh:].to(F64).view(-1, 2, Hkv, dh).abs().amax((0, 3))
            largest = 127.5 if kind == "int8" else 448
            assert bool((top <= largest * scale[..., 0]).all() and (top > largest * scale[..., 0] / 2.02).all())     # and no larger one


@pytest.mark.parametrize("kind", KINDS)
def test_a_block_filled_token_by_token_is_within_one_step(kind):
    """The steps at least double each time the scale grows: half of the last one for the last rounding, a quarter at most for the one before,
    and so on. e4m3 halves exactly but below 2^-6 of the scale, where its step is 2^-9 of it."""
    H, Hkv, dh, page = 2, 2, 16, 32
    x = (rows(page, H, Hkv, dh, seed=3).float() * torch.exp2(torch.arange(page)[:, None] / 3 - 8)).to(BF)
    pool = Q.QuantPool.zeros(2, Hkv, page, dh, kind, 32, "cpu")
    table = torch.tensor([[1]]).int()
    for t in range(page):
        Q.kv_append(x[t:t + 1], H, Hkv, dh, pool, table, torch.tensor([t + 1]).int())
        want = x[:t + 1, H * dh:].to(F64).view(-1, 2, Hkv, dh).permute(1, 2, 0, 3)
        scale = pool.scales[1, :, :, 0].to(F64)[..., None, None]
        off = (values(pool)[1, :, :, :t + 1] - want).abs()
        assert bool((off <= (scale if kind == "int8" else torch.maximum(want.abs() * 2.0 ** -4, scale * 2.0 ** -9))).all())
    # beginning the block anew forgets the large scale
    Q.kv_append(x[:1], H, Hkv, dh, pool, table, torch.tensor([1]).int())
    assert bool((pool.scales[1, :, :, 0].to(F64)[..., None, None] < scale).all())


def test_rotation_in_front_is_the_rotation_and_then_the_append():
    from scirust_b200 import ops
    H, Hkv, dh, page = 4, 2, 16, 8
    cos, sin = ops.rope_table(64, dh, 10000.0, "cpu")
    x = rows(7, H, Hkv, dh, spread=False)
    a, b = Q.QuantPool.zeros(4, Hkv, page, dh, device="cpu"), Q.QuantPool.zeros(4, Hkv, page, dh, device="cpu")
    table, lens, cu = torch.tensor([[2, 0], [1, 3]]).int(), torch.tensor([9, 4]).int(), torch.tensor([0, 3, 7]).int()
    y = x.clone()
    ops.rope_(y, H + Hkv, dh, 1, cos, sin, positions=torch.tensor([6, 7, 8, 0, 1, 2, 3]))
    Q.rope_kv_append(x, H, Hkv, dh, cos, sin, a, table, lens, cu_q=cu)
    Q.kv_append(y, H, Hkv, dh, b, table, lens, cu_q=cu)
    assert torch.equal(x, y) and torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)


@pytest.mark.parametrize("kind", KINDS)
def test_what_a_block_cannot_hold_reads_as_nan_until_it_is_begun_anew(kind):
    H, Hkv, dh, page = 1, 2, 16, 8
    pool = Q.QuantPool.zeros(2, Hkv, page, dh, kind, device="cpu")
    table = torch.tensor([[0, 1]]).int()
    x = rows(3, H, Hkv, dh, spread=False)
    x[1, H * dh + 2] = math.inf                                       # a key of head 0
    x[2, (H + 2 * Hkv) * dh - 1] = math.nan                           # a value of head 1
    Q.kv_append(x, H, Hkv, dh, pool, table, torch.tensor([3]).int(), cu_q=torch.tensor([0, 3]).int())
    bad = torch.tensor([[True, False], [False, True]])
    assert torch.equal(pool.scales[0, :, :, 0].isnan(), bad)
    assert torch.equal(Q.read_pages(pool, [0])[0].isnan().all(-1).all(-1), bad)
    Q.kv_append(x[:1], H, Hkv, dh, pool, table, torch.tensor([4]).int())
    assert torch.equal(pool.scales[0, :, :, 0].isnan(), bad)
    Q.kv_append(x[:1], H, Hkv, dh, pool, table, torch.tensor([1]).int())
    assert not bool(pool.scales.isnan().any())


@pytest.mark.parametrize("kind", KINDS)
def test_zero_and_the_smallest_and_largest_numbers(kind):
    H, Hkv, dh, page = 0, 1, 16, 8
    for top in (0.0, 2.0 ** -133, 2.0 ** -91, 1.9921875 * 2.0 ** 127):
        x = torch.zeros((1, 2 * dh), dtype=BF)
        x[0, ::3] = -top
        x[0, 1::3] = top / 3
        pool = Q.QuantPool.zeros(1, Hkv, page, dh, kind, device="cpu")
        Q.kv_append(x, H, Hkv, dh, pool, torch.zeros((1, 1)).int(), torch.ones(1).int())
        want, scale = x.to(F64).view(2, 1, dh), pool.scales[0, :, :, 0].to(F64)[..., None]
        if kind == "e4m3" and top > 1.9 * 2.0 ** 127:         # with three bits behind the leading one that is 2^128, which fp32 does not have
            assert bool(Q.read_pages(pool, [0])[0, :, :, 0].isnan().all())
            continue
        assert bool(((values(pool)[0, :, :, 0] - want).abs() <= half_steps(want, scale, kind)).all())
        assert bool(torch.isfinite(pool.scales).all() and torch.isfinite(Q.read_pages(pool, [0]).float()).all())


def test_rows_without_a_place_are_left_out():
    H, Hkv, dh, page = 1, 1, 16, 8
    pool = Q.QuantPool.zeros(3, Hkv, page, dh, device="cpu")
    x = rows(6, H, Hkv, dh, spread=False)
    # sequence 0 has four rows but two positions; sequence 1 is an empty slot; sequence 2's page is outside the pool
    cu, lens, table = torch.tensor([0, 4, 5, 6]).int(), torch.tensor([2, 0, 1]).int(), torch.tensor([[1], [2], [3]]).int()
    Q.kv_append(x, H, Hkv, dh, pool, table, lens, cu_q=cu)
    assert bool((pool.scales[1, :, :, 0] > 0).all()) and not bool(pool.scales[[0, 2]].any())
    want = x[2:4, H * dh:].to(F64).view(2, 2, 1, dh).permute(1, 2, 0, 3)
    assert bool(((values(pool)[1, :, :, :2] - want).abs() <= pool.scales[1, :, :, :1, None].to(F64) / 2).all())


def attention(q, pool, table, lens, H, Hkv, dh, scale=None):
    page, out = pool.codes.shape[3], torch.zeros((q.shape[0], H * dh), dtype=F64)
    kv = values(pool)
    for b, n in enumerate(lens.tolist()):
        if n:
            pos = torch.arange(n)
            k, v = kv[table[b].long()[pos // page], :, :, pos % page].unbind(1)
            s = torch.einsum("kgd,jkd->kgj", q[b, :H * dh].to(F64).view(Hkv, H // Hkv, dh), k) * (dh ** -0.5 if scale is None else scale)
            out[b] = torch.einsum("kgj,jkd->kgd", torch.softmax(s, -1), v).reshape(-1)
    return out


def test_pages_outside_the_pool_hold_zeros():
    """Their scores are zeros and their values too: as a page of zeros in their place."""
    H, Hkv, dh, page = 2, 1, 16, 8
    g = torch.Generator().manual_seed(3)
    pool = Q.QuantPool.zeros(4, Hkv, page, dh, "int8", device="cpu")
    x = torch.randn((24, (H + 2 * Hkv) * dh), generator=g).to(BF)
    lens = torch.tensor([24, 20]).int()
    Q.kv_append(x, H, Hkv, dh, pool, torch.tensor([[0, 1, 2]]).int(), lens[:1], cu_q=torch.tensor([0, 24]).int())
    q = torch.randn((2, H * dh), generator=g).to(BF)
    got = Q.decode_attention(q, pool, torch.tensor([[0, -1, 2], [1, 2, 4]]).int(), lens, H, Hkv, dh)
    assert torch.equal(got, Q.decode_attention(q, pool, torch.tensor([[0, 3, 2], [1, 2, 3]]).int(), lens, H, Hkv, dh))


@pytest.mark.parametrize("kind", KINDS)
def test_attention_and_reading_back(kind):
    H, Hkv, dh, page = 4, 2, 16, 8
    g = torch.Generator().manual_seed(0)
    lens = torch.tensor([1, 17, 0, 24]).int()
    x = torch.randn((int(lens.sum()), (H + 2 * Hkv) * dh), generator=g).to(BF)
    pool = Q.QuantPool.zeros(12, Hkv, page, dh, kind, device="cpu")
    table = torch.randperm(12, generator=g).view(4, 3).int()
    cu = torch.cat([torch.zeros(1), lens.cumsum(0)]).int()
    Q.kv_append(x, H, Hkv, dh, pool, table, lens, cu_q=cu)
    q = torch.randn((4, H * dh), generator=g).to(BF)
    o = Q.decode_attention(q, pool, table, lens, H, Hkv, dh)
    want = attention(q, pool, table, lens, H, Hkv, dh)
    assert bool(((o.to(F64) - want).abs() <= 2.0 ** -8 * want.abs() + 1e-5).all()) and not bool(o[2].any())
    back = Q.read_pages(pool, table[1])
    assert torch.equal(back.to(F64), values(pool)[table[1].long()])              # powers of two: bf16 holds every value
    out = torch.empty_like(back)
    assert Q.read_pages(pool, table[1].tolist(), out) is out and torch.equal(out, back)
    # the pages read back are a pool for the attention over bf16
    from scirust_b200.ops import decode as D
    a = D.decode_attention(q[1:2], back, torch.arange(3)[None].int(), page, lens[1:2], H, Hkv, dh)
    assert torch.equal(a, o[1:2])


def test_refusals():
    H, Hkv, dh, page = 2, 1, 16, 8
    pool = Q.QuantPool.zeros(2, Hkv, page, dh, device="cpu")
    table, lens = torch.zeros((1, 2)).int(), torch.ones(1).int()
    x = rows(1, H, Hkv, dh)
    good = dict(H=H, Hkv=Hkv, dh=dh, pool=pool, block_table=table, seq_len=lens)

    def refused(fn, *a, **kw):
        with pytest.raises(ValueError):
            fn(*a, **kw)

    for bad in (dict(Hkv=2), dict(dh=32), dict(pool=(pool.codes, pool.scales[..., :0])), dict(pool=(pool.codes, pool.scales.double())),
                dict(pool=(pool.codes.float(), pool.scales)), dict(pool=(pool.codes, pool.scales[:1])), dict(block_table=table[0]),
                dict(block_table=torch.zeros((2, 2)).int()), dict(block_table=table[:, :0]), dict(H=3), dict(H=-1),
                dict(seq_len=torch.ones(2).int(), block_table=torch.zeros((2, 2)).int()), dict(cu_q=torch.zeros(3).int())):
        refused(Q.kv_append, x, **{**good, **bad})
    refused(Q.kv_append, x.float(), **good)
    refused(Q.kv_append, x[0], **good)
    refused(Q.rope_kv_append, x, H, Hkv, dh, torch.zeros((4, 4)), torch.zeros((4, 8)), pool, table, lens)
    refused(Q.rope_kv_append, x, H, Hkv, dh, torch.zeros((4, 8)).double(), torch.zeros((4, 8)).double(), pool, table, lens)
    q = x[:, :H * dh]
    Q.decode_attention(q, **good)
    for bad in (dict(H=3), dict(H=0), dict(scale=0.0), dict(scale=math.nan), dict(out=torch.zeros((1, H * dh))), dict(out=torch.zeros((2, H * dh), dtype=BF))):
        refused(Q.decode_attention, q, **{**good, **bad})
    refused(Q.decode_attention, q.float(), **good)
    refused(Q.decode_attention, q.repeat(2, 1), **good)
    for bad in ([2], [-1], torch.tensor([2]), torch.zeros((1, 1)).int()):
        refused(Q.read_pages, pool, bad)
    refused(Q.read_pages, pool, [0], out=torch.empty((1, 2, Hkv, page, dh)))
    refused(Q.read_pages, pool, [0], out=torch.empty((2, 2, Hkv, page, dh), dtype=BF))
    for bad in (dict(codes="int4"), dict(block=4), dict(block=16), dict(page=12)):
        refused(Q.QuantPool.zeros, **{**dict(n_blocks=1, Hkv=1, page=8, dh=16, device="cpu"), **bad})
    empty = Q.QuantPool.zeros(0, Hkv, page, dh, device="cpu")
    refused(Q.kv_append, x, **{**good, "pool": empty})
    refused(Q.decode_attention, q, **{**good, "pool": empty})
    headless = Q.QuantPool.zeros(2, 0, page, dh, device="cpu")
    refused(Q.kv_append, x, **{**good, "pool": headless, "Hkv": 0})
    refused(Q.decode_attention, q, **{**good, "pool": headless, "Hkv": 0})
    assert Q.read_pages(pool, []).shape == (0, 2, Hkv, page, dh)
    assert Q.QuantPool.zeros(3, 2, 64, 128, device="cpu").nbytes() == 3 * 2 * 2 * 64 * (128 + 4 / 16)


# ---------------------------------------------------------------------------------------------------------------- the engine
@pytest.fixture(scope="module")
def model():
    return GQADecoder(SciAgentConfig(64, 32, 2, 4, 2, 48, 64, 10000.0), seed=5, init_std=0.3)


def read_all(pool):
    return Q.read_pages(pool, list(range(pool.codes.shape[0])))


@pytest.mark.parametrize("kind", KINDS)
def test_engine_steps_attend_to_what_the_cache_holds(model, kind, monkeypatch):
    """A step over the cache in 8 bits, and the same step of an engine whose bf16 cache is given the values that the codes stand for."""
    prompts = torch.randint(1, 64, (3, 11), generator=torch.Generator().manual_seed(0))
    tokens = torch.randint(1, 64, (3, 5), generator=torch.Generator().manual_seed(1))
    eng = InferenceEngine(model, max_batch=3, max_seq=32, page=16, kv=kind, kv_block=8)
    got = teacher_forced_logits(eng, prompts, tokens)
    other = InferenceEngine(model, max_batch=3, max_seq=32, page=16)
    other.prefill(prompts)
    for b in range(3):
        other.cache.reserve(b, 17)
    other.cache.commit()
    assert torch.equal(other.cache.block_table, eng.cache.block_table)
    other.cache.pools[:] = [read_all(p) for p in eng.cache.pools]
    other.cache.seq_len[:3] = 15
    other._seq_of, other._len_plus1, other._generated = torch.arange(3, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), None
    other.tokens[:3] = tokens[:, 4]
    append = D.rope_kv_append

    def only_rotate(qkv, H, Hkv, dh, cos, sin, pool, *rest):
        append(qkv, H, Hkv, dh, cos, sin, pool.clone(), *rest)

    monkeypatch.setattr(D, "rope_kv_append", only_rotate)
    other._step_eager(3, 17, want_logits=True)
    assert torch.equal(other.logits[:3].float(), got[:, 4])


@pytest.mark.parametrize("kind", KINDS)
def test_engine_generates(model, kind):
    prompts = torch.randint(1, 64, (2, 13), generator=torch.Generator().manual_seed(2))
    eng = InferenceEngine(model, max_batch=4, max_seq=40, page=8, kv=kind)
    whole = eng.generate(prompts, 9)
    assert whole.shape == (2, 9) and torch.equal(whole, eng.generate(prompts, 9))
    alone = InferenceEngine(model, max_batch=1, max_seq=40, page=8, kv=kind)
    assert torch.equal(alone.generate(prompts[1:], 9), whole[1:])
    # sequences behind a common prefix: without suffixes the pages are the prompt's
    assert torch.equal(eng.generate_shared(prompts[0], 3, 9), whole[:1].expand(3, -1))
    suffixes = [torch.tensor([3, 4, 5]), torch.tensor([], dtype=torch.int64), torch.arange(1, 12)]
    for params in (None, SamplingParams(0.8, 10, 0.9)):
        out = eng.generate_shared(prompts[0], suffixes, 6, params, seed=1)
        assert out.shape == (3, 6) and torch.equal(out, eng.generate_shared(prompts[0], suffixes, 6, params, seed=1))


@pytest.mark.parametrize("kind", KINDS)
def test_suffixes_attend_to_the_pages_read_back(model, kind, monkeypatch):
    """The pass over suffixes gives what it gives on a bf16 cache that holds the codes' values, with the suffixes' own as well."""
    from scirust_b200.ops import paged
    prefix, suffixes = torch.arange(1, 20), [torch.tensor([3, 4, 5]), torch.arange(20, 31)]
    seen = []
    attend = paged.shared_prefix_attention

    def watch(q, pool, table, page, total, prefix_table, P, *a, **kw):
        out = attend(q, pool, table, page, total, prefix_table, P, *a, **kw)
        seen.append((pool.clone(), table, prefix_table, out))
        return out

    monkeypatch.setattr(paged, "shared_prefix_attention", watch)
    eng = InferenceEngine(model, max_batch=2, max_seq=40, page=8, kv=kind)
    eng.generate_shared(prefix, suffixes, 1)
    assert len(seen) == 2
    c = eng.cache
    for li, (pool, table, prefix_table, _) in enumerate(seen):
        every = read_all(c.pools[li])
        assert prefix_table.tolist() == table[0, :2].tolist() == table[1, :2].tolist()
        for b, n in enumerate((22, 30)):
            pages = -(-n // 8)
            assert torch.equal(pool[table[b, :pages].long()], every[c.owned[b][:pages]])


@pytest.mark.parametrize("kind", KINDS)
def test_cache_forks_compacts_and_grows(kind):
    H, Hkv, dh, page = 1, 2, 16, 16
    cache = PagedKVCache(2, 9, Hkv, dh, page, 4, 48, torch.device("cpu"), kind, 8)
    for seq, n in ((3, 5), (0, 43)):
        cache.reserve(seq, n)
    cache.commit()
    lens, cu = torch.tensor([43, 0, 0, 5]).int(), torch.tensor([0, 43, 43, 43, 48]).int()
    for li, pool in enumerate(cache.pools):
        Q.kv_append(rows(48, H, Hkv, dh, seed=li), H, Hkv, dh, pool, cache.block_table, lens, cu_q=cu)

    def held(li, seq, n):
        v = Q.read_pages(cache.pools[li], cache.owned[seq]).permute(1, 2, 0, 3, 4).reshape(2, Hkv, -1, dh)
        return v[:, :, :n].clone()

    before = [(held(li, 0, 43), held(li, 3, 5)) for li in range(2)]
    cache.fork(0, [1, 2], 41)
    cache.commit()
    assert cache.owned[1][:2] == cache.owned[0][:2] and cache.owned[1][2] != cache.owned[0][2]
    for li in range(2):
        assert torch.equal(held(li, 1, 41), before[li][0][:, :, :41])
    cache.release(1)
    assert cache.compact() == 5
    cache.resize(12)
    assert cache.pools[0].codes.shape[0] == 12 and cache.pools[0].codes.dtype is Q.CODES[kind] and cache.pools[0].scales.shape[0] == 12
    cache.resize(5)
    for li in range(2):
        assert torch.equal(held(li, 0, 43), before[li][0]) and torch.equal(held(li, 3, 5), before[li][1])
        assert torch.equal(held(li, 2, 41), before[li][0][:, :, :41])
    # the forked sequence writes on in its own page: the other's stays
    x = rows(1, H, Hkv, dh, seed=9, spread=False)
    Q.kv_append(x * 64, H, Hkv, dh, cache.pools[0], cache.block_table[2:3], torch.tensor([42]).int())
    assert torch.equal(held(0, 0, 43), before[0][0])


def test_engine_refusals(model):
    for bad in (dict(kv="int4"), dict(kv="int8", kv_block=12), dict(kv="int8", page=12), dict(kv="e4m3", page=8, kv_block=16)):
        with pytest.raises(ValueError):
            InferenceEngine(model, **{**dict(max_batch=1, max_seq=16, page=16), **bad})


def test_command_takes_the_cache_type(model, tmp_path, capsys):
    from scirust_b200 import cli
    from scirust_b200.io import checkpoint as CK
    CK.save_sciagent_checkpoint(model, tmp_path / "c", step=1, loss=0.0, lr=0.0)
    assert cli.run(["infer", "--checkpoint", str(tmp_path / "c"), "--prompt", "1 2 3", "--max-new", "4", "--kv", "int8", "--device", "cpu"]) == 0
    assert len(capsys.readouterr().out.splitlines()) == 1


@pytest.mark.parametrize("kind", KINDS)
def test_a_rotation_without_positions_leaves_all_rows(kind):
    H, Hkv, dh, page = 2, 1, 16, 8
    x, pool = rows(3, H, Hkv, dh), Q.QuantPool.zeros(3, Hkv, page, dh, kind, device="cpu")
    before, none = x.clone(), torch.empty((0, dh // 2))
    for cu in (None, torch.arange(4).int()):
        Q.rope_kv_append(x, H, Hkv, dh, none, none, pool, torch.arange(3).int()[:, None], torch.tensor([1, 3, 1]).int(), cu_q=cu)
    assert torch.equal(x, before) and not bool(pool.codes.view(torch.int8).any()) and not bool(pool.scales.any())


@pytest.mark.parametrize("world, kv", [(2, 4), (4, 1)])
def test_tensor_parallel_ranks(world, kv):
    """Sharded kv heads, and kv heads that ranks hold in common."""
    root = Path(__file__).resolve().parents[1]
    cmd = [sys.executable, "-m", "torch.distributed.run", "--nnodes=1", f"--nproc-per-node={world}", "--master-addr", "127.0.0.1",
           "--master-port", str(29840 + world), str(root / "tests" / "mp" / "mp_tp_quantized_kv.py")]
    r = subprocess.run(cmd, capture_output=True, text=True, timeout=600, env=dict(os.environ, PYTHONPATH=str(root), SB_TP_KV=str(kv)))
    assert r.returncode == 0 and "TP_QUANTIZED_KV_OK" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]
