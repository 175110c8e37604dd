"""The cache in 8 bits with the workspaces that calls keep: graphs, streams, threads, and the engine that decodes over it."""
import threading

import pytest
import torch

from scirust_b200.generate import SamplingParams
from scirust_b200.models.infer import InferenceEngine, PagedKVCache, teacher_forced_logits
from scirust_b200.models.sciagent import GQADecoder, SciAgentConfig
from scirust_b200.ops import _lib, decode as D, paged, quantized_kv as Q

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
DEV = "cuda"
KINDS = ["int8", "e4m3"]


def make(kind, H, Hkv, dh, page, lens, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    pages = [-(-n // page) for n in lens]
    order = torch.randperm(sum(pages), generator=g, device=DEV).int()
    table = torch.zeros((len(lens), max(pages)), dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n]
        at += n
    pool = Q.QuantPool.zeros(sum(pages), Hkv, page, dh, kind, device=DEV)
    qkv = torch.randn((sum(lens), (H + 2 * Hkv) * dh), generator=g, device=DEV).to(BF)
    seq_len = torch.tensor(lens, dtype=torch.int32, device=DEV)
    cu = torch.tensor([0] + lens).cumsum(0).int().to(DEV)
    Q.kv_append(qkv, H, Hkv, dh, pool, table, seq_len, cu_q=cu)
    q = torch.randn((len(lens), H * dh), generator=g, device=DEV).to(BF)
    return dict(q=q, pool=pool, block_table=table, seq_len=seq_len, H=H, Hkv=Hkv, dh=dh)


CUT = [3000, 5000, 1, 2500]                    # jobs that are cut and joined


def test_two_graphs_of_one_stream_at_once():
    """Graphs captured on one stream and replayed on two: each has parts and counters of its own."""
    cases = [make("int8", 8, 2, 128, 64, CUT, seed=1), make("e4m3", 8, 2, 128, 16, CUT[::-1], seed=2)]
    want = [Q.decode_attention(**c) for c in cases]
    s, graphs, outs = torch.cuda.Stream(), [], []
    s.wait_stream(torch.cuda.current_stream())
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            o = [Q.decode_attention(**c) for _ in range(3)]
        graphs.append(g)
        outs.append(o)
    others = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(10):
        for o in outs:
            for t in o:
                t.zero_()
        torch.cuda.synchronize()
        for g, st in zip(graphs, others):
            with torch.cuda.stream(st):
                for _ in range(5):
                    g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert all(torch.equal(t, w) for t in o)
    _lib.check_status()


def test_a_graph_beside_eager_calls_of_its_stream():
    c, d = make("int8", 8, 2, 64, 16, CUT, seed=3), make("int8", 20, 1, 128, 64, CUT, seed=4)
    want, other = Q.decode_attention(**c), Q.decode_attention(**d)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        Q.decode_attention(**c)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = Q.decode_attention(**c)
    for _ in range(5):
        out.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            eager = [Q.decode_attention(**d) for _ in range(4)]
        g.replay()                                # on the current stream
        torch.cuda.synchronize()
        assert torch.equal(out, want) and all(torch.equal(e, other) for e in eager)


def test_a_captured_step_follows_its_lengths_and_tables():
    """Write and attention replayed while the lengths on the device grow, from inside a block over the end of a page."""
    H, Hkv, dh, page = 8, 2, 128, 16
    pool = Q.QuantPool.zeros(12, Hkv, page, dh, "int8", device=DEV)
    eager = Q.QuantPool.zeros(12, Hkv, page, dh, "int8", device=DEV)
    table = torch.randperm(12, device=DEV).int().view(2, 6)
    lens = torch.tensor([9, 14], dtype=torch.int32, device=DEV)
    cos, sin = (torch.randn((128, dh // 2), device=DEV) for _ in range(2))
    step = torch.zeros((2, (H + 2 * Hkv) * dh), dtype=BF, device=DEV)
    data = [torch.randn(step.shape, device=DEV).to(BF) for _ in range(30)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        Q.rope_kv_append(step, H, Hkv, dh, cos, sin, pool, table, lens)
        out = Q.decode_attention(step, pool, table, lens, H, Hkv, dh)
    for x in data:
        lens += 1
        step.copy_(x)
        g.replay()
        y = x.clone()
        Q.rope_kv_append(y, H, Hkv, dh, cos, sin, eager, table, lens)
        assert torch.equal(out, Q.decode_attention(y, eager, table, lens, H, Hkv, dh))
    assert torch.equal(pool.codes, eager.codes) and torch.equal(pool.scales, eager.scales)


def test_streams_and_threads_at_once():
    cases = [make(k, 8, 2, 128, 64, CUT, seed=i) for i, k in enumerate(KINDS * 2)]
    want = [Q.decode_attention(**c) for c in cases]
    torch.cuda.synchronize()
    bad = []

    def work(i, stream):
        with torch.cuda.stream(stream):
            for _ in range(50):
                if not torch.equal(Q.decode_attention(**cases[i]), want[i]):
                    bad.append(i)

    shared = torch.cuda.Stream()
    for streams in ([torch.cuda.Stream() for _ in cases], [shared] * len(cases)):      # each its own, and all one
        threads = [threading.Thread(target=work, args=(i, s)) for i, s in enumerate(streams)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    torch.cuda.synchronize()
    assert not bad


def test_workspaces_are_given_back():
    s = torch.cuda.Stream()
    c = make("int8", 8, 2, 128, 64, CUT)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        Q.decode_attention(**c)
    assert any(k[1] == s.cuda_stream for k in Q._ws)
    torch.cuda.synchronize()
    Q.drop_workspace(torch.device("cuda", torch.cuda.current_device()), s.cuda_stream)
    assert not any(k[1] == s.cuda_stream for k in Q._ws)


def test_more_jobs_than_the_workspace_began_with():
    c = make("int8", 40, 20, 64, 8, [20] * 300)              # 6000 counters
    want = Q.decode_attention(**c)
    assert torch.equal(want, Q.decode_attention(**c)) and bool(torch.isfinite(want).all())


# ---------------------------------------------------------------------------------------------------------------- the engine
@pytest.fixture(scope="module", params=[(64, 16), (128, 8)], ids=["dh64", "dh128"])
def model(request):
    dh, H = request.param
    return GQADecoder(SciAgentConfig(1024, dh * H, 2, H, 2, 512, 512, 10000.0), device=DEV, seed=5, init_std=0.05)


@pytest.mark.parametrize("kv", KINDS)
def test_engine_graph_equals_eager(model, kv):
    prompts = torch.randint(1, 1024, (3, 100), generator=torch.Generator().manual_seed(1)).to(DEV)
    engines = [InferenceEngine(model, max_batch=3, max_seq=200, page=16, use_graph=g, kv=kv) for g in (False, True)]
    for params in (None, SamplingParams(0.8, 20, 0.9)):
        a, b = (e.generate(prompts, 40, params, seed=3) for e in engines)
        assert torch.equal(a, b) and torch.equal(a, engines[1].generate(prompts, 40, params, seed=3))
    _lib.check_status()


@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("quant", [None, "int8"])
def test_engine_steps_attend_to_what_the_cache_holds(model, kv, quant, monkeypatch):
    """A step over the cache in 8 bits, and the same step of an engine whose bf16 cache is given the values that the codes stand for: the same
    mathematics, with P in fp16 in one and in bf16 in the other and a rotation that is fused in one. About 16 roundings of 2^-9 rms on
    either side of a difference, independent: 2^-9 * sqrt(32) = 0.011 of the logits' size; three times that."""
    prompts = torch.randint(1, 1024, (3, 100), generator=torch.Generator().manual_seed(0)).to(DEV)
    tokens = torch.randint(1, 1024, (3, 5), generator=torch.Generator().manual_seed(1)).to(DEV)
    eng = InferenceEngine(model, quant=quant, max_batch=3, max_seq=128, page=16, kv=kv)
    got = teacher_forced_logits(eng, prompts, tokens)
    other = InferenceEngine(model, quant=quant, max_batch=3, max_seq=128, page=16)
    other.prefill(prompts)
    for b in range(3):
        other.cache.reserve(b, 106)
    other.cache.commit()
    assert torch.equal(other.cache.block_table, eng.cache.block_table)
    other.cache.pools[:] = [Q.read_pages(p, list(range(p.codes.shape[0]))) for p in eng.cache.pools]
    other.cache.seq_len[:3] = 104
    other._seq_of, other._len_plus1 = torch.arange(3, dtype=torch.int32, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV)
    other._generated = None
    other.tokens[:3] = tokens[:, 4]
    append = D.rope_kv_append

    def only_rotate(qkv, H, Hkv, dh, cos, sin, pool, *rest):
        append(qkv, H, Hkv, dh, cos, sin, pool.clone(), *rest)

    monkeypatch.setattr(D, "rope_kv_append", only_rotate)
    other._step_eager(3, 106, want_logits=True)
    want = other.logits[:3].float()
    assert bool(((want - got[:, 4]).norm(dim=1) <= 0.033 * want.norm(dim=1)).all())
    _lib.check_status()


@pytest.mark.parametrize("kv", KINDS)
def test_engine_behind_a_common_prefix(model, kv, monkeypatch):
    prefix = torch.randint(1, 1024, (70,), generator=torch.Generator().manual_seed(2)).to(DEV)
    suffixes = [torch.randint(1, 1024, (n,), generator=torch.Generator().manual_seed(n)) for n in (5, 0, 33)]
    eng = InferenceEngine(model, max_batch=4, max_seq=192, page=16, kv=kv)
    out = eng.generate_shared(prefix, suffixes, 20, SamplingParams(0.8, 20, 0.9), seed=1)
    assert out.shape == (3, 20) and torch.equal(out, eng.generate_shared(prefix, suffixes, 20, SamplingParams(0.8, 20, 0.9), seed=1))
    # without suffixes all sequences are the prompt's; the first token is chosen as for it alone (later ones by a batch's products, which may
    # differ in the last bits from one sequence's)
    alone, three = eng.generate(prefix[None], 20), eng.generate_shared(prefix, 3, 20)
    assert torch.equal(three, three[:1].expand(3, -1)) and three[0, 0] == alone[0, 0]
    # the pass over the suffixes reads what the pages stand for
    seen, attend = [], paged.shared_prefix_attention

    def watch(q, pool, table, *a, **kw):
        seen.append((pool.clone(), table.clone()))
        return attend(q, pool, table, *a, **kw)

    monkeypatch.setattr(paged, "shared_prefix_attention", watch)
    eng.generate_shared(prefix, suffixes, 1)
    assert len(seen) == 2
    for li, (pool, table) in enumerate(seen):
        every = Q.read_pages(eng.cache.pools[li], list(range(eng.cache.pools[li].codes.shape[0])))
        for b, n in enumerate((75, 70, 103)):
            pages = -(-n // 16)
            assert torch.equal(pool[table[b, :pages].long()], every[eng.cache.owned[b][:pages]])
    _lib.check_status()


@pytest.mark.parametrize("kv", ["int8", "e4m3"])
@pytest.mark.parametrize("Hkv,page,block", [(1, 8, 8), (1, 16, 16), (3, 64, 16)])
def test_cache_forks_compacts_and_grows(kv, Hkv, page, block):
    """Down to a page whose scales are 8 bytes."""
    H, dh, n = 4 * Hkv, 64, 5 * page // 2
    cache = PagedKVCache(2, 9, Hkv, dh, page, 4, 3 * page, torch.device(DEV), kv, block)
    cache.reserve(3, 5)
    cache.reserve(0, n)
    cache.commit()
    lens, cu = (torch.tensor(t, dtype=torch.int32, device=DEV) for t in ([n, 0, 0, 5], [0, n, n, n, n + 5]))
    g = torch.Generator(device=DEV).manual_seed(0)
    for pool in cache.pools:
        Q.kv_append(torch.randn((n + 5, (H + 2 * Hkv) * dh), generator=g, device=DEV).to(BF), H, Hkv, dh, pool, cache.block_table, lens, cu_q=cu)
    q = torch.randn((4, H * dh), generator=g, device=DEV).to(BF)[:1].repeat(4, 1)

    def answers(lens):
        return [Q.decode_attention(q, pool, cache.block_table, lens, H, Hkv, dh) for pool in cache.pools]

    before = answers(lens)
    cache.fork(0, [1, 2], n)
    cache.release(1)
    lens[2] = n
    cache.compact()
    cache.resize(12)
    cache.resize(5)
    cache.commit()
    for a, b in zip(answers(lens), before):
        assert torch.equal(a[[0, 3]], b[[0, 3]]) and torch.equal(a[2], b[0]) and not bool(a[1].any())


def test_engine_refusals():
    m = GQADecoder(SciAgentConfig(64, 128, 1, 4, 2, 128, 64, 10000.0), device=DEV)                # heads of 32
    with pytest.raises(ValueError):
        InferenceEngine(m, max_batch=1, max_seq=32, page=16, kv="int8")
    m = GQADecoder(SciAgentConfig(64, 128, 1, 2, 2, 128, 64, 10000.0), device=DEV)
    with pytest.raises(ValueError):
        InferenceEngine(m, max_batch=1, max_seq=32, page=24, kv="int8", kv_block=8)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_another_device_than_the_current_one():
    c = make("int8", 8, 2, 128, 64, CUT)
    want = Q.decode_attention(**c)
    there = {k: (Q.QuantPool(*(t.to("cuda:1") for t in v)) if isinstance(v, Q.QuantPool) else v.to("cuda:1") if torch.is_tensor(v) else v) for k, v in c.items()}
    assert torch.equal(Q.decode_attention(**there).to(DEV), want)
    assert torch.equal(Q.read_pages(there["pool"], [0, 1]).to(DEV), Q.read_pages(c["pool"], [0, 1]))
