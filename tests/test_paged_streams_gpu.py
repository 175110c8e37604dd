"""Attention behind a common prefix as it is called in earnest: from the streams' own workspaces, which keep what earlier calls left."""
import threading
import time

import pytest
import torch

from scirust_b200.ops import _lib, paged
from test_paged_gpu import F64, batch, statement

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _in_earnest(monkeypatch):
    """No fresh workspace for each call, and none that an earlier test has left."""
    monkeypatch.setattr(_lib, "DEBUG_POISON", False)
    monkeypatch.setattr(paged, "_ws", {})
    yield
    torch.cuda.synchronize()
    _lib.check_status(torch.device(DEV, 0))


def batches():
    """Small and large, one token a sequence and ragged, few rows and tiles of them, both head dimensions, with and without a prefix."""
    return [batch(2, 16, 4, 64, 64, 128, [5, 70], seed=1),
            batch(33, 32, 8, 128, 16, 1000, [1 + 11 * b for b in range(33)], seed=2),
            batch(5, 32, 8, 128, 64, 600, [30, 7, 200, 1, 90], [30, 7, 150, 1, 90], seed=3),
            batch(8, 32, 32, 128, 64, 512, [700] * 8, seed=4),
            batch(3, 16, 4, 64, 64, 0, [400, 1, 77], seed=5),
            batch(4, 16, 4, 64, 64, 200, [3, 300, 1, 40], [3, 290, 1, 40], seed=6),
            batch(1, 4, 1, 128, 8, 640, [9], seed=7)]


def right(a, out):
    want, bound = statement(a)
    return bool(((out.to(F64) - want).abs() <= bound).all())


def test_calls_one_after_another_share_a_workspace():
    todo = batches()
    first = [paged.shared_prefix_attention(**a) for a in todo]           # it grows
    assert all(right(a, o) for a, o in zip(todo, first)) and len(paged._ws) == 1
    (w,) = paged._ws.values()
    kept = w.buffer.data_ptr()
    for order in (range(len(todo)), reversed(range(len(todo))), [3, 0, 3, 6, 1, 4, 2, 2, 5, 0]):
        for i in order:
            assert torch.equal(paged.shared_prefix_attention(**todo[i]), first[i])
    assert w.buffer.data_ptr() == kept


def test_what_is_left_in_a_workspace_does_not_matter():
    todo = batches()
    first = [paged.shared_prefix_attention(**a) for a in todo]
    (w,) = paged._ws.values()
    for byte in (0xff, 0x7f, 0x00):                                      # NaN and -1, large numbers, zeros
        for a, o in zip(todo, first):
            w.buffer.fill_(byte)
            assert torch.equal(paged.shared_prefix_attention(**a), o)


def test_streams_have_workspaces_of_their_own():
    todo = batches()
    want = [paged.shared_prefix_attention(**a) for a in todo]
    streams, outs = [torch.cuda.Stream() for _ in range(2)], [[torch.zeros_like(w) for w in want] for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(4):
        for i in range(len(todo)):
            for s, o, j in ((streams[0], outs[0], i), (streams[1], outs[1], len(todo) - 1 - i)):
                with torch.cuda.stream(s):
                    paged.shared_prefix_attention(**todo[j], out=o[j])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for o in outs for a, b in zip(o, want))
    ws = [paged._ws[(0, s.cuda_stream)].buffer for s in streams]
    assert len(paged._ws) == 3 and ws[0].data_ptr() != ws[1].data_ptr()


def in_threads(*work):
    failed = []

    def guarded(f):
        try:
            f()
        except BaseException as e:                # noqa: B902
            failed.append(e)

    threads = [threading.Thread(target=guarded, args=(f,)) for f in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    if failed:
        raise failed[0]


def test_launches_of_a_call_stay_together(monkeypatch):
    """Two threads on one stream: while one launches what belongs together, the other does not."""
    todo = batches()[1:3]
    want = [paged.shared_prefix_attention(**a) for a in todo]
    call, guard, inside, most = _lib.call, threading.Lock(), [0], [0]

    def slow(name, *args):
        with guard:
            inside[0] += 1
            most[0] = max(most[0], inside[0])
        time.sleep(0.02)
        with guard:
            inside[0] -= 1
            return call(name, *args)

    monkeypatch.setattr(_lib, "call", slow)
    got = [[], []]
    in_threads(*[lambda i=i: got[i].extend(paged.shared_prefix_attention(**todo[i]) for _ in range(5)) for i in range(2)])
    assert most[0] == 1
    assert all(torch.equal(o, w) for g, w in zip(got, want) for o in g)


def test_threads_on_one_stream():
    todo = batches()
    want = [paged.shared_prefix_attention(**a) for a in todo]

    def run(first):
        for k in range(300):
            i = (first + k) % len(todo)
            assert torch.equal(paged.shared_prefix_attention(**todo[i]), want[i])

    in_threads(lambda: run(0), lambda: run(3), lambda: run(5))
    assert len(paged._ws) == 1


def test_a_generation_leaves_no_workspace_with_its_stream():
    from scirust_b200.models.infer import InferenceEngine
    from scirust_b200.models.sciagent import GQADecoder, SciAgentConfig
    eng = InferenceEngine(GQADecoder(SciAgentConfig(64, 512, 1, 4, 1, 128, 512, 10000.0), device=DEV, seed=5, init_std=0.08), max_batch=3, max_seq=400, page=16)
    prefix = torch.arange(300) % 63 + 1
    outs = []
    assert eng._shares(3, 300)                       # the steps go through the workspace
    for _ in range(3):
        outs.append(eng.generate_shared(prefix, 3, 6))
        outs.append(eng.generate_shared(prefix, [prefix[:5], prefix[:9]], 6)[:1])
        assert set(paged._ws) == {(0, torch.cuda.current_stream().cuda_stream)}       # the suffixes' pass
    assert all(torch.equal(o, w) for o, w in zip(outs[2:], outs))
