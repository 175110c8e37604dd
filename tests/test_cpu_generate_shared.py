"""Generation of sequences with a common prefix against generation of each prompt by itself (CPU statements)."""
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from scirust_b200.generate import SamplingParams
from scirust_b200.models.infer import InferenceEngine
from scirust_b200.models.sciagent import GQADecoder, SciAgentConfig


@pytest.fixture(scope="module")
def model():
    return GQADecoder(SciAgentConfig(64, 32, 2, 4, 2, 48, 64, 10000.0), seed=5, init_std=0.3)


@pytest.fixture(autouse=True)
def _any_size(request, monkeypatch):
    """Also where the kernel that reads a prefix once would not pay."""
    if "rule" not in request.node.name:
        monkeypatch.setattr(InferenceEngine, "_shares", lambda self, B, P: True)


def alone(model, prompt, new, params=None, seed=0):
    eng = InferenceEngine(model, max_batch=1, max_seq=len(prompt) + new + 1, page=8)
    return eng.generate(torch.tensor([prompt]), new, params, seed=seed)[0].tolist()


@pytest.mark.parametrize("P", [5, 8, 19])
@pytest.mark.parametrize("params", [None, SamplingParams(0.8, 10, 0.9, 1.2)])
def test_suffixes_of_any_length(model, P, params):
    g = torch.Generator().manual_seed(P)
    prefix = torch.randint(1, 64, (P,), generator=g)
    suffixes = [torch.randint(1, 64, (n,), generator=g) for n in (3, 0, 11, 1)]
    eng = InferenceEngine(model, max_batch=5, max_seq=48, page=8)
    for _ in range(2):                                 # the engine can be used again
        out = eng.generate_shared(prefix, suffixes, 6, params, seed=3)
        for b, s in enumerate(suffixes):
            assert out[b].tolist() == alone(model, prefix.tolist() + s.tolist(), 6, params, seed=3 + b)
    again = eng.generate(torch.stack([prefix, prefix]), 6, params, seed=3)
    assert again[1].tolist() == alone(model, prefix.tolist(), 6, params, seed=4)


def test_samples_of_one_prompt_share_its_pages(model):
    prefix = torch.arange(1, 20)
    eng = InferenceEngine(model, max_batch=4, max_seq=32, page=8)
    out = eng.generate_shared(prefix, 4, 5, SamplingParams(1.0), seed=7)
    for b in range(4):
        assert out[b].tolist() == alone(model, prefix.tolist(), 5, SamplingParams(1.0), seed=7 + b)
    c = eng.cache
    assert all(c.owned[b][:2] == c.owned[0][:2] for b in range(4)) and c.alloc.owners(c.owned[0][0]) == 4
    assert len({c.owned[b][2] for b in range(4)}) == 4
    matrix = eng.generate_shared(prefix[None], torch.ones(2, 3, dtype=torch.int64), 4)
    assert torch.equal(matrix[0], matrix[1])


def test_sequences_that_do_not_take_part_keep_their_pages(model):
    eng = InferenceEngine(model, max_batch=4, max_seq=32, page=8)
    eng.prefill(torch.arange(1, 41).view(4, 10))
    kept, held = eng.cache.owned[3][:], eng.cache.pools[0][eng.cache.owned[3]].clone()
    out = eng.generate_shared(torch.arange(1, 20), 3, 5)
    assert out.tolist() == [alone(model, list(range(1, 20)), 5)] * 3
    assert eng.cache.owned[3] == kept and eng.cache.block_table[3, :2].tolist() == kept
    assert torch.equal(eng.cache.pools[0][kept], held)


def test_refusals(model):
    eng = InferenceEngine(model, max_batch=2, max_seq=16, page=8)
    p = torch.arange(1, 6)
    for args in ((p, 3, 4), (p, 2, 12), (p, [torch.ones(9, dtype=torch.int64)], 3), (p, 0, 4), (p[:0], 2, 4), (p, 2, 0), (p, [], 2), (torch.ones(2, 2, dtype=torch.int64), 2, 3)):
        with pytest.raises(ValueError):
            eng.generate_shared(*args)


def test_command_prints_a_line_for_each_sample(model, tmp_path, capsys):
    from scirust_b200 import cli
    from scirust_b200.io import checkpoint as CK
    CK.save_sciagent_checkpoint(model, tmp_path / "step_1", step=1, loss=0.0, lr=0.0)
    args = ["infer", "--checkpoint", str(tmp_path / "step_1"), "--prompt", "1 2 3 4 5 6 7 8 9", "--max-new", "4", "--device", "cpu"]
    assert cli.run(args) == 0
    one = capsys.readouterr().out.splitlines()
    assert cli.run(args + ["--samples", "3"]) == 0
    assert capsys.readouterr().out.splitlines() == one * 3           # greedy
    assert cli.run(args + ["--samples", "0"]) != 0
    assert cli.run(["sciagent", "ask"] + args[1:] + ["--samples", "2"]) != 0


@pytest.mark.parametrize("H, Hkv, dh, B, P, want", [(32, 8, 128, 2, 255, False), (32, 8, 128, 2, 256, True), (32, 8, 128, 1, 4096, False),
                                                    (16, 8, 128, 16, 511, False), (16, 8, 128, 2, 512, True), (16, 16, 64, 4, 1024, False),
                                                    (16, 16, 64, 8, 1024, True), (16, 16, 64, 64, 1000, False), (12, 4, 64, 2, 4096, True)])
def test_rule_of_which_attention_runs(H, Hkv, dh, B, P, want):
    eng = InferenceEngine(GQADecoder(SciAgentConfig(16, dh * H, 0, H, Hkv, 16, 64, 10000.0)), max_batch=1, max_seq=8, page=8)
    assert eng._shares(B, P) is want
    eng.cache.page = 12
    assert not eng._shares(B, P)


def test_rule_keeps_the_answers(model):
    eng = InferenceEngine(model, max_batch=3, max_seq=32, page=8)
    out = eng.generate_shared(torch.arange(1, 12), 3, 4)               # too little for the other kernel
    assert eng._shared is None and out.tolist() == [alone(model, list(range(1, 12)), 4)] * 3


@pytest.mark.parametrize("world, kv", [(2, 4), (4, 1)])
def test_tensor_parallel_ranks(world, kv):
    """Sharded heads, and kv heads that ranks hold in common."""
    root = Path(__file__).resolve().parents[1]
    cmd = [sys.executable, "-m", "torch.distributed.run", "--nnodes=1", f"--nproc-per-node={world}", "--master-addr", "127.0.0.1",
           "--master-port", str(29780 + world), str(root / "tests" / "mp" / "mp_tp_generate_shared.py")]
    r = subprocess.run(cmd, capture_output=True, text=True, timeout=600, env=dict(os.environ, PYTHONPATH=str(root), SB_TP_KV=str(kv)))
    assert r.returncode == 0 and "TP_GENERATE_SHARED_OK" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]
