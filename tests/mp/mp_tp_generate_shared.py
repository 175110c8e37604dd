"""Child of the test of generation behind a common prefix on tensor-parallel ranks (CPU, gloo): every rank serves the same small decoder
through ``TPInferenceEngine.generate_shared`` and compares the logits behind the prefix and the suffixes with a single-rank prefill of the whole
prompts; all ranks must give the same tokens, greedy and sampled."""
import os
import sys

import torch
import torch.distributed as dist

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__)))))

from scirust_b200.generate import SamplingParams  # noqa: E402
from scirust_b200.models import GQADecoder, SciAgentConfig  # noqa: E402
from scirust_b200.models.infer import InferenceEngine  # noqa: E402
from scirust_b200.models.infer_tp import TPInferenceEngine  # noqa: E402


def main():
    dist.init_process_group("gloo")
    W, rank = dist.get_world_size(), dist.get_rank()
    cfg = SciAgentConfig(vocab_size=256, d_model=256, n_layers=2, n_heads=8, n_kv_heads=int(os.environ["SB_TP_KV"]), d_ff=384, max_seq_len=128)
    model = GQADecoder(cfg, seed=3, init_std=0.08)
    g = torch.Generator().manual_seed(1)
    prefix = torch.randint(1, 256, (21,), generator=g)
    suffixes = [torch.randint(1, 256, (n,), generator=g) for n in (3, 0, 11)]
    B, NEW = len(suffixes), 5
    tp = TPInferenceEngine(model, max_batch=B, max_seq=48, page=8)
    steps, first = tp._decode_steps, []

    def seen(*a):
        first.append(tp.logits[:B].float().clone())
        return steps(*a)

    tp._decode_steps = seen
    for shares in (True, False):                  # the attention that reads the prefix once, and the other
        tp._shares = lambda B, P, shares=shares: shares
        for params in (None, SamplingParams(0.9, 20, 0.95, 1.1)):
            tokens = tp.generate_shared(prefix, suffixes, NEW, params, seed=2)
            assert tokens.shape == (B, NEW) and torch.equal(tokens, tp.generate_shared(prefix, suffixes, NEW, params, seed=2))
            all_of = [torch.empty_like(tokens) for _ in range(W)]
            dist.all_gather(all_of, tokens)
            assert all(torch.equal(t, tokens) for t in all_of), "ranks disagree on the generated tokens"
            if params is None:
                assert torch.equal(tokens[:, 0], first[-1].argmax(-1))
    single = InferenceEngine(model, max_batch=1, max_seq=48, page=8)
    for b, s in enumerate(suffixes):
        # about 40 roundings of 2^-9 rms on either side of a difference, independent: 2^-9 * sqrt(80) = 0.017 of the logits' size; twice that
        whole = single.prefill(torch.cat([prefix, s])[None])[0].float()
        for logits in first:
            assert (logits[b] - whole).norm() <= 0.034 * whole.norm(), f"rank {rank}: sequence {b}"
    tp.close()
    dist.barrier()
    if rank == 0:
        print("TP_GENERATE_SHARED_OK")
    dist.destroy_process_group()


if __name__ == "__main__":
    main()
