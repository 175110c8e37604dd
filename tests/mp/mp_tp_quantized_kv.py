"""Child of the test of a cache in 8 bits on tensor-parallel ranks (CPU, gloo): every rank decodes with ``TPInferenceEngine(kv=...)`` from prompts
and behind a common prefix. What its first layer's pages hold is compared with the heads of a single-rank engine's, the logits with that
engine's; all ranks must give the same tokens, greedy and sampled."""
import os
import sys

import torch
import torch.distributed as dist

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__)))))

from scirust_b200.generate import SamplingParams  # noqa: E402
from scirust_b200.models import GQADecoder, SciAgentConfig  # noqa: E402
from scirust_b200.models.infer import InferenceEngine, teacher_forced_logits  # noqa: E402
from scirust_b200.models.infer_tp import TPInferenceEngine  # noqa: E402
from scirust_b200.ops import quantized_kv as Q  # noqa: E402

# Of the logits' size. Some 40 roundings of 2^-9 rms on either side, independent: 2^-9 * sqrt(80) = 0.017. A key or value that differs by d gets
# another code with probability d / step, so its codes differ by sqrt(d * step) rms: with d = 2^-9 of it and steps of 2^-5 (int8, a
# value of half of its block's power of two) or 2^-3 (e4m3) of it 2^-7 and 2^-6. Each of two layers passes it on through the scores and the
# values: twice that. sqrt(0.017^2 + (2 * 2^-7)^2) = 0.023 and sqrt(0.017^2 + (2 * 2^-6)^2) = 0.036; twice these.
TOLERANCE = {"int8": 0.046, "e4m3": 0.072}


def values(pool, heads=slice(None)):
    codes, scales = pool.codes[:, :, heads], pool.scales[:, :, heads]
    steps = scales.repeat_interleave(pool.block, -1)[..., None]
    return codes.float() * steps, steps


def main():
    dist.init_process_group("gloo")
    W, rank = dist.get_world_size(), dist.get_rank()
    Hkv = int(os.environ["SB_TP_KV"])
    cfg = SciAgentConfig(vocab_size=256, d_model=256, n_layers=2, n_heads=8, n_kv_heads=Hkv, d_ff=384, max_seq_len=128)
    model = GQADecoder(cfg, seed=3, init_std=0.08)
    g = torch.Generator().manual_seed(1)
    prefix = torch.randint(1, 256, (21,), generator=g)
    suffixes = [torch.randint(1, 256, (n,), generator=g) for n in (3, 0, 11)]
    prompts, fed = torch.randint(1, 256, (3, 13), generator=g), torch.randint(1, 256, (3, 7), generator=g)
    first = rank * Hkv // W
    heads = slice(first, first + max(1, Hkv // W))

    def same_on_all_ranks(tokens):
        all_of = [torch.empty_like(tokens) for _ in range(W)]
        dist.all_gather(all_of, tokens)
        assert all(torch.equal(t, tokens) for t in all_of), "ranks disagree on the generated tokens"

    def close(a, b):
        assert bool(((a - b).norm(dim=-1) <= TOLERANCE[kind] * b.norm(dim=-1)).all()), f"rank {rank}, {kind}"

    for kind in ("int8", "e4m3"):
        size = dict(max_batch=3, max_seq=48, page=16, kv=kind, kv_block=8)
        engines = TPInferenceEngine(model, **size), InferenceEngine(model, **size)
        tp, single = engines
        assert tp.cache.pools[0].codes.shape[2] == heads.stop - heads.start and tp.cache.pools[0].codes.dtype is Q.CODES[kind]
        # prompts, and steps that are fed the same tokens
        got, want = (teacher_forced_logits(e, prompts, fed) for e in engines)
        close(got, want)
        # the first layer's rows differ by their last bit at most, and so by one step of their codes (e4m3: of at most 2^-3 of the value)
        (a, step), (b, _) = values(tp.cache.pools[0]), values(single.cache.pools[0], heads)
        assert bool(((a - b).abs() <= (step if kind == "int8" else torch.maximum(step * 2.0 ** -9, b.abs() * 2.0 ** -3))).all())
        for params in (None, SamplingParams(0.9, 20, 0.95, 1.1)):
            tokens = tp.generate(prompts, 6, params, seed=2)
            assert tokens.shape == (3, 6) and torch.equal(tokens, tp.generate(prompts, 6, params, seed=2))
            same_on_all_ranks(tokens)
        # behind a common prefix, whose pages the suffixes read back
        seen = {}
        for e in engines:
            steps = e._decode_steps

            def watch(*args, e=e, steps=steps):
                seen[e] = e.logits[:3].float().clone()
                return steps(*args)

            e._decode_steps = watch
            for params in (SamplingParams(0.9, 20, 0.95, 1.1), None):
                tokens = e.generate_shared(prefix, suffixes, 5, params, seed=2)
                assert tokens.shape == (3, 5)
                if e is tp:
                    same_on_all_ranks(tokens)
        close(seen[tp], seen[single])
        tp.close()
    dist.barrier()
    if rank == 0:
        print("TP_QUANTIZED_KV_OK")
    dist.destroy_process_group()


if __name__ == "__main__":
    main()
