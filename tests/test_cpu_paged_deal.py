"""Where the pieces of a call lie in the workspace of the attention behind a common prefix: the deal of
csrc/paged_attention_tcgen05.cu stated over the whole line at once. No two pieces of a call may share a place, and the joining
launch has to find every one of them from what it is told: the CTA of the first, whether that one begins the CTA's share, and their number."""
import math
import random
import re
from pathlib import Path

import pytest

SOURCE = (Path(__file__).resolve().parents[1] / "scirust_b200" / "csrc" / "paged_attention_tcgen05.cu").read_text()
BM = BN = 128


def constant(name):
    return int(re.search(rf"\b{name} = (\d+)", SOURCE).group(1))


FEW = constant("FEW")
BLOCK = {k: constant(f"BLOCK_{k}") for k in ("FEW", "ONE", "TWO")}
ITEM = {k: constant(f"ITEM_{k}") for k in ("FEW", "ONE", "TWO")}


def kind(tokens, TT, few):
    return "FEW" if few else "TWO" if tokens > TT else "ONE"


def line(H, Hkv, prefix, runs, ragged):
    """Items in their order, shared ones and then own ones, as (name, positions, kind); ``runs`` is (length, rows) of each sequence."""
    G = H // Hkv
    TT, NT = BM // G, sum(n for _, n in runs)
    few = 0 if ragged or G > FEW else 1 if NT * G > FEW else 3
    shared, own = [], []
    if prefix:
        for h in range(Hkv):
            for t in range(0, NT, 2 * TT):
                n = min(2 * TT, NT - t)
                shared.append((("shared", h, t), prefix, kind(n, TT, few & 2 and n == NT - t)))
    for b, (length, n) in enumerate(runs):
        for t in range(0, n, 2 * TT):
            m = min(2 * TT, n - t)
            end = length - n + t + m
            own += [(("own", b, t, h), end - prefix, kind(m, TT, few & 1)) for h in range(Hkv) if end > prefix]
    return shared, own, kind(NT, TT, few & 2), kind(1, TT, few & 1)


def units(item):
    return -(-item[1] // BN) * BLOCK[item[2]] + ITEM[item[2]]


def deal(shared, own, common_kind, own_kind, grid):
    """(first CTA, CTAs' first units, last unit + 1) of either part of the line."""
    U, V = sum(map(units, shared)), sum(map(units, own))
    n = grid if U else 0
    if U and V:
        more = ITEM[common_kind] - ITEM[own_kind]
        b = more * grid - U - V
        below = math.sqrt(b * b + 4 * more * U * grid) - b
        n = max(1, min(grid - 1, math.ceil(2 * U * grid / below) if below > 0 else grid - 1))
    for first, count, total in ((0, n, U), (n, grid - n, V)):
        share = max(1, min(count, total // BLOCK["TWO"]))
        per, rem = divmod(total, share)
        yield first, [min(total, c * per + min(c, rem)) for c in range(count + 1)]


def pieces(shared, own, common_kind, own_kind, grid):
    """(CTA, item, first block, block behind the last, of how many, whether it begins the CTA's share)"""
    for items, (cta, edges) in zip((shared, own), deal(shared, own, common_kind, own_kind, grid)):
        at = 0
        for item in items:
            size, head, each = units(item), ITEM[item[2]], BLOCK[item[2]]
            for c, (lo, hi) in enumerate(zip(edges, edges[1:])):
                lo, hi = max(lo, at), min(hi, at + size)
                if lo < hi:                      # a block is with the CTA that has its first unit
                    j0, j1 = ((max(0, u - at - head) + each - 1) // each for u in (lo, hi))
                    if j0 < j1:
                        yield cta + c, item[0], j0, j1, (size - head) // each, lo == edges[c]
            at += size


def place(cta, item, j0, j1, blocks, first):
    """As in attend_kernel: a slot of the CTA for what is cut, the rows of the batch for what is not."""
    return ("cut", 2 * cta + (0 if first else 1)) if j1 - j0 < blocks else ("whole", item)


def look_over(H, Hkv, prefix, runs, ragged=False, most=None):
    found = list(pieces(*line(H, Hkv, prefix, runs, ragged), grid=max(2, min(148, most or 148))))
    places = [place(*p) for p in found]
    assert len(set(places)) == len(places)
    of = {}
    for p in found:
        of.setdefault(p[1], []).append(p)
    for parts in of.values():
        assert parts[0][2] == 0 and parts[-1][3] == parts[0][4] and all(a[3] == b[2] for a, b in zip(parts, parts[1:]))
        if len(parts) > 1:                       # those behind the first lie with the CTAs behind its, each in its first slot
            assert [p[0] for p in parts] == list(range(parts[0][0], parts[0][0] + len(parts))) and all(p[5] for p in parts[1:])
    return found


@pytest.mark.parametrize("H, Hkv, B, prefix, own, most", [
    (32, 32, 8, 512, 257, None), (32, 32, 8, 512, 2000, None), (32, 32, 8, 1024, 385, None), (32, 32, 4, 512, 513, None),
    (16, 16, 8, 1024, 2000, None), (32, 8, 2, 256, 8192, None), (32, 8, 2, 512, 7810, None), (32, 8, 2, 128, 1, 8), (32, 8, 2, 128, 300, 8)])
def test_a_cta_may_have_many_shared_items_of_few_rows(H, Hkv, B, prefix, own, most):
    found = look_over(H, Hkv, prefix, [(prefix + own, 1)] * B, most=most)
    slots = [(p[0], p[5]) for p in found if p[1][0] == "shared"]
    assert len(set(slots)) < len(slots)                 # more than a CTA has slots: whole ones may not go there


@pytest.mark.parametrize("seed", range(8))
def test_no_two_pieces_have_one_place(seed):
    rng = random.Random(seed)
    for _ in range(60):
        Hkv, G = rng.choice([1, 2, 4, 8, 16, 32]), rng.choice([1, 1, 2, 3, 4, 8, 9, 16])
        B, ragged = rng.choice([1, 2, 3, 4, 8, 9, 33]), rng.random() < 0.4
        prefix = 8 * round(math.exp(rng.uniform(0, math.log(1024)))) * (rng.random() < 0.9)
        most = round(math.exp(rng.uniform(math.log(300), math.log(16384))))
        runs = []
        for _ in range(B):
            n = rng.randint(0, 300) if ragged else 1
            runs.append((max(0, prefix + rng.choice([-5, n, n + rng.randint(0, most)])), n))
        look_over(G * Hkv, Hkv, prefix, runs, ragged, most=rng.choice([None, None, 2, rng.randint(2, 148)]))
