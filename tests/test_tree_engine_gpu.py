"""Tree rounds over a small target: one packed forward of ragged trees against plain verify forwards
of each root-to-node chain, and whole rounds against plain decoding of what they accepted.

Bar: both forwards are bf16 dataflows that the suite holds to 1e-2 of max|logit| of the oracle each,
so they may differ by twice that."""

from __future__ import annotations

import random

import pytest
import torch
import tree_reference as ref

pytestmark = pytest.mark.gpu

REL = 2e-2


def _targets(dev, position_major, max_rows=96):
    from mlx_dspark_b200.target import Target, tiny_config

    kw = dict(slot_caps=[400, 300, 500]) if position_major else dict(kv_cap=500, slots=3)
    t = Target(tiny_config(), seed=3, max_rows=max_rows, **kw)
    plain = Target(tiny_config(), seed=3, kv_cap=500, max_rows=32)
    return t, plain


def _prefix(t, lens, dev):
    g = torch.Generator(device=dev).manual_seed(5)
    for b, n in enumerate(lens):
        for li in range(len(t.layers)):
            for which in "kv":
                t.slot_view(li, b, which)[:, :n] = torch.randn(
                    (t.cfg.n_kv_heads, n, t.cfg.head_dim), device=dev, generator=g).to(torch.bfloat16)


def _chain_logits(plain, t, slot, L0, ids, dev):
    """Logits of the last token of `ids` after slot's first L0 cached tokens, by the plain forward."""
    for li in range(len(t.layers)):
        for which in "kv":
            plain.slot_view(li, 0, which)[:, :L0] = t.slot_view(li, slot, which)[:, :L0]
    lens = torch.tensor([L0], dtype=torch.int32, device=dev)
    return plain.verify(torch.tensor(ids, dtype=torch.int32, device=dev), lens)[-1].float()


@pytest.mark.parametrize("position_major", [False, True])
@pytest.mark.parametrize("counts", [[9, 1, 13], [40, 0, 21], [24, 40, 30]])
def test_tree_forward_matches_chains(cuda, position_major, counts):
    from mlx_dspark_b200 import tree
    from mlx_dspark_b200.tree_engine import TreeSpec

    t, plain = _targets(cuda, position_major)
    eng = TreeSpec(t, max(counts))
    L0 = [150, 37, 211]
    _prefix(t, L0, cuda)
    eng.lens.copy_(torch.tensor(L0, dtype=torch.int32))
    rng = random.Random(sum(counts))
    parents = [ref.random_parents(n, rng) if n else [] for n in counts]
    R = sum(counts)
    ids = torch.tensor([rng.randrange(t.cfg.vocab) for _ in range(R)], dtype=torch.int32, device=cuda)
    par = torch.tensor([p for x in parents for p in x], dtype=torch.int32, device=cuda)
    cu = torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32, device=cuda)
    meta = tree.pack(cu, par, eng.lens, R, max(counts), kv_start=eng.kv_start)
    got = eng.forward(ids, meta, cu).float().clone()
    r0 = 0
    for b, n in enumerate(counts):
        for i in sorted({0, n - 1, n // 2} if n else set()):
            path = sorted(ref.ancestors(parents[b])[i])[-32:]
            want = _chain_logits(plain, t, b, L0[b], [int(ids[r0 + j]) for j in path], cuda)
            err = float((got[r0 + i] - want).abs().max())
            assert err <= REL * float(want.abs().max()), (b, i, err)
        r0 += n


@pytest.mark.parametrize("position_major", [False, True])
def test_greedy_rounds_leave_the_cache_of_plain_decoding(cuda, position_major):
    """Two rounds of trees that hold the target's own greedy continuation among wrong branches."""
    from mlx_dspark_b200.tree_engine import TreeSpec

    t, plain = _targets(cuda, position_major)
    L0 = [60, 200, 133]
    _prefix(t, L0, cuda)
    eng = TreeSpec(t, 16)
    eng.lens.copy_(torch.tensor(L0, dtype=torch.int32))
    rng = random.Random(0)
    V = t.cfg.vocab
    pending = [rng.randrange(V) for _ in L0]
    said = [[p] for p in pending]
    for round_ in range(2):
        counts, parents, ids, expect = [], [], [], []
        for b in range(3):
            if b == 2 and round_ == 0:  # an idle slot
                counts.append(0)
                expect.append(None)
                continue
            good, margin = [], []
            for _ in range(3):
                lg = _chain_logits(plain, t, b, L0[b], said[b] + good, cuda)
                top = lg.topk(2)
                good.append(int(top.indices[0]))
                margin.append(float(top.values[0] - top.values[1]) > 2 * REL * float(lg.abs().max()))
            # wrong leaves around the greedy chain: node places 2, 4, 6 continue it
            wrong = [(x + 1 + rng.randrange(V - 1)) % V for x in good]
            counts.append(7)
            parents += [-1, 0, 0, 2, 2, 4, 4]
            ids += [said[b][-1], wrong[0], good[0], wrong[1], good[1], wrong[2], good[2]]
            expect.append((good, margin))
        dev = dict(dtype=torch.int32, device=cuda)
        R = sum(counts)
        cu = torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), **dev)
        out = eng.step(torch.tensor(ids, **dev), cu, torch.full((R,), 0.5, device=cuda),
                       torch.ones(3, V, device=cuda), parent=torch.tensor(parents, **dev))
        n, nxt, lens = out["n"].tolist(), out["next"].tolist(), eng.lens.tolist()
        for b in range(3):
            if expect[b] is None:
                assert n[b] == 0 and nxt[b] == -1 and lens[b] == L0[b] + len(said[b]) - 1
                continue
            good, margin = expect[b]
            sure = margin.index(False) if False in margin else 3
            assert n[b] >= sure  # a near tie may be broken the other way by the tree's own rounding
            assert lens[b] == L0[b] + len(said[b]) + n[b]
            said[b] += good[: n[b]] + [nxt[b]]
    for b in range(3):  # the caches are those of plain decoding of what was said
        done = said[b][:-1]
        if not done:
            continue
        _chain_logits(plain, t, b, L0[b], done, cuda)
        for li in range(len(t.layers)):
            for which in "kv":
                want = plain.slot_view(li, 0, which)[:, L0[b] : L0[b] + len(done)].float()
                got = t.slot_view(li, b, which)[:, L0[b] : L0[b] + len(done)].float()
                assert float((got - want).abs().max()) <= REL * float(want.abs().max()) + 1e-3, (b, li, which)


def test_sampled_round_in_a_graph(cuda):
    """A step holds no host wait: it is captured once and replayed with other numbers."""
    from mlx_dspark_b200.tree_engine import TreeSpec

    t, _ = _targets(cuda, False)
    eng = TreeSpec(t, 8)
    _prefix(t, [50, 60, 70], cuda)
    start = torch.tensor([50, 60, 70], dtype=torch.int32, device=cuda)
    V, counts = t.cfg.vocab, [8, 5, 1]
    dev = dict(dtype=torch.int32, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(1)
    ids = torch.randint(0, V, (14,), generator=g, **dev)
    cu = torch.tensor([0, 8, 13, 14], **dev)
    par = torch.tensor([-1, 0, 0, 1, 1, 2, 5, 5] + [-1, 0, 1, 1, 0] + [-1], **dev)
    u, noise = torch.empty(14, device=cuda), torch.empty(3, V, device=cuda)
    temp = torch.tensor([0.7, 0.0, 1.3], device=cuda)

    def fill(seed):
        gg = torch.Generator(device=cuda).manual_seed(seed)
        eng.lens.copy_(start)
        u.uniform_(generator=gg)
        noise.exponential_(generator=gg)

    def step():
        return eng.step(ids, cu, u, noise, parent=par, temperature=temp)

    eager = []
    for seed in (2, 3, 4):
        fill(seed)
        out = step()
        eager.append([out[k].clone() for k in ("n", "next", "prob", "path")] + [eng.lens.clone()])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fill(9)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step()
    torch.cuda.current_stream().wait_stream(side)
    for seed, want in zip((2, 3, 4), eager):
        fill(seed)
        graph.replay()
        for got, exp in zip([out[k] for k in ("n", "next", "prob", "path")] + [eng.lens], want):
            assert torch.equal(got, exp)
