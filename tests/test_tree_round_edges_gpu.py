"""Edges of the tree-round operators on the GPU: widest slices, slots that run out of room, refused
calls, waits that run out, long tails. Bounds as in test_tree_round_gpu.py."""

from __future__ import annotations

import random

import numpy as np
import pytest
import torch
import tree_reference as ref

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def _i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _cu(counts, dev):
    return _i32([0] + np.cumsum(counts).tolist(), dev)


# ----------------------------------------------------------------- sampled accept

@pytest.mark.parametrize("form", ["tree", "chain"])
@pytest.mark.parametrize("V", [262121, 262143, 327679, 393209])
def test_sample_accept_widest_slices(cuda, form, V):
    """Many requests over a vocabulary just below a multiple of 65536: slices of the widest kind, the
    tokens tried and drawn among their last values."""
    from mlx_dspark_b200 import sampling

    B, rows = 150, 3
    g = torch.Generator().manual_seed(V)
    row = torch.randn(V, generator=g)
    row[-3:] = torch.tensor([15.0, 16.0, 17.0])
    noise = torch.empty(V).exponential_(generator=g)
    noise[-3:] = torch.tensor([0.5, 1e-3, 1e-3])  # without the bars V - 2 or V - 1 would be drawn
    ids = _i32([7, V - 1, V - 2] * B, cuda)
    u = torch.rand(B, rows, generator=g)
    u[::3] = 0.9999  # nothing accepted: the token after is drawn without those tried
    temp = torch.ones(B)
    temp[1::7] = 0.0
    parents = [-1, 0, 0] if form == "tree" else None
    got = sampling.sample_accept(
        row.to(cuda).expand(B * rows, V), ids, _cu([rows] * B, cuda), u.flatten().to(cuda),
        noise.to(cuda).expand(B, V), temperature=temp.to(cuda), max_rows=rows,
        parent=None if parents is None else _i32(parents * B, cuda))
    n, nxt, path = got["n"].tolist(), got["next"].tolist(), got["path"].view(B, rows).tolist()
    p = {T: ref.probabilities(row[None].numpy(), T).repeat(rows, 0) for T in (0.0, 1.0)}
    for b in range(B):
        T = float(temp[b])
        pth, tok, close = ref.accept(p[T], [7, V - 1, V - 2], parents, u[b].numpy(), noise.numpy(), None, T == 0)
        if not close:
            assert (n[b], nxt[b]) == (len(pth) - 1, tok), (b, T)
            assert path[b] == pth + [-1] * (rows - len(pth))


# ----------------------------------------------------------------- engine

def _engine(dev, max_nodes=8, **kw):
    from mlx_dspark_b200.target import Target, tiny_config
    from mlx_dspark_b200.tree_engine import TreeSpec

    t = Target(tiny_config(), seed=3, max_rows=40, **(kw or dict(kv_cap=200, slots=3)))
    return t, TreeSpec(t, max_nodes)


def test_a_refused_step_leaves_the_slots_as_they_were(cuda):
    from mlx_dspark_b200 import DSparkError, DSparkUnsupported

    t, eng = _engine(cuda)
    V, counts = t.cfg.vocab, [5, 0, 3]
    g = torch.Generator().manual_seed(2)
    ids = torch.randint(0, V, (8,), generator=g, dtype=torch.int32).to(cuda)
    cu, par = _cu(counts, cuda), _i32([-1, 0, 0, 1, 1, -1, 0, 1], cuda)
    u, noise = torch.rand(8, generator=g).to(cuda), torch.empty(3, V).exponential_(generator=g).to(cuda)
    temp = torch.ones(3, device=cuda)
    start = _i32([9, 20, 31], cuda)

    def step(u=u, noise=noise, **kw):
        return eng.step(ids, cu, u, noise, temperature=temp, **{"parent": par, **kw})

    eng.lens.copy_(start)
    want = [step()[k].tolist() for k in ("n", "next", "path")], eng.lens.tolist()
    assert want[1] != start.tolist()
    eng.lens.copy_(start)
    q = torch.full((8, V), 1.0 / V, device=cuda)
    with pytest.raises(DSparkUnsupported):
        step(draft_probs=q)  # a tree has none
    for bad in (dict(noise=noise[:2]), dict(noise=noise.double()), dict(u=u.double()), dict(u=u[:7])):
        with pytest.raises(DSparkError):
            step(**bad)
    assert eng.lens.tolist() == start.tolist()
    assert ([step()[k].tolist() for k in ("n", "next", "path")], eng.lens.tolist()) == want


def test_forward_checks_what_its_kernels_index(cuda):
    """Metadata of another round's size and buffers that the logits do not fit are refused."""
    from mlx_dspark_b200 import DSparkError, tree

    t, eng = _engine(cuda)
    V = t.cfg.vocab
    ids, cu = torch.zeros(6, dtype=torch.int32, device=cuda), _cu([4, 0, 2], cuda)
    eng.lens.copy_(_i32([5, 6, 7], cuda))

    def meta(**kw):
        return {**tree.pack(cu, None, eng.lens, 6, 8), **kw}

    want = eng.forward(ids, meta(), cu).clone()
    short = tree.pack(_cu([3, 0, 2], cuda), None, eng.lens, 5, 8)
    for k in ("row_pos", "row_slot", "row_req", "anc"):
        with pytest.raises(DSparkError):
            eng.forward(ids, meta(**{k: short[k]}), cu)
    for k in ("row_slot", "anc", "kv_len_new"):
        with pytest.raises(DSparkError):
            eng.forward(ids, meta(**{k: meta()[k].long()}), cu)
    for bad in (dict(kv_len_new=_i32([9, 6], cuda)), dict(anc=meta()["anc"].flatten())):
        with pytest.raises(DSparkError):
            eng.forward(ids, meta(**bad), cu)
    for logits in (torch.empty(5, V, dtype=BF, device=cuda), torch.empty(6, V - 2, dtype=BF, device=cuda),
                   torch.empty(6, V, device=cuda), torch.empty(V, 6, dtype=BF, device=cuda).t(),
                   torch.empty(1, V, dtype=BF, device=cuda).expand(6, V), torch.empty(6, V, dtype=BF)):
        with pytest.raises(DSparkError):
            eng.forward(ids, meta(), cu, logits)
    out = torch.empty(9, V + 8, dtype=BF, device=cuda)[:, :V]
    assert torch.equal(eng.forward(ids, meta(), cu, out), want)
