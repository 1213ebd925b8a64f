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


# ----------------------------------------------------------------- capacity

def test_pack_marks_rows_past_the_capacity(cuda):
    from mlx_dspark_b200 import tree

    counts, lens, cap, start = [5, 4, 0, 3, 2], [7, 10, 1, 20, 6], [9, 10, 4, 12, 9], [0, 9, 19, 23, 35]
    got = tree.pack(_cu(counts, cuda), None, _i32(lens, cuda), 14, 5, kv_start=_i32(start, cuda),
                    kv_cap=_i32(cap, cuda))
    assert got["room"].tolist() == [2, 0, 0, 0, 2]
    assert got["row_slot"].tolist() == [7, 8] + [-1] * 10 + [41, 42]
    assert got["kv_len_new"].tolist() == [12, 14, 1, 23, 8]


@pytest.mark.parametrize("form", ["chain", "draft", "tree"])
def test_sample_accept_row_limit(cuda, form):
    """Rows past a request's limit count as not tried: the decisions of the block cut there."""
    from mlx_dspark_b200 import sampling

    V, n = 500, 9
    limits = [9, 5, 1, 0, 2, 20, 3, -4]
    B = len(limits)
    rng = np.random.default_rng(1)
    logits = torch.tensor(2 * rng.standard_normal((B * n, V)), dtype=torch.float32)
    ids = logits.reshape(B, n, V).argsort(-1)[:, :, -1].roll(1, 1).contiguous()  # a row's favourite next
    parent = [-1, 0, 0, 1, 2, 2, 3, 4, 4]
    if form == "tree":
        top = logits.reshape(B, n, V).argsort(-1, descending=True)
        for i in range(1, n):
            ids[:, i] = top[:, parent[i], i % 3]
    q = None
    if form == "draft":
        q = torch.softmax(logits + torch.tensor(rng.standard_normal((B * n, V)), dtype=torch.float32), -1)
    u = torch.tensor(0.6 * rng.random(B * n), dtype=torch.float32)
    noise = torch.tensor(rng.exponential(size=(B, V)), dtype=torch.float32)
    lens = _i32([50] * B, cuda)
    got = sampling.sample_accept(
        logits.to(cuda), _i32(ids.flatten().tolist(), cuda), _cu([n] * B, cuda), u.to(cuda), noise.to(cuda),
        draft_probs=None if q is None else q.to(cuda), parent=_i32(parent * B, cuda) if form == "tree" else None,
        max_rows=n, row_limit=_i32(limits, cuda), lens=lens)
    path = got["path"].view(B, n).tolist()
    for b, lim in enumerate(limits):
        if lim <= 0:
            assert (int(got["n"][b]), int(got["next"][b]), int(lens[b])) == (0, -1, 50 - n)
            assert path[b] == [-1] * n and got["prob"][b * n : (b + 1) * n].tolist() == [0.0] * n
            continue
        rows, lim = slice(b * n, (b + 1) * n), min(lim, n)
        p = ref.probabilities(logits[rows].numpy(), 1.0)
        pth, tok, close = ref.accept(p[:lim], ids[b, :lim].tolist(), parent[:lim] if form == "tree" else None,
                                     u[rows].numpy(), noise[b].numpy(),
                                     None if q is None else q[rows].numpy()[:lim], False)
        assert not close
        assert (int(got["n"][b]), int(got["next"][b]), int(lens[b])) == (len(pth) - 1, tok, 50 - n + len(pth))
        assert path[b] == pth + [-1] * (n - len(pth))


@pytest.mark.parametrize("position_major", [False, True])
def test_a_tree_past_its_slots_end_stays_in_its_slot(cuda, position_major):
    """Slot 0 has room for two of five nodes, then for none: nothing of its neighbours moves, what does not
    fit is not accepted, and the device status tells."""
    from mlx_dspark_b200 import _lib

    caps = [40, 40, 40]
    t, eng = _engine(cuda, **(dict(slot_caps=caps) if position_major else dict(kv_cap=40, slots=3)))
    big, wide = _engine(cuda, **(dict(slot_caps=[90, 90, 90]) if position_major else dict(kv_cap=90, slots=3)))
    start = [38, 3, 20]
    g = torch.Generator(device=cuda).manual_seed(5)
    for li in range(len(t.layers)):
        for w in "kv":
            for b in range(3):
                x = torch.randn((t.cfg.n_kv_heads, 40, t.cfg.head_dim), device=cuda, generator=g).to(BF)
                t.slot_view(li, b, w)[:] = x
                big.slot_view(li, b, w)[:, :40] = x
    before = [[t.slot_view(li, b, w).clone() for b in range(3)] for li in range(len(t.layers)) for w in "kv"]
    V, counts = t.cfg.vocab, [5, 3, 0]
    ids = torch.randint(0, V, (8,), device=cuda, dtype=torch.int32, generator=g)
    cu, par = _cu(counts, cuda), _i32([-1, 0, 1, 2, 2, -1, 0, 0], cuda)
    u, noise = torch.zeros(8, device=cuda), torch.empty(3, V, device=cuda).exponential_(generator=g)
    temp = torch.full((3,), 50.0, device=cuda)  # u of zero: any tried token is accepted

    def step(e):
        return e.step(ids, cu, u, noise, parent=par, temperature=temp)

    wide.lens.copy_(_i32(start, cuda))
    all_fit = step(wide)
    assert all_fit["n"].tolist() == [3, 1, 0] and _lib.device_status(cuda.index) == 0
    eng.lens.copy_(_i32(start, cuda))
    out = step(eng)
    assert _lib.device_status(cuda.index) == 0x203  # recorded, and cleared by reading
    assert out["n"].tolist() == [1, 1, 0] and eng.lens.tolist() == [40, 5, 20]
    assert out["path"].tolist() == [0, 1, -1, -1, -1, 0, 1, -1]
    assert int(out["next"][1]) == int(all_fit["next"][1])
    assert int(out["next"][0]) >= 0 and int(out["next"][2]) == -1
    i = 0
    for li in range(len(t.layers)):
        for w in "kv":
            now = [t.slot_view(li, b, w) for b in range(3)]
            assert torch.equal(now[0][:, :38], before[i][0][:, :38])
            assert torch.equal(now[0][:, 38:], big.slot_view(li, 0, w)[:, 38:40])
            assert torch.equal(now[1][:, :3], before[i][1][:, :3])
            assert torch.equal(now[1][:, 3:5], big.slot_view(li, 1, w)[:, 3:5])
            assert torch.equal(now[1][:, 6:], before[i][1][:, 6:]) and torch.equal(now[2], before[i][2])
            i += 1
    state = [t.slot_view(li, 0, w).clone() for li in range(len(t.layers)) for w in "kv"]
    out = step(eng)  # no room at all: the slot stays, the other one goes on
    assert _lib.device_status(cuda.index) != 0
    assert out["n"].tolist()[0] == 0 and int(out["next"][0]) == -1 and eng.lens.tolist() == [40, 7, 20]
    for x, y in zip(state, (t.slot_view(li, 0, w) for li in range(len(t.layers)) for w in "kv")):
        assert torch.equal(x, y)
    assert all(torch.equal(t.slot_view(li, 2, w), before[2 * li + (w == "v")][2])
               for li in range(len(t.layers)) for w in "kv")


# ----------------------------------------------------------------- attention

U = {BF: 2.0 ** -8, HF: 2.0 ** -11}


def _sees(parents, n, L, chain=False):
    """bool [n, L] on the CPU: a request's cached keys and each row's ancestors."""
    m = torch.ones(n, L, dtype=torch.bool)
    m[:, L - n :] = torch.ones(n, n, dtype=torch.bool).tril() if chain else False
    if not chain:
        for i, a in enumerate(ref.ancestors(parents)):
            m[i, [L - n + j for j in a]] = True
    return m


def _exact(q, kc, vc, sees, scale, dtype):
    """One request in 64 bits on the GPU, and the bound of test_tree_round_gpu.py."""
    n, hq, d = q.shape
    hk, L = kc.shape[0], sees.shape[1]
    z = torch.einsum("nhgd,hld->hgnl", q.double().view(n, hk, hq // hk, d), kc[:, :L].double()) * scale
    w = torch.softmax(z.masked_fill(~sees.to(q.device), float("-inf")), -1)
    v = vc[:, :L].double()
    o = torch.einsum("hgnl,hld->nhgd", w, v).reshape(n, hq, d)
    absum = torch.einsum("hgnl,hld->nhgd", w, v.abs()).reshape(n, hq, d)
    tail = 2.0 ** -25 * v.abs().sum(1).amax() if dtype == HF else 0.0
    return o, (U[dtype] + 1e-4) * absum + U[dtype] * o.abs() + tail + 1e-7


def test_a_wait_that_runs_out_leaves_nothing_behind(cuda):
    """A captured call whose waits run out tells so and returns; replayed with the usual limit on other
    rows it is right, whatever flags and counts the former run has left."""
    from mlx_dspark_b200 import _lib, tree

    rng = random.Random(0)
    B, Hq, Hk, D, nodes = 24, 16, 4, 128, 9
    counts = [rng.randint(1, nodes) for _ in range(B)]
    lens = [rng.randint(nodes, 6000) for _ in counts]
    parents = [ref.random_parents(n, rng) for n in counts]
    g = torch.Generator(device=cuda).manual_seed(1)
    kc, vc = (torch.randn(B, Hk, max(lens), D, device=cuda, generator=g).to(BF) for _ in range(2))
    rows = [torch.randn(sum(counts), Hq, D, device=cuda, generator=g).to(BF) for _ in range(2)]
    anc = _i32([w for p in parents for w in ref.words_of(ref.ancestors(p), 1)], cuda)
    want = []
    for x in rows:
        r0, parts = 0, []
        for b, n in enumerate(counts):
            parts.append(_exact(x[r0 : r0 + n], kc[b], vc[b], _sees(parents[b], n, lens[b]), D ** -0.5, BF))
            r0 += n
        want.append([torch.cat(t) for t in zip(*parts)])
    q, out = rows[0].clone(), torch.empty_like(rows[0])
    args = (q, kc, vc, _cu(counts, cuda), _i32(lens, cuda), anc)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        tree.tree_sdpa(*args, scale=D ** -0.5, max_nodes=nodes, out=out)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            tree.tree_sdpa(*args, scale=D ** -0.5, max_nodes=nodes, out=out)
    torch.cuda.synchronize()
    ran_out = 0
    for k, limit_ns in enumerate((0, 300, 1000, 2000, 4000, 8000, 16000)):
        if limit_ns:
            _lib.set_wait_limit_ns(cuda.index, limit_ns)
            try:
                graph.replay()
                torch.cuda.synchronize()
            finally:
                _lib.set_wait_limit_ns(cuda.index, 0)
            ran_out += _lib.device_status(cuda.index) != 0
        q.copy_(rows[k % 2])
        out.fill_(float("nan"))
        graph.replay()
        o, bound = want[k % 2]
        assert ((out.double() - o).abs() <= bound).all(), limit_ns
        assert _lib.device_status(cuda.index) == 0
    assert ran_out


@pytest.mark.parametrize("pool", [False, True])
def test_rows_of_no_request_are_not_appended(cuda, pool):
    """A round packed for more rows than its requests have, into arrays of a former round."""
    from mlx_dspark_b200 import _lib, rope, tree

    R, B, Hk, cap, D = 12, 2, 2, 20, 64
    out = {k: torch.full((R,), 5, dtype=torch.int32, device=cuda) for k in ("row_pos", "row_slot")}
    out |= {"row_req": torch.zeros(R, dtype=torch.int32, device=cuda),
            "anc": torch.full((R, 2), -1, dtype=torch.int32, device=cuda), "kv_len_new": _i32([0, 0], cuda)}
    start = _i32([0, cap], cuda) if pool else None
    meta = tree.pack(_cu([3, 4], cuda), None, _i32([8, 2], cuda), R, 40, kv_start=start, out=out)
    assert meta["row_slot"].tolist() == [8, 9, 10] + [2 + i + cap * pool for i in range(4)] + [-1] * 5
    assert meta["row_req"].tolist() == ([0] * 7 if pool else [0] * 3 + [1] * 4) + [-1] * 5
    assert meta["row_pos"].tolist()[7:] == [0] * 5 and not meta["anc"][7:].any()
    x = torch.ones(R, Hk, D, dtype=BF, device=cuda)
    kc = torch.zeros((1, Hk, B * cap, D) if pool else (B, Hk, cap, D), dtype=BF, device=cuda)
    vc = torch.zeros_like(kc)
    rope.rope_append(x, x, x, rope.RopeTable(D, device=cuda), meta["row_pos"], kc, vc, meta["row_slot"],
                     row_req=meta["row_req"])
    assert float(vc.sum()) == 7 * Hk * D
    assert _lib.device_status(cuda.index) == 0


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("late", [False, True])
@pytest.mark.parametrize("drop", [16.0, 18.0, 20.0])
def test_attention_keeps_the_mass_of_a_long_tail(cuda, dtype, late, drop):
    """One key far above 30000 others whose values are all the output. The weights' bound: rounded to the
    type relative to themselves, and for fp16 below 2^-14 of 2^7 times the row's reference by 2^-25 of that
    at most, so by 2^-32 a key (the sum they are divided by is not below the reference)."""
    from mlx_dspark_b200 import tree

    L, n, Hq, Hk, D, B = 30011, 3, 8, 2, 64, 150  # requests enough that a row's keys are in one or two parts
    g = torch.Generator(device=cuda).manual_seed(int(drop))
    q = 0.01 * torch.randn(n, Hq, D, device=cuda, generator=g)
    k = 0.5 * torch.randn(1, Hk, L, D, device=cuda, generator=g)
    v = 1.0 + 0.25 * torch.randn(1, Hk, L, D, device=cuda, generator=g)
    q[..., 0], k[..., 0] = 4.0, -drop / 8
    top = L - 400 if late else 5
    k[:, :, top, 0], v[:, :, top] = drop / 8, 0.0
    q, k, v = q.to(dtype), k.to(dtype), v.to(dtype)
    out = tree.tree_sdpa(q.repeat(B, 1, 1), k, v, _cu([n] * B, cuda), _i32([L] * B, cuda), None, scale=1.0,
                         max_nodes=n).view(B, n, Hq, D)
    o, _ = _exact(q, k[0], v[0], _sees(None, n, L, chain=True), 1.0, dtype)
    size = o.abs()  # the values are positive (but for chance): sum p |v| is the output
    bound = (U[dtype] + 1e-4) * size + U[dtype] * size + (2.0 ** -32 * 3.0 * L if dtype == HF else 0.0) + 2.0 ** -25
    assert ((out.double() - o).abs() <= bound).all(), float(((out.double() - o).abs() / bound).max())


def test_sample_accept_returns_results_alone(cuda):
    """The result's values are its tensors, whether it is a new one or a former one, with lengths or not."""
    from mlx_dspark_b200 import sampling

    V = 90
    args = (torch.zeros(3, V, device=cuda), _i32([0, 0, 0], cuda), _cu([1, 2], cuda), torch.rand(3, device=cuda),
            torch.ones(2, V, device=cuda))
    out, lens = None, _i32([4, 5], cuda)
    for given in (None, lens, None, lens):
        out = sampling.sample_accept(*args, max_rows=2, lens=given, out=out)
        want = {"n", "next", "prob", "path"} | ({"lens"} if given is not None else set())
        assert set(out) == want and all(isinstance(v, torch.Tensor) for v in out.values())
    assert {k: v.clone() for k, v in out.items()}["lens"].tolist() == lens.tolist()


@pytest.mark.parametrize("tree", [False, True])
def test_a_round_of_idle_slots(cuda, tree):
    """No nodes at all: every slot stays."""
    t, eng = _engine(cuda)
    eng.lens.copy_(_i32([4, 0, 9], cuda))
    none = torch.empty(0, dtype=torch.int32, device=cuda)
    out = eng.step(none, _cu([0, 0, 0], cuda), torch.empty(0, device=cuda),
                   torch.ones(3, t.cfg.vocab, device=cuda), parent=none if tree else None)
    assert out["n"].tolist() == [0, 0, 0] and out["next"].tolist() == [-1] * 3 and eng.lens.tolist() == [4, 0, 9]


# ----------------------------------------------------------------- wider ranges of what was there

@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("counts,lens,Hq,Hk,D", [
    ([384], [1000], 16, 2, 128),
    ([700, 3, 300], [900, 2500, 300], 8, 4, 64),
    ([1024], [1024], 4, 4, 128),
    ([1024, 1000], [5000, 1013], 12, 2, 128),
])
def test_attention_of_big_trees(cuda, dtype, counts, lens, Hq, Hk, D):
    """Up to 1024 nodes: many row blocks a request, trees over many key tiles."""
    from mlx_dspark_b200 import tree

    rng = random.Random(sum(counts))
    parents = [ref.random_parents(n, rng) for n in counts]
    g = torch.Generator(device=cuda).manual_seed(len(counts))
    q = torch.randn(sum(counts), Hq, D, device=cuda, generator=g).to(dtype)
    kc, vc = (torch.randn(len(counts), Hk, max(lens) + 7, D, device=cuda, generator=g).to(dtype) for _ in range(2))
    for b, L in enumerate(lens):
        kc[b, :, L:], vc[b, :, L:] = float("inf"), float("nan")
    words = tree.anc_words(max(counts))
    anc = _i32([w for p in parents for w in ref.words_of(ref.ancestors(p), words)], cuda)
    out = tree.tree_sdpa(q, kc, vc, _cu(counts, cuda), _i32(lens, cuda), anc, scale=D ** -0.5,
                         max_nodes=max(counts))
    r0 = 0
    for b, n in enumerate(counts):
        o, bound = _exact(q[r0 : r0 + n], kc[b], vc[b], _sees(parents[b], n, lens[b]), D ** -0.5, dtype)
        assert ((out[r0 : r0 + n].double() - o).abs() <= bound).all(), b
        r0 += n


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("counts,lens,Hq,Hk,D", [
    ([129], [129], 8, 2, 128),
    ([500], [1700], 16, 4, 64),
    ([2048], [2048], 8, 2, 128),
    ([1000, 1, 333], [1001, 4096, 2000], 4, 4, 128),
])
def test_attention_of_prompt_chunks(cuda, dtype, counts, lens, Hq, Hk, D):
    """anc None over whole chunks of a prompt, in a position-major pool."""
    from mlx_dspark_b200 import tree

    g = torch.Generator(device=cuda).manual_seed(sum(lens))
    start = [11 + sum(lens[:b]) for b in range(len(lens))]
    q = torch.randn(sum(counts), Hq, D, device=cuda, generator=g).to(dtype)
    kc, vc = (torch.randn(sum(lens) + 40, Hk, D, device=cuda, generator=g).to(dtype).permute(1, 0, 2)[None]
              for _ in range(2))
    out = tree.tree_sdpa(q, kc, vc, _cu(counts, cuda), _i32(lens, cuda), None, scale=D ** -0.5,
                         max_nodes=max(counts), kv_start=_i32(start, cuda))
    r0 = 0
    for b, n in enumerate(counts):
        o, bound = _exact(q[r0 : r0 + n], kc[0, :, start[b] :], vc[0, :, start[b] :],
                          _sees(None, n, lens[b], chain=True), D ** -0.5, dtype)
        assert ((out[r0 : r0 + n].double() - o).abs() <= bound).all(), b
        r0 += n


@pytest.mark.parametrize("form", ["chain", "draft", "tree"])
def test_sample_accept_blocks_beyond_max_rows_and_second_roots(cuda, form):
    """max_rows below the blocks' rows cuts them; a node whose parent is not before it is nobody's child."""
    from mlx_dspark_b200 import sampling

    V, n, cut, B = 3001, 21, 8, 70
    rng = np.random.default_rng(3)
    logits = torch.tensor(3 * rng.standard_normal((B * n, V)), dtype=torch.float32).to(HF)
    best = logits.float().view(B, n, V).argsort(-1, descending=True)[:, :, :3]
    pr = random.Random(4)
    parents, ids = [], torch.zeros(B, n, dtype=torch.long)
    for b in range(B):
        par = list(range(-1, n - 1)) if form != "tree" else ref.random_parents(n, pr)
        for i in range(1, n):
            ids[b, i] = best[b, par[i], pr.randrange(3)]
            if form == "tree" and pr.random() < 0.2:
                par[i] = pr.choice([i, i + 1, n, n + 50, -1, -7])
        parents.append(par)
    q = None
    if form == "draft":
        q = torch.softmax(logits.float() + torch.tensor(rng.standard_normal((B * n, V)), dtype=torch.float32), -1)
    u = torch.tensor(rng.random(B * n), dtype=torch.float32)
    noise = torch.tensor(rng.exponential(size=(B, V)), dtype=torch.float32)
    lens, close = _i32([60] * B, cuda), 0
    got = sampling.sample_accept(
        logits.to(cuda), _i32(ids.flatten().tolist(), cuda), _cu([n] * B, cuda), u.to(cuda), noise.to(cuda),
        draft_probs=None if q is None else q.to(cuda),
        parent=_i32([p for x in parents for p in x], cuda) if form == "tree" else None, max_rows=cut, lens=lens)
    path = got["path"].view(B, n).tolist()
    for b in range(B):
        rows = slice(b * n, (b + 1) * n)
        p = ref.probabilities(logits[rows].float().numpy(), 1.0)
        want = [p[x, ids[b, i]] if 0 <= x < i else 1.0 for i, x in enumerate(parents[b])]
        np.testing.assert_allclose(got["prob"][rows].cpu().numpy(), want, rtol=2.0 ** -23 * 208, atol=1e-30)
        up = [x if x < i else -9 for i, x in enumerate(parents[b])][:cut]
        pth, tok, near = ref.accept(p[:cut], ids[b, :cut].tolist(), up if form == "tree" else None, u[rows].numpy(),
                                    noise[b].numpy(), None if q is None else q[rows].numpy()[:cut], False)
        close += near
        if not near:
            assert (int(got["n"][b]), int(got["next"][b]), int(lens[b])) == (len(pth) - 1, tok, 60 - n + len(pth)), b
            assert path[b] == pth + [-1] * (n - len(pth))
    assert close <= 4


def test_calls_repeat_themselves_bit_for_bit(cuda):
    """The attention's joins and the accept's comparisons have one order, whatever the CTAs' timing."""
    from mlx_dspark_b200 import sampling, tree

    rng = random.Random(8)
    for B, longest, nodes in ((1, 9000, 40), (37, 3000, 20)):
        counts = [rng.randint(1, nodes) for _ in range(B)]
        lens = [rng.randint(nodes, longest) for _ in counts]
        g = torch.Generator(device=cuda).manual_seed(B)
        q = torch.randn(sum(counts), 16, 128, device=cuda, generator=g).to(BF)
        kc, vc = (torch.randn(B, 4, longest, 128, device=cuda, generator=g).to(BF) for _ in range(2))
        args = (q, kc, vc, _cu(counts, cuda), _i32(lens, cuda), None)
        outs = [tree.tree_sdpa(*args, scale=0.09, max_nodes=nodes) for _ in range(12)]
        assert all(torch.equal(x, outs[0]) for x in outs)
        V, R = 70001, sum(counts)
        logits = torch.randn(R, V, device=cuda, generator=g)
        par = _i32([p for n in counts for p in ref.random_parents(n, rng)], cuda)
        args = (logits, logits.argmax(1).roll(1).int(), _cu(counts, cuda), torch.rand(R, device=cuda, generator=g),
                torch.empty(B, V, device=cuda).exponential_(generator=g))
        outs = [sampling.sample_accept(*args, parent=par, max_rows=nodes) for _ in range(12)]
        assert all(torch.equal(x[k], outs[0][k]) for x in outs for k in ("n", "next", "prob", "path"))
