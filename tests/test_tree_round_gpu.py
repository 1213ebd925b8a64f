"""Tree-round operators on the GPU against plain 64-bit forms.

Bounds, from the formulas: u is the type's unit roundoff (bf16 2^-8, fp16 2^-11).
* rope: one rounding of a value whose fp32 evaluation is off by at most ~1e-6 of the inputs'
  magnitude (phase 2^-25 turns, sin / cos, two products): u |ref| + 4e-6 max|x|;
* attention: the weights are rounded to the type before the product with V (u sum p|v|), the
  output once (u |ref|), scores and sums are fp32 (1e-4 sum p|v| covers both), and fp16 weights
  below its normal range lose at most 2^-25 each;
* probabilities: (l - m) / T carries 2^-24 of its size into the exponent;
* integers and copies: equal (a decision closer than 1e-5 may fall either way, and is told apart).
"""

from __future__ import annotations

import random

import numpy as np
import pytest
import torch
import tree_reference as ref

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def _i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _cu(counts, dev):
    return _i32([0] + np.cumsum(counts).tolist(), dev)


# ----------------------------------------------------------------- packing

@pytest.mark.parametrize("counts", [[1], [5, 1, 0, 33], [64, 65, 100], [300]])
@pytest.mark.parametrize("chain", [False, True])
def test_pack(cuda, counts, chain):
    from mlx_dspark_b200 import tree

    rng = random.Random(sum(counts))
    parents = [list(range(-1, n - 1)) if chain else ref.random_parents(n, rng) for n in counts if n]
    kv = [rng.randint(0, 50) for _ in counts]
    R, mx = sum(counts), max(counts)
    par = None if chain else _i32([p for x in parents for p in x], cuda)
    got = tree.pack(_cu(counts, cuda), par, _i32(kv, cuda), R, mx)
    words = tree.anc_words(mx)
    full = iter(parents)
    pos, slot, req, anc = [], [], [], []
    for b, n in enumerate(counts):
        if n:
            par_b = next(full)
            pos += [kv[b] + d for d in ref.depths(par_b)]
            slot += [kv[b] + i for i in range(n)]
            req += [b] * n
            anc += ref.words_of(ref.ancestors(par_b), words)
    assert got["row_pos"].tolist() == pos and got["row_slot"].tolist() == slot
    assert got["row_req"].tolist() == req and got["anc"].tolist() == anc
    assert got["kv_len_new"].tolist() == [a + n for a, n in zip(kv, counts)]


# ----------------------------------------------------------------- rope

SCALINGS = [None, {"type": "linear", "factor": 4.0}, {"type": "ntk", "factor": 8.0},
            {"type": "yarn", "factor": 4.0, "original_max_position": 32768},
            {"type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
             "original_max_position": 8192}]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("R,Hq,Hk,D,rot,layout,norm,scaling,pos0", [
    (1, 32, 8, 128, 128, "half", True, 0, 2047),
    (1, 1, 1, 16, 16, "interleaved", False, 0, 0),
    (7, 24, 4, 256, 64, "interleaved", False, 1, 131000),
    (13, 6, 2, 64, 32, "half", True, 2, 999),
    (9, 5, 5, 80, 48, "half", False, 3, 100000),
    (67, 8, 2, 96, 96, "interleaved", True, 4, 70000),
    (33, 3, 1, 192, 16, "half", False, 0, 5),
    (130, 4, 2, 512, 512, "half", True, 3, 1 << 20),
])
def test_rope_append(cuda, dtype, R, Hq, Hk, D, rot, layout, norm, scaling, pos0):
    from mlx_dspark_b200 import rope

    g = torch.Generator().manual_seed(R * D + rot)
    B, cap = 3, R + 4
    qkv = torch.randn(R, (Hq + 2 * Hk) * D, generator=g).to(dtype).to(cuda)
    q = qkv[:, : Hq * D].view(R, Hq, D)
    k = qkv[:, Hq * D : (Hq + Hk) * D].view(R, Hk, D)
    v = qkv[:, (Hq + Hk) * D :].view(R, Hk, D)
    qn = (1 + 0.1 * torch.randn(D, generator=g)).to(dtype).to(cuda) if norm else None
    kn = (1 + 0.1 * torch.randn(D, generator=g)).to(dtype).to(cuda) if norm else None
    table = rope.RopeTable(D, rot, theta=1e4, layout=layout, scaling=SCALINGS[scaling], device=cuda)
    rng = random.Random(R)
    pos = [pos0 + rng.randint(0, 9) for _ in range(R)]
    req = [rng.randrange(B) for _ in range(R)]
    slot = rng.sample(range(cap), R)
    mark = torch.full((B, Hk, cap + 5, D), 7.0, dtype=dtype, device=cuda)
    kc, vc = mark.clone()[:, :, :cap], mark.clone()[:, :, 5:]
    keep = qkv.clone()
    out = rope.rope_append(q, k, v, table, _i32(pos, cuda), kc, vc, _i32(slot, cuda),
                           row_req=_i32(req, cuda), q_norm=qn, k_norm=kn)
    assert torch.equal(qkv, keep)
    p = torch.tensor(pos)

    def check(got, x, w):
        x = x.double().cpu()
        want = ref.rope(x, table.inv_freq, table.mscale, p, rot, layout,
                        None if w is None else w.double().cpu())
        size = float(torch.maximum(want.abs().max(), x.abs().max())) * max(table.mscale, 1.0)
        assert ((got.double().cpu() - want).abs() <= U[dtype] * want.abs() + 4e-6 * size + 1e-7).all()

    check(out, q, qn)
    check(torch.stack([kc[b, :, s] for b, s in zip(req, slot)]), k, kn)
    assert torch.equal(torch.stack([vc[b, :, s] for b, s in zip(req, slot)]), v)
    touched = torch.zeros(B, cap, dtype=torch.bool)
    touched[req, slot] = True
    for c in (kc, vc):
        assert (c.cpu().transpose(1, 2)[~touched] == 7.0).all()
    # q alone, in place, gives the same values
    x = q.clone()
    assert rope.rotate(x, table, _i32(pos, cuda), norm=qn, out=x) is x
    assert torch.equal(x, out)


def test_rope_unaligned_views(cuda):
    """Rows and heads that start at odd elements."""
    from mlx_dspark_b200 import rope

    R, H, D = 5, 3, 64
    g = torch.Generator().manual_seed(0)
    buf = torch.randn(R, H * (D + 1) + 1, generator=g).to(BF).to(cuda)
    x = buf[:, 1:].view(R, H, D + 1)[:, :, :D]
    table = rope.RopeTable(D, layout="half", device=cuda)
    pos = _i32([3, 0, 9, 100, 4], cuda)
    a = rope.rotate(x, table, pos)
    b = rope.rotate(x.contiguous(), table, pos)
    assert torch.equal(a, b)
    kc = torch.zeros(1, H, 10, D + 3, dtype=BF, device=cuda)[..., :D]
    vc = torch.zeros_like(kc)
    q = rope.rope_append(x, x, x, table, pos, kc, vc, _i32([0, 2, 4, 6, 8], cuda))
    assert torch.equal(q, b) and torch.equal(kc[0, :, ::2].transpose(0, 1), b)
    assert torch.equal(vc[0, :, ::2].transpose(0, 1), x)


def test_rope_drops_rows_outside_the_cache(cuda):
    from mlx_dspark_b200 import _lib, rope

    D = 64
    table = rope.RopeTable(D, device=cuda)
    x = torch.ones(4, 2, D, dtype=BF, device=cuda)
    kc = torch.zeros(2, 2, 6, D, dtype=BF, device=cuda)
    vc = torch.zeros_like(kc)
    q = rope.rope_append(x, x, x, table, _i32([0, 0, 0, 0], cuda), kc, vc, _i32([6, -1, 0, 5], cuda),
                         row_req=_i32([0, 0, 2, 1], cuda))
    assert _lib.device_status(cuda.index) != 0  # recorded, and cleared by reading
    assert torch.equal(q, x)  # position 0 turns nothing
    assert float(vc.sum()) == 2 * D and float(vc[1, :, 5].sum()) == 2 * D and float(kc[1, :, 5].sum()) == 2 * D


# ----------------------------------------------------------------- attention

def _attn_case(dev, dtype, counts, lens, Hq, Hk, D, parents, seed, scale_q=1.0):
    g = torch.Generator().manual_seed(seed)
    R, B, cap = sum(counts), len(counts), max(lens) + 9
    q = (scale_q * torch.randn(R, Hq, D, generator=g)).to(dtype)
    k = torch.randn(B, Hk, cap, D, generator=g).to(dtype)
    v = torch.randn(B, Hk, cap, D, generator=g).to(dtype)
    return q, k, v


def _check_attn(got, q, k, v, counts, lens, parents, scale, dtype, start=None):
    r0 = 0
    for b, n in enumerate(counts):
        if not n:
            continue
        L, s0 = lens[b], 0 if start is None else start[b]
        kb = k[b] if start is None else k[0]
        vb = v[b] if start is None else v[0]
        anc = ref.ancestors(parents[b])
        vis = torch.zeros(n, L, dtype=torch.bool)
        for i in range(n):
            vis[i, : max(L - n, 0)] = True
            for j in anc[i]:
                if 0 <= L - n + j < L:
                    vis[i, L - n + j] = True
        want, absum, vsum = ref.attention(q[r0 : r0 + n].double(), kb[:, s0 : s0 + L].double(),
                                          vb[:, s0 : s0 + L].double(), vis, scale)
        u = U[dtype]
        bound = (u + 1e-4) * absum + u * want.abs() + (2.0 ** -25 * vsum if dtype == HF else 0) + 1e-7
        err = (got[r0 : r0 + n].double().cpu() - want).abs()
        assert torch.isfinite(want).all() and (err <= bound).all(), (b, float((err - bound).max()))
        r0 += n


ATTN = [
    # counts, lens, Hq, Hk, D
    ([1], [1], 4, 4, 64),
    ([1], [2049], 32, 8, 128),
    ([1, 1, 1], [1, 130, 77], 8, 2, 128),
    ([5], [5], 8, 2, 64),                       # nothing cached before the tree
    ([61], [700], 8, 2, 128),
    ([33, 1, 0, 17], [200, 128, 0, 129], 12, 4, 128),   # groups of 3, an idle request
    ([40, 9], [300, 257], 20, 4, 128),          # groups of 5
    ([100], [1111], 24, 3, 64),                 # groups of 8, 3 kv heads
    ([130, 64, 3], [400, 64, 383], 4, 2, 128),  # more than 128 rows a kv head, a tree from nothing
    ([257], [513], 2, 1, 128),
    ([3], [9000], 7, 1, 64),                    # groups of 7
    ([2], [4100], 64, 1, 128),                  # one kv head for 64
]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("case", range(len(ATTN)))
def test_tree_sdpa(cuda, dtype, case):
    from mlx_dspark_b200 import tree

    counts, lens, Hq, Hk, D = ATTN[case]
    rng = random.Random(case)
    parents = [ref.random_parents(n, rng) if n else [] for n in counts]
    q, k, v = _attn_case(cuda, dtype, counts, lens, Hq, Hk, D, parents, case)
    kg, vg = k.to(cuda), v.to(cuda)
    for b, L in enumerate(lens):  # what lies behind the cached rows takes no part
        kg[b, :, L:] = float("nan")
        vg[b, :, L:] = float("inf")
    words = tree.anc_words(max(counts))
    anc = _i32([w for p in parents if p for w in ref.words_of(ref.ancestors(p), words)], cuda)
    out = tree.tree_sdpa(q.to(cuda), kg, vg, _cu(counts, cuda), _i32(lens, cuda), anc,
                         scale=D ** -0.5, max_nodes=max(counts))
    _check_attn(out, q, k, v, counts, lens, parents, D ** -0.5, dtype)


def test_tree_sdpa_large_scores_and_late_maximum(cuda):
    """Scores that grow along the cache (the running maximum moves in every tile), up to about 90."""
    from mlx_dspark_b200 import tree

    counts, lens, Hq, Hk, D = [9], [1500], 4, 1, 128
    parents = [ref.random_parents(9, random.Random(1))]
    q, k, v = _attn_case(cuda, BF, counts, lens, Hq, Hk, D, parents, 5, 3.0)
    ramp = torch.linspace(-3, 3, k.shape[2])[None, None, :, None]
    k = (k.float() + ramp * q[0, 0].float()).to(BF)
    anc = _i32(ref.words_of(ref.ancestors(parents[0]), 1), cuda)
    out = tree.tree_sdpa(q.to(cuda), k.to(cuda), v.to(cuda), _cu(counts, cuda), _i32(lens, cuda), anc,
                         scale=D ** -0.5, max_nodes=9)
    _check_attn(out, q, k, v, counts, lens, parents, D ** -0.5, BF)


@pytest.mark.parametrize("scale", [-0.11, 0.0, 2.0])
def test_tree_sdpa_scales(cuda, scale):
    """A negative scale, a scale of zero (the mean of what is seen), and a large one."""
    from mlx_dspark_b200 import tree

    counts, lens, Hq, Hk, D = [7, 150], [400, 333], 4, 2, 64
    rng = random.Random(4)
    parents = [ref.random_parents(n, rng) for n in counts]
    q, k, v = _attn_case(cuda, HF, counts, lens, Hq, Hk, D, parents, 11)
    anc = _i32([w for p in parents for w in ref.words_of(ref.ancestors(p), 5)], cuda)
    out = tree.tree_sdpa(q.to(cuda), k.to(cuda), v.to(cuda), _cu(counts, cuda), _i32(lens, cuda), anc,
                         scale=scale, max_nodes=150)
    _check_attn(out, q, k, v, counts, lens, parents, scale, HF)


@pytest.mark.parametrize("batch,nodes,longest", [(40, 9, 700), (23, 70, 900), (200, 3, 300), (9, 33, 5000)])
def test_tree_sdpa_ragged_batches(cuda, batch, nodes, longest):
    """Many requests of mixed sizes: shares that cross from request to request, items in several
    parts, requests beyond one warp's lookup, idle ones between."""
    from mlx_dspark_b200 import tree

    rng = random.Random(batch)
    counts = [rng.choice([0, 1, rng.randint(1, nodes)]) for _ in range(batch)]
    lens = [max(n, rng.choice([n, rng.randint(1, longest)])) for n in counts]
    Hq, Hk, D = 4, 2, 64
    parents = [ref.random_parents(n, rng) if n else [] for n in counts]
    q, k, v = _attn_case(cuda, BF, counts, lens, Hq, Hk, D, parents, batch)
    words = tree.anc_words(nodes)
    anc = _i32([w for p in parents if p for w in ref.words_of(ref.ancestors(p), words)], cuda)
    out = tree.tree_sdpa(q.to(cuda), k.to(cuda), v.to(cuda), _cu(counts, cuda), _i32(lens, cuda), anc,
                         scale=D ** -0.5, max_nodes=nodes)
    _check_attn(out, q, k, v, counts, lens, parents, D ** -0.5, BF)


@pytest.mark.parametrize("batch,nodes,longest,Hq,Hk", [(48, 2, 4000, 16, 8), (20, 19, 3000, 8, 4),
                                                       (24, 40, 2000, 8, 4)])
def test_tree_sdpa_back_to_back(cuda, batch, nodes, longest, Hq, Hk):
    """Calls on two states in turn with nothing between them, head_dim 128 (the short ring): many
    segments a CTA, whose last tiles are put right while other tiles are still on their way. Every
    row of every call against the form in 64 bits: p rounded to the type, the output too."""
    from mlx_dspark_b200 import tree

    rng = random.Random(batch)
    counts = [rng.randint(1, nodes) for _ in range(batch)]
    D, words, calls = 128, tree.anc_words(nodes), []
    for k in range(2):
        lens = [max(n, rng.randint(1, longest)) for n in counts]
        parents = [ref.random_parents(n, rng) for n in counts]
        g = torch.Generator(device=cuda).manual_seed(k)
        q = torch.randn(sum(counts), Hq, D, device=cuda, generator=g).to(HF)
        kc, vc = (torch.randn(batch, Hk, max(lens) + 5, D, device=cuda, generator=g).to(HF) for _ in range(2))
        anc = _i32([w for p in parents for w in ref.words_of(ref.ancestors(p), words)], cuda)
        want, bound, r0 = torch.empty(q.shape, device=cuda, dtype=torch.float64), torch.empty_like(q, dtype=torch.float64), 0
        for b, n in enumerate(counts):
            sees = torch.ones(n, lens[b], dtype=torch.bool)
            for i, a in enumerate(ref.ancestors(parents[b])):
                sees[i, lens[b] - n :] = False
                sees[i, [lens[b] - n + j for j in a]] = True
            qb = q[r0 : r0 + n].double().view(n, Hk, Hq // Hk, D)
            z = torch.einsum("nhgd,hld->hgnl", qb, kc[b, :, : lens[b]].double()) * D ** -0.5
            w = torch.softmax(z.masked_fill(~sees.to(cuda), float("-inf")), -1)
            v = vc[b, :, : lens[b]].double()
            o = torch.einsum("hgnl,hld->nhgd", w, v).reshape(n, Hq, D)
            absum = torch.einsum("hgnl,hld->nhgd", w, v.abs()).reshape(n, Hq, D)
            want[r0 : r0 + n] = o
            bound[r0 : r0 + n] = (U[HF] + 1e-4) * absum + U[HF] * o.abs() + 2.0 ** -25 * v.abs().sum(1).amax() + 1e-7
            r0 += n
        calls.append((q, kc, vc, _cu(counts, cuda), _i32(lens, cuda), anc, want, bound))
    outs = []
    for k in range(24):
        c = calls[k % 2]
        outs.append(tree.tree_sdpa(*c[:6], scale=D ** -0.5, max_nodes=nodes))
    for k, out in enumerate(outs):
        assert ((out.double() - calls[k % 2][6]).abs() <= calls[k % 2][7]).all(), k


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_tree_sdpa_hidden_keys_take_no_part(cuda, bad):
    """A branch with non-finite keys and values spoils its own descendants only."""
    from mlx_dspark_b200 import tree

    counts, lens, Hq, Hk, D = [70], [333], 8, 2, 128
    parents = [[-1, 0, 0] + [1 if i % 2 else 2 for i in range(3, 70)]]  # leaves below 1 (odd) and 2 (even)
    q, k, v = _attn_case(cuda, BF, counts, lens, Hq, Hk, D, parents, 3)
    kg, vg = k.to(cuda), v.to(cuda)
    first = lens[0] - counts[0]
    for j in (1, 3, 69):  # the odd branch
        kg[0, :, first + j] = bad
        vg[0, :, first + j] = bad
    anc = _i32(ref.words_of(ref.ancestors(parents[0]), 3), cuda)
    out = tree.tree_sdpa(q.to(cuda), kg, vg, _cu(counts, cuda), _i32(lens, cuda), anc, scale=D ** -0.5,
                         max_nodes=70)
    clean = tree.tree_sdpa(q.to(cuda), k.to(cuda), v.to(cuda), _cu(counts, cuda), _i32(lens, cuda), anc,
                           scale=D ** -0.5, max_nodes=70)
    even = [0, 2] + list(range(4, 70, 2))
    _check_attn(clean, q, k, v, counts, lens, parents, D ** -0.5, BF)
    assert torch.equal(out[even], clean[even])
    assert not torch.isfinite(out[[1] + list(range(3, 70, 2))]).any()


def test_tree_sdpa_rows_that_see_nothing(cuda):
    from mlx_dspark_b200 import tree

    D = 64
    q = torch.randn(40, 4, D, device=cuda).to(BF)
    k = torch.randn(1, 2, 64, D, device=cuda).to(BF)
    anc = torch.zeros(40, 2, dtype=torch.int32, device=cuda)
    anc[7, 0] = 1 << 3
    out = tree.tree_sdpa(q, k, k, _cu([40], cuda), _i32([40], cuda), anc, scale=0.1, max_nodes=40)
    assert torch.equal(out[7], k[0, :, 3].repeat_interleave(2, 0))
    out[7] = 0
    assert not out.any()


def test_tree_sdpa_chain_pool_strides_and_stream(cuda):
    """anc None is the causal rule; a position-major pool with starts; heads-last q; a side stream."""
    from mlx_dspark_b200 import tree

    counts, lens, Hq, Hk, D = [20, 1, 37], [90, 300, 37], 8, 4, 128
    parents = [list(range(-1, n - 1)) for n in counts]
    g = torch.Generator().manual_seed(9)
    start = [300, 0, 420]
    pool_k = torch.randn(500, Hk, D, generator=g).to(HF)
    pool_v = torch.randn(500, Hk, D, generator=g).to(HF)
    q = torch.randn(Hq, sum(counts), D, generator=g).to(HF).transpose(0, 1)
    side = torch.cuda.Stream()
    qg, kg, vg = q.to(cuda), pool_k.to(cuda), pool_v.to(cuda)
    cu, ln, st = _cu(counts, cuda), _i32(lens, cuda), _i32(start, cuda)
    out = torch.empty(sum(counts), D, Hq, dtype=HF, device=cuda).transpose(1, 2).contiguous()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        tree.tree_sdpa(qg, kg.permute(1, 0, 2)[None], vg.permute(1, 0, 2)[None], cu, ln, None,
                       scale=D ** -0.5, max_nodes=37, kv_start=st, out=out)
    torch.cuda.current_stream().wait_stream(side)
    _check_attn(out, q, pool_k.permute(1, 0, 2)[None], pool_v.permute(1, 0, 2)[None], counts, lens,
                parents, D ** -0.5, HF, start)


def test_tree_sdpa_offsets_past_32_bits(cuda):
    """A cache entry that starts more than 2^31 elements into the pool."""
    from mlx_dspark_b200 import tree

    D, Hk, P = 128, 8, 2_200_000  # 2.25e9 elements each
    free, _ = torch.cuda.mem_get_info()
    if free < 12 << 30:
        pytest.skip("needs 10 GB of device memory")
    pk = torch.zeros(P, Hk, D, dtype=BF, device=cuda)
    pv = torch.zeros(P, Hk, D, dtype=BF, device=cuda)
    counts, lens, start = [6, 4], [190, 100], [P - 200, 50]
    g = torch.Generator().manual_seed(2)
    tail_k, tail_v = (torch.randn(200, Hk, D, generator=g).to(BF) for _ in range(2))
    pk[-200:], pv[-200:] = tail_k.to(cuda), tail_v.to(cuda)
    q = torch.randn(10, 16, D, generator=g).to(BF)
    out = tree.tree_sdpa(q.to(cuda), pk.permute(1, 0, 2)[None], pv.permute(1, 0, 2)[None],
                         _cu(counts, cuda), _i32(lens, cuda), None, scale=D ** -0.5, max_nodes=6,
                         kv_start=_i32(start, cuda))
    _check_attn(out[:6], q[:6], tail_k.permute(1, 0, 2)[None], tail_v.permute(1, 0, 2)[None], [6], [190],
                [list(range(-1, 5))], D ** -0.5, BF, [0])
    assert not out[6:].any()


# ----------------------------------------------------------------- sampled accept

def _accept_case(counts, V, tree, draft, seed, dtype, sharp=4.0):
    rng = np.random.default_rng(seed)
    R, B = sum(counts), len(counts)
    logits = torch.tensor(sharp * rng.standard_normal((R, V)), dtype=torch.float32).to(dtype)
    pr = random.Random(seed)
    parents = [ref.random_parents(n, pr) if n else [] for n in counts]
    ids = np.zeros(R, dtype=np.int64)
    q = None
    if draft is not None:
        q = torch.softmax(logits.float() + torch.tensor(rng.standard_normal((R, V)), dtype=torch.float32),
                          -1).to(draft)
    r0 = 0
    for n, par in zip(counts, parents):
        for i in range(n):
            up = r0 + (par[i] if tree else i - 1)
            if i == 0:
                ids[r0] = rng.integers(V)
            elif q is not None:
                w = q[up].double().numpy()
                ids[r0 + i] = rng.choice(V, p=w / w.sum())
            else:
                top = np.argsort(-logits[up].float().numpy(), kind="stable")[:4]
                ids[r0 + i] = top[rng.integers(len(top))]
        r0 += n
    u = rng.random(R).astype(np.float32)
    noise = rng.exponential(size=(B, V)).astype(np.float32)
    temp = (0.4 + rng.random(B)).astype(np.float32)
    temp[rng.random(B) < 0.25] = 0.0
    return logits, parents, ids, q, u, noise, temp


ACCEPT = [
    # counts, V, tree, draft type
    ([1], 17, False, None),
    ([1], 17, True, None),
    ([5], 151936, False, None),
    ([4, 0, 1, 16, 2], 5003, False, BF),
    ([7, 7, 7], 4096, False, FP),
    ([3, 12], 32001, False, HF),
    ([61, 1, 0, 40], 2051, True, None),
    ([20] * 9, 999, True, None),
    ([200], 50, True, None),
    ([9] * 40, 130, False, BF),
    ([2, 2], 2, False, None),
    ([3], 1, False, None),
]


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("case", range(len(ACCEPT)))
def test_sample_accept(cuda, dtype, case):
    from mlx_dspark_b200 import sampling

    counts, V, tree, draft = ACCEPT[case]
    logits, parents, ids, q, u, noise, temp = _accept_case(counts, V, tree, draft, case, dtype)
    R, B = sum(counts), len(counts)
    lens = _i32([100 + n for n in counts], cuda)
    wide = torch.full((R, V + 3), float("nan"), dtype=dtype, device=cuda)
    wide[:, :V] = logits.to(cuda)
    got = sampling.sample_accept(
        wide[:, :V], _i32(ids.tolist(), cuda), _cu(counts, cuda), torch.tensor(u, device=cuda),
        torch.tensor(noise, device=cuda), temperature=torch.tensor(temp, device=cuda),
        draft_probs=None if q is None else q.to(cuda),
        parent=_i32([p for x in parents for p in x], cuda) if tree else None, max_rows=max(counts), lens=lens)
    n, nxt, prob, path = (got[k].cpu().numpy() for k in ("n", "next", "prob", "path"))
    r0 = told_apart = 0
    for b, cnt in enumerate(counts):
        if not cnt:
            assert n[b] == 0 and nxt[b] == -1 and int(lens[b]) == 100
            continue
        T = float(temp[b])
        rows = slice(r0, r0 + cnt)
        p = ref.probabilities(logits[rows].float().numpy(), T)
        want = [1.0] + [p[parents[b][i] if tree else i - 1, ids[r0 + i]] for i in range(1, cnt)]
        span = 200.0 / max(T, 0.4)
        np.testing.assert_allclose(prob[rows], want, rtol=2.0 ** -23 * (span + 8), atol=1e-30)
        pth, tok, close = ref.accept(p, ids[rows].tolist(), parents[b] if tree else None, u[rows], noise[b],
                                     None if q is None else q[rows].float().numpy(), T == 0)
        if close:
            told_apart += 1
        else:
            assert n[b] == len(pth) - 1 and nxt[b] == tok, (b, n[b], pth, nxt[b], tok)
            assert path[rows].tolist() == pth + [-1] * (cnt - len(pth))
            assert int(lens[b]) == 100 + len(pth)
        r0 += cnt
    assert told_apart <= 1 + len(counts) // 20


def test_sample_accept_masked_logits(cuda):
    """-inf, NaN, +inf and the type's lowest value; a row with no mass; a draft outside the vocabulary."""
    from mlx_dspark_b200 import sampling

    V = 77
    lo = torch.finfo(BF).min
    rows = torch.full((9, V), float("-inf"), dtype=BF)
    rows[0, 5], rows[0, 6] = 1.0, float("nan")          # request 0: only token 5
    rows[1, :] = lo                                      # then everything equal
    rows[2, 3] = float("inf")                            # request 1: +inf takes all
    rows[2, 8] = 4.0
    # row 3 has no mass
    rows[4, 10], rows[4, 11] = lo, 0.0                   # request 2: the lowest value has none next to 0
    rows[5, 12] = 2.0
    rows[6, :] = float("nan")                            # request 3: nothing at all
    rows[7, 20] = 1.0                                    # request 4: draft outside the vocabulary
    counts = [2, 2, 2, 1, 2]
    ids = [0, 5, 0, 3, 0, 11, 0, 0, V + 4]
    noise = torch.ones(5, V)
    noise[0, 9] = 0.5
    for T in (1.0, 0.7):
        got = sampling.sample_accept(rows.to(cuda), _i32(ids, cuda), _cu(counts, cuda),
                                     torch.full((9,), 0.999, device=cuda), noise.to(cuda),
                                     temperature=torch.full((5,), T, device=cuda), max_rows=2)
        assert got["n"].tolist() == [1, 1, 1, 0, 0]
        assert got["next"].tolist() == [9, -1, 12, -1, 20]
        assert got["prob"].tolist() == [1, 1, 1, 1, 1, 1, 1, 1, 0]


def test_sample_accept_ties_go_to_the_first(cuda):
    from mlx_dspark_b200 import sampling

    V = 40000
    logits = torch.zeros(2, V, dtype=HF, device=cuda)
    noise = torch.ones(2, V, device=cuda)
    got = sampling.sample_accept(logits, _i32([0, 0], cuda), _cu([1, 1], cuda), torch.zeros(2, device=cuda),
                                 noise, temperature=torch.tensor([0.0, 1.0], device=cuda), max_rows=1)
    assert got["next"].tolist() == [0, 0]
    logits[:, 31003] = 3.0
    logits[:, 39990] = 3.0
    got = sampling.sample_accept(logits, _i32([0, 0], cuda), _cu([1, 1], cuda), torch.zeros(2, device=cuda),
                                 noise, temperature=torch.tensor([0.0, 1.0], device=cuda), max_rows=1)
    assert got["next"].tolist() == [31003, 31003]


def test_sample_accept_into_a_former_result(cuda):
    """The tensors and the workspace of a former call are used again, also for more slices a row and on
    another stream, with the result of a call that makes its own."""
    from mlx_dspark_b200 import sampling

    out = None
    side = torch.cuda.Stream()
    g = torch.Generator().manual_seed(7)
    for V, stream in ((500, None), (90000, None), (30011, side), (90000, side), (500, None)):
        logits = torch.randn(6, V, generator=g).to(cuda)
        u, noise = torch.rand(6, generator=g).to(cuda), torch.empty(2, V).exponential_(generator=g).to(cuda)
        ids = _i32([0] + logits[:3].argmax(1).tolist() + [1] + logits[4:5].argmax(1).tolist(), cuda)
        a = (logits, ids, _cu([4, 2], cuda), u, noise)
        kw = dict(temperature=torch.tensor([0.1, 0.3], device=cuda), max_rows=4)
        want = sampling.sample_accept(*a, **kw)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            out = sampling.sample_accept(*a, **kw, out=out)
        torch.cuda.synchronize()
        for k in ("n", "next", "prob", "path"):
            assert torch.equal(out[k], want[k]), (V, k)


@pytest.mark.parametrize("form", ["chain", "draft", "tree"])
def test_sample_accept_keeps_the_targets_distribution(cuda, form):
    """The first emitted token of 60000 rounds is distributed as p: each frequency within five
    standard deviations (chance of a false alarm below 1e-4)."""
    from mlx_dspark_b200 import sampling

    N, V = 60000, 8
    g = torch.Generator().manual_seed({"chain": 0, "draft": 1, "tree": 2}[form])
    l = 1.5 * torch.randn(V, generator=g)
    p = torch.softmax(l.double() / 0.8, 0)
    q = torch.softmax(1.5 * torch.randn(V, generator=g), 0)
    rows = 4 if form == "tree" else 2
    logits = l.repeat(N * rows, 1).to(cuda)
    ids = torch.zeros(N, rows, dtype=torch.int32)
    if form == "draft":
        ids[:, 1] = torch.multinomial(q, N, True, generator=g).int()
    elif form == "chain":
        ids[:, 1] = int(l.argmax())
    else:
        ids[:, 1:] = torch.tensor([2, 5, 2])  # three children of the root, one of them twice
    parent = _i32([-1, 0, 0, 0] * N, cuda) if form == "tree" else None
    got = sampling.sample_accept(
        logits, ids.flatten().to(cuda), _i32(list(range(0, N * rows + 1, rows)), cuda),
        torch.rand(N * rows, generator=g).to(cuda), torch.empty(N, V).exponential_(generator=g).to(cuda),
        temperature=torch.full((N,), 0.8, device=cuda), parent=parent, max_rows=rows,
        draft_probs=q.repeat(N * rows, 1).to(cuda) if form == "draft" else None)
    n, nxt = got["n"].cpu(), got["next"].cpu().long()
    path = got["path"].cpu().view(N, rows)
    first = torch.where(n > 0, ids.gather(1, path[:, 1:2].clamp(min=0).long())[:, 0].long(), nxt)
    freq = torch.bincount(first, minlength=V).double() / N
    assert ((freq - p).abs() <= 5 * torch.sqrt(p * (1 - p) / N)).all(), (freq, p)


# ----------------------------------------------------------------- kept path

@pytest.mark.parametrize("dtype,H,D,layers,pool", [(BF, 8, 128, 3, False), (HF, 1, 64, 2, True),
                                                   (BF, 3, 256, 5, False), (FP, 2, 20, 1, False)])
def test_keep_path(cuda, dtype, H, D, layers, pool):
    from mlx_dspark_b200 import tree

    rng = random.Random(D)
    counts = [61, 1, 0, 9, 40, 33]
    cap, B = 90, len(counts)
    base = [rng.randint(0, cap - 61 - 1) if n else 7 for n in counts]
    g = torch.Generator().manual_seed(D)
    shape = (B, H, cap, D)
    start = None
    if pool:
        start = [b * cap for b in range(B)]
        ks, vs = ([torch.randn(B * cap, H, D, generator=g).to(dtype).to(cuda).permute(1, 0, 2)[None]
                   for _ in range(layers)] for _ in range(2))
    else:
        ks, vs = ([torch.randn(shape, generator=g).to(dtype).to(cuda) for _ in range(layers)]
                  for _ in range(2))
    paths = []
    for i, n in enumerate(counts):
        depth = [0, 0, 0, 8, 20, 30][i]
        paths.append([0] + sorted(rng.sample(range(1, n), min(depth, n - 1))) if n else [])
    paths[0] = [0] + list(range(21, 61))  # 40 rows that move onto one another
    flat = [x for p, n in zip(paths, counts) for x in p + [-1] * (n - len(p))]
    want = [[t.clone() for t in x] for x in (ks, vs)]
    for group in want:
        for t in group:
            old = t.clone()
            for b, p in enumerate(paths):
                for i, x in enumerate(p):
                    if pool:
                        t[0, :, start[b] + base[b] + i] = old[0, :, start[b] + base[b] + x]
                    else:
                        t[b, :, base[b] + i] = old[b, :, base[b] + x]
    n_acc = [max(len(p) - 1, 0) for p in paths]
    lens = [base[b] + (len(p) if p else 0) for b, p in enumerate(paths)]
    tree.PathKeeper(ks, vs).keep(_i32(flat, cuda), _cu(counts, cuda), _i32(n_acc, cuda), _i32(lens, cuda),
                                 kv_start=None if start is None else _i32(start, cuda))
    for got, exp in zip((ks, vs), want):
        for a, b in zip(got, exp):
            assert torch.equal(a, b)
