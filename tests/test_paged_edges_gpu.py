"""The paged 8-bit cache and token scores on the GPU where calls meet an edge: NaN codes beside the rows' own keys,
zeros of either sign among the logits, begun pages without a scale,
q of no number in rows that see nothing."""

from __future__ import annotations

import math
import random

import paged_reference as ref
import pytest
import torch
from test_paged_gpu import (BF, FP, HF, _append_values, _check_scores, _cpu, _cu, _far, _finite_pool, _i32, _identity, _pool,
                            _tables, _with_room)

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------- NaN codes of v

NAN_VALUES = [
    # counts, lens, Hq, Hk, D, page, type: with far tables all go to the kernel for many rows
    ([20], [470], 2, 1, 64, 16, BF),                     # 40 rows: the slots share them; items cut at every tile
    ([80], [470], 2, 1, 64, 16, HF),                     # 160 rows: a slot each
    ([40, 3, 90], [129, 700, 333], 8, 2, 128, 32, HF),   # requests that begin inside a tile
    ([33] * 70, [33 + 37 * i % 800 for i in range(70)], 8, 4, 64, 64, BF),   # whole items and cut ones, 66 rows each
    ([50] * 60, [128 + 53 * i % 700 for i in range(60)], 16, 2, 64, 128, BF),  # 400 rows: pairs of slots and a rest
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("far", [True, False])
@pytest.mark.parametrize("case", NAN_VALUES, ids=range(len(NAN_VALUES)))
def test_nan_values_reach_all_rows_that_see_them(cuda, case, far, causal):
    """A NaN code of v just before the rows' own keys, at the first key of the 128 that hold the first of them, just before
    those, and among the own ones: it makes exactly the values NaN that it belongs to, of every row that sees its key."""
    counts, lens, Hq, Hk, D, page, dt = case
    rng, g = random.Random(D + page), torch.Generator().manual_seed(len(counts) + page)
    need = [-(-x // page) for x in lens]
    cache = _finite_pool(cuda, sum(need) + 2, Hk, page, D, g)
    rows = _tables(need, sum(need) + 2, rng)
    table = _i32(_far(rows, page) if far else rows, cuda)
    q = torch.randn(sum(counts), Hq, D, generator=g).to(dt).to(cuda)
    cu, ln = _cu(counts, cuda), _i32(lens, cuda)
    clean = cache.attention(q, cu, ln, table, scale=0.1, causal=causal)
    assert not bool(clean.isnan().any())
    codes, before = cache.v.view(torch.uint8), [x - n for n, x in zip(counts, lens)]
    for place in range(4):
        kept, want = codes.clone(), torch.zeros(clean.shape, dtype=torch.bool)
        r0 = 0
        for b, (n, x) in enumerate(zip(counts, lens)):
            first = before[b] // 128 * 128
            key = max((before[b] - 1, first, first - 1, before[b] + n // 2)[place], 0)
            h, d = rng.randrange(Hk), rng.randrange(D)
            codes[rows[b][key // page], h, key % page, d] = rng.choice([0x7F, 0xFF])
            sees = max(0, key - before[b]) if causal else 0  # the first row that does
            want[r0 + sees : r0 + n, h * (Hq // Hk) : (h + 1) * (Hq // Hk), d] = True
            r0 += n
        out = cache.attention(q, cu, ln, table, scale=0.1, causal=causal)
        codes.copy_(kept)
        assert torch.equal(out.isnan().cpu(), want), place
        assert torch.equal(out.cpu()[~want], clean.cpu()[~want]), place


def test_a_nan_value_in_a_long_prompt_holds_nobody_up(cuda):
    """Putting a NaN code back is a few tiles' work for every row block, however many rows the request has: the kernel's waits
    do not run out meanwhile, here after 20 ms."""
    from mlx_dspark_b200 import _lib

    R, before, page, D, Hk, Hq = 16384, 77, 64, 128, 1, 4
    g = torch.Generator().manual_seed(3)
    n = -(-(R + before) // page)
    cache = _finite_pool(cuda, n, Hk, page, D, g)
    q = torch.randn(R, Hq, D, generator=g).to(BF).to(cuda)
    args = _cu([R], cuda), _i32([R + before], cuda), _i32([list(range(n))], cuda)
    clean = cache.attention(q, *args, scale=0.1)
    places = [R // 3, R - 1]
    for i in places:
        cache.v.view(torch.uint8)[(before + i) // page, 0, (before + i) % page, 7 + i % 3] = 0x7F
    _lib.set_wait_limit_ns(cuda.index, 20_000_000)
    try:
        out = cache.attention(q, *args, scale=0.1)
        torch.cuda.synchronize()
        assert _lib.device_status(cuda.index) == 0
    finally:
        _lib.set_wait_limit_ns(cuda.index, 0)
    want = torch.zeros(out.shape, dtype=torch.bool, device=cuda)
    for i in places:
        want[i:, :, 7 + i % 3] = True
    assert torch.equal(out.isnan(), want) and torch.equal(out[~want], clean[~want])


# ------------------------------------------------------------------------------- zeros of either sign

def _zeros(V, dt, at, g):
    """Rows of negative logits with zeros at the given places: {token: sign}."""
    x = (-1 - torch.rand(len(at), V, generator=g)).to(dt)
    for r, row in enumerate(at):
        for token, sign in row.items():
            x[r, token] = sign * 0.0
    return x


@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("rows,V", [(1, 600), (1, 151937), (40, 9001)])  # one block a row, a cluster, ragged rows of a cluster
def test_zeros_of_either_sign_are_one_logit(cuda, dt, rows, V):
    """-0 and +0 are equal: the lower token comes first, in the rank and in the alternatives, greedy or not, at the head and at
    the end of the list, and where more values are equal than a block sorts at once."""
    from mlx_dspark_b200 import sampling

    g = torch.Generator().manual_seed(V)
    at = [{5: -1, V - 2: 1}, {5: 1, V - 2: -1}, {0: -1, 7: 1, V // 2: -1, V - 1: 1}, {V - 1: -1, V // 2: 1, 3: 1}]
    x = _zeros(V, dt, at, g)
    many = x.repeat(rows, 1).to(cuda)
    for temp in (None, 0.0, 0.7):
        T = None if temp is None else torch.full((4 * rows,), temp, device=cuda)
        for pick in (min, max):
            tokens = [pick(a) for a in at]
            _check_scores(cuda, x, tokens, None if temp is None else [temp] * 4, 3)
            for top in (1, 2, 3, 20, 32):
                got = sampling.token_logprobs(many, _i32(tokens * rows, cuda), temperature=T, top=top)
                ids, rank, lp = (got[k].tolist() for k in ("top_ids", "rank", "logprob"))
                for r in range(4 * rows):
                    a = at[r % 4]
                    assert ids[r][: len(a)] == sorted(a)[:top] and rank[r] == sorted(a).index(pick(a))
                    if rank[r] < top:  # the alternative in its place is the token itself
                        assert got["top_logprobs"][r, rank[r]].item() == lp[r]
    # a larger value before them, and the list's end among them
    x[:, 11] = 1.0
    _check_scores(cuda, x[:4], [max(a) for a in at], None, 2)
    # zeros of both signs everywhere, in turn and at random
    y = torch.zeros(3, V, dtype=dt)
    y[0, ::2] = -0.0
    y[1, 1::2] = -0.0
    y[2] = torch.where(torch.rand(V, generator=g) < 0.5, -0.0, 0.0).to(dt)
    for temp in (None, [0.0, 1.0, 0.0]):
        got = _check_scores(cuda, y, [0, 1, V - 1], temp, 32)
        assert got["top_ids"].tolist() == [list(range(32))] * 3 and got["rank"].tolist() == [0, 1, V - 1]


# ------------------------------------------------------------------------------- begun pages without a scale

@pytest.mark.parametrize("scale", [0.0, -0.25, -1e30, math.nan])
@pytest.mark.parametrize("page,D,n", [(16, 64, 3), (64, 128, 50), (128, 64, 120)])
def test_append_to_a_begun_page_without_a_scale(cuda, page, D, n, scale):
    """Tokens of a page whose scale is not positive keep their values, code * scale, under the scale that the new tokens give the
    page (a NaN one: zeros), instead of becoming whatever their codes mean under it."""
    begin, g = 5, torch.Generator().manual_seed(page)
    cache = _pool(cuda, 3, 2, page, D, g)
    for t in (cache.k_scale, cache.v_scale):
        t[1, 0] = scale  # the other head's page has one
    x, y = (3 * torch.randn(n, 2, D, generator=g).to(BF) for _ in range(2))
    old = _cpu(cache)
    _append_values(cuda, cache, _i32([[1]], cuda), begin, x, y, _identity(cuda, D))
    new = _cpu(cache)
    for i, z in ((0, x), (1, y)):
        lo, hi, s_lo, s_hi = ref.append(old[i], old[i + 2].nan_to_num(0.0), [1], begin, z.double(), torch.zeros(n, 2, D))
        assert torch.equal(lo.nan_to_num(-1), hi.nan_to_num(-1)) and torch.equal(new[i + 2].double(), s_lo)
        got, want = new[i].double(), lo
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))


# ------------------------------------------------------------------------------- pools that share their memory

def test_pools_that_share_memory_are_read_but_not_written(cuda):
    """One scale for all pages, as an expanded tensor, and k that is v: the attention reads them, an append is refused. A pool of
    one page or one head may have any stride there."""
    from mlx_dspark_b200 import DSparkError, paged

    g = torch.Generator().manual_seed(1)
    own = _finite_pool(cuda, 4, 2, 16, 64, g)
    own.k_scale.fill_(0.5), own.v_scale.fill_(0.5)
    one = torch.full((1, 1), 0.5, device=cuda).expand(4, 2)
    x, table = torch.randn(5, 2, 64, generator=g).to(BF).to(cuda), _i32([[3, 1]], cuda)
    args = x, _cu([5], cuda), _i32([20], cuda), table
    want = own.attention(*args, scale=0.1)
    shared = paged.PagedCache(own.k, own.v, one, one)
    assert torch.equal(shared.attention(*args, scale=0.1), want)
    same = paged.PagedCache(own.k, own.k, own.k_scale, own.k_scale)
    assert not bool(same.attention(*args, scale=0.1).isnan().any())
    for bad in (shared, same, paged.PagedCache(own.k, own.v, own.k_scale, own.k_scale),
                paged.PagedCache(own.k[:1].expand(4, 2, 16, 64), own.v, own.k_scale, own.v_scale)):
        with pytest.raises(DSparkError, match="share"):
            _append_values(cuda, bad, table, 15, x.cpu(), x.cpu(), _identity(cuda, 64))
    none = torch.empty(0, 2, 64, dtype=BF)  # no rows: nothing is written but the lengths
    assert _append_values(cuda, shared, table, 15, none, none, _identity(cuda, 64))[1].tolist() == [15]
    single = paged.PagedCache(own.k[:1, :1].as_strided((1, 1, 16, 64), (0, 0, 64, 1)), own.v[:1, :1],
                              one[:1, :1].clone().as_strided((1, 1), (0, 0)), one[:1, :1].clone().as_strided((1, 1), (0, 0)))
    y = torch.zeros(1, 1, 64, dtype=BF)
    _append_values(cuda, single, _i32([[0]], cuda), 0, y, y, _identity(cuda, 64))
    assert single.k_scale.item() == 2.0 ** -64


# ------------------------------------------------------------------------------- q of no number

@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("room", ["tight", "clusters", "shares", "far"])
@pytest.mark.parametrize("n,dt", [(3, BF), (3, HF), (12, BF), (40, HF), (90, BF)])
def test_q_of_no_number_in_rows_that_see_nothing(cuda, n, dt, room, causal):
    """An infinite or NaN q makes its head NaN where the row sees a key, and takes no part where it sees none: more rows than keys,
    no keys, pages that are not there or have no positive scale."""
    from mlx_dspark_b200 import _lib

    g, D, page, dev = torch.Generator().manual_seed(n), 64, 16, cuda.index
    cache = _finite_pool(cuda, 40, 2, page, D, g)
    cache.k_scale[20:30] = 0.0
    rows = [list(range(20)), list(range(30, 36)), [33], [20, 21, 22], [-1, -1], [20, 34, -1]]
    lens = [300, max(n - 2, 1), 0, 40, 20, 48]
    tables = {"tight": lambda r: r, "clusters": lambda r: _with_room(r, page, 6000),
              "shares": lambda r: _with_room(r, page, 40000), "far": lambda r: _far(r, page)}[room]
    width = max(map(len, rows))
    table = _i32(tables([r + [-1] * (width - len(r)) for r in rows]), cuda)
    counts = [n] * len(rows)
    q = torch.randn(n * len(rows), 4, D, generator=g).to(dt)
    bad = torch.zeros(n * len(rows), 4, dtype=torch.bool)
    for r in range(bad.shape[0]):
        if r % 3 != 1:
            h, value = r % 4, (math.inf, math.nan, -math.inf)[r % 7 % 3]
            q[r, h, (5 * r) % D] = value
            bad[r, h] = True
    sees = torch.zeros(n * len(rows), dtype=torch.bool)
    for b, x in enumerate(lens):
        for i in range(n):
            last = x - n + i + 1 if causal else x  # keys before it
            seen = [j for j in range(max(0, min(x, last))) if 0 <= rows[b][j // page] < 20 or rows[b][j // page] >= 30]
            sees[b * n + i] = bool(seen)
    out = cache.attention(q.to(cuda), _cu(counts, cuda), _i32(lens, cuda), table, scale=0.2, causal=causal).cpu()
    clean = cache.attention(torch.where(bad[..., None], 1.0, q).to(dt).to(cuda), _cu(counts, cuda), _i32(lens, cuda), table,
                            scale=0.2, causal=causal).cpu()
    assert _lib.device_status(dev) != 0  # (the pages that are not there)
    assert bool((out[~sees] == 0).all())
    want = bad & sees[:, None]
    assert torch.equal(out.isnan().any(-1), want) and bool(out[want].isnan().all())
    assert torch.equal(out[~want], clean[~want])
