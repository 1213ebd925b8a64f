"""The paged 8-bit cache and token scores on the GPU, against 64 bits.

Bounds. A rotated key of a pair (a, b) is off by at most 2^-20 (|a| + |b|) before it is rounded to a code: the norm's
reciprocal root and the cosine and sine are good to 2^-21 each, the rest is fp32. Codes then lie between those of the
ends, values that are not rotated are exact.

Attention, with A = sum p |v| (p the normalised weights) and S the largest scale * sum |q_d k_d| of a visible key: a
score is off by at most S (D + 8) 2^-23 (fp32 products and sums, whichever way the tensor core cuts them off), a weight
relatively by eps = ln 2 * 2^-21 |log2 weight| + twice that + 2^-22 and by half an fp16 step, 2^-11; the denominator has no
fp16 step. Sums of n terms add n 2^-24. The result is rounded to its type, half a step. What fp16 loses of a weight far
below the largest is at most 2^-36 of it a key: it counts with sum |v|.

Half a step of a type is eps / 2 of the value down to its smallest normal number, tiny, and stays tiny * eps / 2 below (fp16:
subnormal values are 2^-24 apart, half of that is 2^-25 = 2^-14 * 2^-10 / 2).
"""

from __future__ import annotations

import math
import random

import paged_reference as ref
import pytest
import torch
import tree_reference

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
E4M3 = torch.float8_e4m3fn


def _half_step(dt, x):
    f = torch.finfo(dt)
    return f.eps / 2 * x.abs().clamp(min=f.tiny)


def _i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _cu(counts, dev):
    at = [0]
    for n in counts:
        at.append(at[-1] + n)
    return _i32(at, dev)


def _tables(need, n_pages, rng, width=None):
    """A table of different pages for each request; places behind its last hold -1."""
    ids = rng.sample(range(n_pages), sum(need))
    width = width or max(1, max(need))
    rows, at = [], 0
    for n in need:
        rows.append(ids[at : at + n] + [-1] * (width - n))
        at += n
    return rows


def _pool(cuda, pages, H, page, D, g, layout="heads"):
    """A cache full of random codes (NaN codes among them) and scales."""
    from mlx_dspark_b200 import paged

    shape = (pages, H, page, D) if layout == "heads" else (pages, page, H, D)
    made = []
    for _ in range(2):
        x = torch.randint(0, 256, shape, generator=g, dtype=torch.uint8).to(cuda)
        made.append((x if layout == "heads" else x.permute(0, 2, 1, 3)).view(E4M3) if layout == "heads"
                    else x.view(E4M3).permute(0, 2, 1, 3))
    sc = [torch.exp2(torch.randint(-7, 0, (pages, H), generator=g).float()).to(cuda) for _ in range(2)]
    return paged.PagedCache(made[0], made[1], *sc)


def _cpu(cache):
    """Copies of codes (contiguous) and scales."""
    u8 = lambda t: t.view(torch.uint8).cpu().contiguous().clone().view(E4M3)  # noqa: E731
    return u8(cache.k), u8(cache.v), cache.k_scale.cpu().clone(), cache.v_scale.cpu().clone()


def _same_codes(a, b):
    return torch.equal(a.view(torch.uint8), b.view(torch.uint8))


# ------------------------------------------------------------------------------- append

APPENDS = [
    # counts, cached before, Hq, Hk, D, rot, layout, page, type, norm, pool layout, own positions
    ([1], [0], 4, 1, 128, 128, "half", 64, BF, True, "heads", False),
    ([1, 1, 1], [63, 64, 65], 8, 2, 128, 128, "half", 64, BF, False, "heads", False),
    ([0, 5, 0, 17, 0], [9, 15, 16, 31, 0], 6, 2, 64, 32, "interleaved", 16, HF, True, "heads", False),
    ([3, 1, 40], [1, 30, 33], 7, 1, 64, 64, "half", 32, BF, False, "tokens", True),
    ([130, 1], [127, 128], 8, 8, 128, 64, "half", 128, HF, True, "tokens", False),
    ([300], [37], 5, 5, 128, 96, "interleaved", 128, BF, False, "heads", True),
    ([33, 64, 16, 15], [0, 64, 1, 17], 16, 2, 128, 16, "half", 16, HF, False, "heads", False),
    ([1] * 70, list(range(70)), 2, 1, 64, 64, "interleaved", 16, BF, True, "heads", False),
    ([0, 0, 0], [5, 0, 64], 4, 2, 64, 64, "half", 32, BF, False, "heads", False),
    # a page of one request with more rows than the others' average: its rows are made twice
    ([1] * 20 + [70] + [2] * 9, list(range(40, 70)), 4, 3, 128, 128, "half", 64, BF, True, "heads", False),
    ([150] + [1] * 40, [7] + [3] * 40, 2, 2, 64, 32, "interleaved", 128, HF, False, "tokens", True),
]


@pytest.mark.parametrize("case", APPENDS, ids=range(len(APPENDS)))
def test_append(cuda, case):
    from mlx_dspark_b200 import rope

    counts, before, Hq, Hk, D, rot, layout, page, dt, norm, pool, own_pos = case
    rng, g = random.Random(len(counts) + D), torch.Generator().manual_seed(page + D)
    R, B, pad = sum(counts), len(counts), 3  # three rows of nobody behind the last request's
    need = [-(-(n + x) // page) for n, x in zip(counts, before)]
    n_pages = sum(need) + 5
    cache = _pool(cuda, n_pages, Hk, page, D, g, pool)
    rows = _tables(need, n_pages, rng, max(need) + 1)
    table = rope.RopeTable(D, rot, theta=1e4, layout=layout, device=cuda)
    qkv = torch.randn(R + pad, (Hq + 2 * Hk) * D, generator=g).to(dt)
    wq, wk = ((1 + 0.2 * torch.randn(D, generator=g)).to(dt) if norm else None for _ in range(2))
    dev = qkv.to(cuda)
    q = dev[:, : Hq * D].view(-1, Hq, D)
    k = dev[:, Hq * D : (Hq + Hk) * D].view(-1, Hk, D)
    v = dev[:, (Hq + Hk) * D :].view(-1, Hk, D)
    pos = [x + i for n, x in zip(counts, before) for i in range(n)]
    if own_pos:
        pos = [rng.randint(0, 100000) for _ in pos]
    row_pos = _i32(pos + [0] * pad, cuda) if own_pos else None
    old = _cpu(cache)
    out = torch.full((R + pad, Hq, D), 7.0, dtype=dt, device=cuda)
    got, lens = cache.append(q, k, v, table, _cu(counts, cuda), _i32(before, cuda), _i32(rows, cuda), row_pos=row_pos,
                             q_norm=None if wq is None else wq.to(cuda), k_norm=None if wk is None else wk.to(cuda),
                             eps=1e-5, q_out=out)
    assert got is out and lens.tolist() == [n + x for n, x in zip(counts, before)]
    assert bool((out[R:] == 7.0).all())
    p = torch.tensor(pos, dtype=torch.int64)

    def turned(x, w):
        x = x.double()
        y = ref_norm(x, w)
        z = tree_reference.rope(x, table.inv_freq, table.mscale, p, rot, layout, None if w is None else w.double(), 1e-5)
        half = rot // 2
        size = y.abs().clone()  # |a| + |b| of each pair, the value itself where nothing turns
        i0 = slice(0, half) if layout == "half" else slice(0, rot, 2)
        i1 = slice(half, rot) if layout == "half" else slice(1, rot, 2)
        both = y[..., i0].abs() + y[..., i1].abs()
        size[..., i0], size[..., i1] = both, both
        return z, size * 2.0 ** -20

    def ref_norm(x, w):
        return x if w is None else x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-5) * w.double()

    qv, kv, vv = (t[:R].double().cpu() for t in (q, k, v))
    zq, dq = turned(qv, wq)
    assert bool(((out[:R].double().cpu() - zq).abs() <= _half_step(dt, zq) + dq * 1.01).all())
    zk, dk = turned(kv, wk)
    new = _cpu(cache)
    for x, spread, before_, after, s_before, s_after in ((zk, dk, old[0], new[0], old[2], new[2]),
                                                         (vv, torch.zeros_like(vv), old[1], new[1], old[3], new[3])):
        lo, hi = before_.double(), before_.double()
        s_lo, s_hi = s_before.double(), s_before.double()
        r0, touched = 0, torch.zeros(before_.shape[:3], dtype=torch.bool)
        for b, n in enumerate(counts):
            l1, h1, sl, sh = ref.append(before_, s_before, rows[b], before[b], x[r0 : r0 + n], spread[r0 : r0 + n])
            for first in {(before[b] + i) // page for i in range(n)}:
                pid, end = rows[b][first], min(page, before[b] + n - first * page)
                lo[pid, :, :end], hi[pid, :, :end] = l1[pid, :, :end], h1[pid, :, :end]
                s_lo[pid], s_hi[pid] = sl[pid], sh[pid]
                touched[pid, :, :end] = True
            r0 += n
        c = after.double()
        nan = c.isnan()
        assert torch.equal(nan & touched[..., None], lo.isnan() & touched[..., None])
        fine = touched[..., None] & ~nan
        assert bool(((c >= lo) & (c <= hi))[fine.expand_as(c)].all())
        assert bool(((s_after >= s_lo) & (s_after <= s_hi)).all())
        keep = ~touched
        assert torch.equal(after.view(torch.uint8)[keep], before_.view(torch.uint8)[keep])  # nothing else is written


@pytest.mark.parametrize("off", [0, 1, 2, 4])
def test_append_of_rows_at_any_alignment(cuda, off):
    """q, k, v and q_out as slices that begin and step off the 16-byte boundaries; q rotated in place."""
    from mlx_dspark_b200 import rope

    g, Hq, Hk, D, page, R = torch.Generator().manual_seed(off), 3, 2, 64, 16, 21
    table = rope.RopeTable(D, 32, theta=1e4, device=cuda)
    x = torch.randn(R, (Hq + 2 * Hk) * D + 8, generator=g).to(BF).to(cuda)
    cut = [x[:, off + a * D : off + b * D].unflatten(1, (-1, D)) for a, b in ((0, 3), (3, 5), (5, 7))]
    plain = [t.contiguous() for t in cut]
    got = []
    for q, k, v in (cut, plain):
        cache = _pool(cuda, 4, Hk, page, D, torch.Generator().manual_seed(1))
        out, _ = cache.append(q, k, v, table, _cu([R], cuda), _i32([9], cuda), _i32([[3, 0]], cuda), q_out=q)
        assert out is q
        got.append((out.clone(), cache))
    assert torch.equal(got[0][0], got[1][0])
    assert _same_codes(got[0][1].k, got[1][1].k) and _same_codes(got[0][1].v, got[1][1].v)
    assert torch.equal(got[0][1].k_scale, got[1][1].k_scale)


def _identity(cuda, D):
    """A rotation by nothing: positions 0."""
    from mlx_dspark_b200 import rope
    return rope.RopeTable(D, 16, theta=1e4, device=cuda)


def _append_values(cuda, cache, table, kv_len, x, y, rope_table):
    """k = x, v = y (both [n, H, D]) of one request at position 0."""
    n = x.shape[0]
    zero = torch.zeros(n, dtype=torch.int32, device=cuda)
    q = torch.zeros(n, cache.heads, cache.head_dim, dtype=x.dtype, device=cuda)
    return cache.append(q, x.to(cuda), y.to(cuda), rope_table, _cu([n], cuda), _i32([kv_len], cuda), table, row_pos=zero)


@pytest.mark.parametrize("page,D", [(16, 64), (64, 128), (128, 128)])
def test_append_scales_over_rounds(cuda, page, D):
    """A page's scale starts with its first tokens, rises with larger ones (its codes are rounded to it), stays when
    smaller ones come and when tokens are taken back, and starts anew with a page begun anew."""
    from mlx_dspark_b200 import paged

    H, g = 2, torch.Generator().manual_seed(D + page)
    cache = paged.PagedCache.empty(4, H, page, D, cuda)
    table, none = _i32([[2, 0]], cuda), _identity(cuda, D)
    sizes = [1.0, 0.01, 50.0, 1e-3, 3000.0, 1.0]
    want = _cpu(cache)
    kv_len = 0
    for step, size in enumerate(sizes + [0.5]):
        if step == len(sizes):
            kv_len = 0  # taken back altogether: the page begins anew, with a smaller scale
        x, y = (size * torch.randn(2, H, D, generator=g).to(BF) for _ in range(2))
        _append_values(cuda, cache, table, kv_len, x, y, none)
        now = _cpu(cache)
        for z, i in ((x, 0), (y, 1)):
            lo, hi, s_lo, s_hi = ref.append(want[i], want[i + 2], [2, 0], kv_len, z.double(), torch.zeros(2, H, D))
            assert torch.equal(lo, hi) and torch.equal(now[i + 2].double(), s_lo) and torch.equal(s_lo, s_hi)
            assert torch.equal(now[i].double(), lo)
        if step == 4:
            assert bool((now[3][2] == 64.0).all() | (now[3][2] == 32.0).all() | (now[3][2] > 8).all())
        want = now
        kv_len += 2 if step != 3 else 1  # one token is taken back on the way
    assert bool((want[3][2] <= 2.0 ** -6).all())


@pytest.mark.parametrize("dt", [BF, HF])
def test_append_special_values(cuda, dt):
    from mlx_dspark_b200 import paged

    H, D, page = 1, 64, 16
    cache = paged.PagedCache.empty(3, H, page, D, cuda)
    x = torch.zeros(4, H, D, dtype=dt)
    x[0, 0, 20] = math.inf
    x[1, 0, 21] = -math.inf
    x[2, 0, 22] = math.nan
    x[3, 0, 23] = 3.0  # the largest finite value: scale 2^-7
    _append_values(cuda, cache, _i32([[1]], cuda), 0, x, x, _identity(cuda, D))
    for codes, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        assert scale[1].tolist() == [2.0 ** -7]
        got = codes[1, 0, :4].cpu().double()
        assert got[0, 20] == 448 and got[1, 21] == -448 and math.isnan(got[2, 22]) and got[3, 23] == 384
        got[2, 22] = 0
        assert float(got.abs().sum()) == 448 + 448 + 384
    # zeros alone have the smallest scale
    _append_values(cuda, cache, _i32([[2]], cuda), 0, torch.zeros(1, H, D, dtype=dt), torch.zeros(1, H, D, dtype=dt),
                   _identity(cuda, D))
    assert cache.v_scale[2].item() == 2.0 ** -64 and bool((cache.v[2, 0, 0].double() == 0).all())
    if dt is BF:  # beyond the largest scale values saturate
        big = torch.full((1, H, D), 1e38, dtype=dt)
        _append_values(cuda, cache, _i32([[0]], cuda), 0, big, big, _identity(cuda, D))
        assert cache.v_scale[0].item() == 2.0 ** 64 and bool((cache.v[0, 0, 0].double() == 448).all())
    # a scale that is none (NaN, negative, zero) gives way to the new tokens'
    for bad in (math.nan, -1.0, 0.0):
        cache.v_scale[1] = bad
        _append_values(cuda, cache, _i32([[1]], cuda), 4, x[3:], x[3:], _identity(cuda, D))
        assert cache.v_scale[1].item() == 2.0 ** -7 and cache.v[1, 0, 4, 23].double() == 384


def test_append_rows_without_a_page_are_dropped(cuda):
    """Page ids outside the pool and tokens past the table: dropped and recorded, everybody else served."""
    from mlx_dspark_b200 import _lib

    g = torch.Generator().manual_seed(3)
    cache = _pool(cuda, 4, 1, 16, 64, g)
    old = _cpu(cache)
    x = torch.randn(24, 1, 64, generator=g).to(BF).to(cuda)
    dev = cuda.index
    assert _lib.device_status(dev) == 0
    counts, before = [8, 8, 8], [10, 28, 0]
    table = _i32([[0, -1], [1, 2], [99, 3]], cuda)  # second page absent; past the table's 32; no page 99
    q, lens = cache.append(x, x, x, _identity(cuda, 64), _cu(counts, cuda), _i32(before, cuda), table)
    assert _lib.device_status(dev) != 0 and _lib.device_status(dev) == 0
    assert lens.tolist() == [18, 32, 8]
    new = _cpu(cache)
    changed = (new[1].view(torch.uint8) != old[1].view(torch.uint8)).any(-1)[:, 0]
    assert not bool(changed[3].any())
    # page 0: tokens 10 to 15 are new, those before rounded to the new scale perhaps; page 2: tokens 12 to 15
    assert not bool(changed[1].any()) and not bool(changed[2, :12].any() and new[3][2, 0] == old[3][2, 0])
    y = x[:6, 0].double().cpu()
    s = float(new[3][0, 0])
    assert torch.equal(new[1][0, 0, 10:16].double(), ref.nearest(y / s))
    assert torch.equal(new[1][2, 0, 12:16].double(), ref.nearest(x[8:12, 0].double().cpu() / float(new[3][2, 0])))


# ------------------------------------------------------------------------------- attention

def _bound(q, k, absum, vsum, n, scale, dt, want):
    D = q.shape[-1]
    S = float((q.abs().amax((0, 1)) * k.abs().amax((0, 1))).sum()) * abs(scale)
    eps = 2 * (math.log(2) * 2.0 ** -21 * 2 * S / math.log(2) + S * (D + 8) * 2.0 ** -23 + 2.0 ** -22)
    return (_half_step(dt, want) + (2.0 ** -11 + 2 * eps + n * 2.0 ** -23) * absum * 1.01 +
            2.0 ** -36 * vsum + 1e-30)


def _check(cuda, cache, q, counts, lens, rows, causal, scale, out=None):
    """Attention of the packed rows against 64 bits, request by request. Returns the output."""
    kc, vc, ks, vs = _cpu(cache)
    cu = _cu(counts, cuda)
    got = cache.attention(q, cu, _i32(lens, cuda), _i32(rows, cuda), scale=scale, causal=causal, out=out)
    host, r0 = got.double().cpu(), 0
    for b, n in enumerate(counts):
        L = max(0, min(lens[b], len(rows[b]) * cache.page_size))
        qd = q[r0 : r0 + n].double().cpu()
        k, v = (ref.values(c, s, rows[b], L) for c, s in ((kc, ks), (vc, vs)))
        i, j = torch.arange(n)[:, None], torch.arange(L)[None]
        seen = (j <= lens[b] - n + i) if causal else torch.ones(n, L, dtype=torch.bool)
        want, absum, vsum = tree_reference.attention(qd, k, v, seen, scale)
        if n:
            far = (host[r0 : r0 + n] - want).abs()
            lim = _bound(qd, k, absum, vsum, L, scale, q.dtype, want) if L else torch.zeros_like(far)
            # a result of 65520 or more is fp16's infinity: 65504 is its largest value, 32 its step there
            over = (host[r0 : r0 + n] == want.sign() * math.inf) & (want.abs() + lim >= 65520) & (q.dtype is HF)
            assert bool(((far <= lim) | over).all()), (b, float((far / lim.clamp(min=1e-30)).max()))
        r0 += n
    return got


def _finite_pool(cuda, pages, H, page, D, g, layout="heads", span=2):
    """A cache of ordinary codes, scales 2^-span to 2^span about 2^-6."""
    from mlx_dspark_b200 import paged

    shape = (pages, H, page, D) if layout == "heads" else (pages, page, H, D)
    made = []
    for _ in range(2):
        x = (64 * torch.randn(shape, generator=g)).clamp(-448, 448).to(E4M3).view(torch.uint8).to(cuda).view(E4M3)
        made.append(x if layout == "heads" else x.permute(0, 2, 1, 3))
    sc = [torch.exp2(torch.randint(-6 - span, -5 + span, (pages, H), generator=g).float()).to(cuda) for _ in range(2)]
    return paged.PagedCache(made[0], made[1], *sc)


ATTNS = [
    # counts, lens, Hq, Hk, D, page, type, causal, pool layout
    ([1], [1], 4, 1, 128, 64, BF, True, "heads"),
    ([1, 1, 1, 1], [15, 16, 17, 129], 8, 2, 64, 16, HF, True, "heads"),
    ([1, 0, 2, 0], [257, 40, 2, 0], 7, 1, 128, 32, BF, True, "tokens"),
    ([5, 16, 3], [5, 700, 33], 8, 2, 128, 16, BF, True, "heads"),
    ([5, 16, 3], [5, 700, 33], 8, 2, 128, 16, HF, False, "tokens"),
    ([70, 1], [513, 96], 6, 3, 64, 128, BF, True, "heads"),
    ([33], [33], 32, 8, 128, 64, HF, True, "heads"),
    ([9, 9], [1500, 31], 16, 1, 128, 64, BF, False, "heads"),
    ([1] * 150, [1 + 7 * i % 90 for i in range(150)], 4, 2, 64, 32, BF, True, "heads"),
]


@pytest.mark.parametrize("case", ATTNS, ids=range(len(ATTNS)))
def test_attention(cuda, case):
    counts, lens, Hq, Hk, D, page, dt, causal, layout = case
    rng, g = random.Random(D + page), torch.Generator().manual_seed(len(counts) + page)
    need = [-(-x // page) for x in lens]
    cache = _finite_pool(cuda, sum(need) + 4, Hk, page, D, g, layout)
    rows = _tables(need, sum(need) + 4, rng, max(need) + 1)
    q = torch.randn(sum(counts) + 2, Hq + 1, D, generator=g).to(dt).to(cuda)[:, :Hq]  # rows with room between
    out = torch.full(q.shape, 5.0, dtype=dt, device=cuda)
    _check(cuda, cache, q, counts, lens, rows, causal, D ** -0.5, out)
    assert bool((out[sum(counts):] == 5.0).all())  # rows of nobody


def _with_room(rows, page, tokens):
    """The tables widened to so many tokens: small calls go to clusters of 8 blocks a row block, with room for 6000 tokens of
    16 where there are few of them, with room for 40,000 tokens as shares of a line over the whole grid."""
    width = max(-(-tokens // page), len(rows[0]))
    return [r + [-1] * (width - len(r)) for r in rows]


FORMS = [
    # counts, lens, Hq, Hk, D, page, type, causal, pool layout
    ([1], [5000], 4, 1, 128, 64, BF, True, "heads"),
    ([2, 0, 1], [1030, 9, 3001], 8, 2, 64, 16, HF, True, "tokens"),
    ([7], [4099], 8, 2, 128, 128, HF, True, "heads"),                # 28 rows of a product
    ([16, 5, 1], [31, 2049, 700], 4, 2, 64, 32, BF, False, "heads"),
    ([1] * 33, [1 + 97 * i % 900 for i in range(33)], 4, 1, 64, 16, BF, True, "heads"),  # more requests than a warp has lanes
    ([20], [3], 4, 4, 128, 64, BF, True, "heads"),                   # more rows than keys
]


@pytest.mark.parametrize("tokens", [0, 6000, 40000])
@pytest.mark.parametrize("case", FORMS, ids=range(len(FORMS)))
def test_attention_few_rows_forms(cuda, case, tokens):
    counts, lens, Hq, Hk, D, page, dt, causal, layout = case
    rng, g = random.Random(D + page), torch.Generator().manual_seed(len(counts) + page + 2)
    need = [-(-x // page) for x in lens]
    cache = _finite_pool(cuda, sum(need) + 4, Hk, page, D, g, layout)
    rows = _with_room(_tables(need, sum(need) + 4, rng, max(need) + 1), page, tokens)
    q = torch.randn(sum(counts) + 2, Hq + 1, D, generator=g).to(dt).to(cuda)[:, :Hq]
    out = torch.full(q.shape, 5.0, dtype=dt, device=cuda)
    _check(cuda, cache, q, counts, lens, rows, causal, D ** -0.5, out)
    assert bool((out[sum(counts):] == 5.0).all())
    again = cache.attention(q, _cu(counts, cuda), _i32(lens, cuda), _i32(rows, cuda), scale=D ** -0.5, causal=causal)
    assert torch.equal(again[: sum(counts)], out[: sum(counts)])


@pytest.mark.parametrize("tokens", [0, 6000, 40000])
@pytest.mark.parametrize("n", [3, 12])
def test_attention_few_rows_hidden_values(cuda, n, tokens):
    """A NaN code reaches the rows that see its key and no others; infinite q makes its own head NaN; a page without a
    positive scale is not seen."""
    g = torch.Generator().manual_seed(n)
    L, D, page = 2000, 64, 16
    cache = _finite_pool(cuda, 125, 2, page, D, g)
    table = _i32(_with_room([list(range(125))], page, tokens), cuda)
    q = torch.randn(n, 4, D, generator=g).to(BF).to(cuda)
    args = _cu([n], cuda), _i32([L], cuda), table
    clean = cache.attention(q, *args, scale=0.1)
    own = L - 2  # the last row but one's token
    for t in (cache.v, cache.k):
        at = t.view(torch.uint8)[own // page, 0, own % page]
        old = at.clone()
        at[10] = 0x7F
        out = cache.attention(q, *args, scale=0.1)
        assert torch.equal(out[: n - 2], clean[: n - 2]) and torch.equal(out[:, 2:], clean[:, 2:])
        bad = out[n - 2 :, :2].isnan()
        assert bool(bad[..., 10].all()) and bool(bad.all()) == (t is cache.k)
        at.copy_(old)
    x = q.clone()
    x[1, 2, 5] = math.inf
    out = cache.attention(x, *args, scale=0.1)
    assert bool(out[1, 2].isnan().all()) and torch.equal(out[2:], clean[2:]) and torch.equal(out[1, :2], clean[1, :2])
    cache.k_scale[3] = 0.0
    cache.v_scale[7] = -1.0
    seen = cache.attention(q, *args, scale=0.1)
    gone = [x for x in range(125) if x not in (3, 7)]  # the same keys without them
    want = cache.attention(q, args[0], _i32([L - 2 * page], cuda), _i32(_with_room([gone], page, tokens), cuda), scale=0.1)
    # weights rounded in another grouping: two fp16 roundings (2^-11 each) of sums whose values are at most vmax, and bf16's
    # own half steps (2^-8) of either result
    vmax = 448 * float(cache.v_scale.abs().max())
    assert float((seen - want).abs().max()) <= (2 * 2.0 ** -11 + 2 * 2.0 ** -8) * vmax


def _far(rows, page):
    """The tables widened to 200,000 tokens: with that much room, calls of more than 32 rows a request and kv head on
    average go to the kernel for many rows (the narrow tables of small tests do not)."""
    width = 200000 // page
    return [r + [-1] * (width - len(r)) for r in rows]


MANY = [
    # counts, lens, Hq, Hk, D, page, type, causal, pool layout
    ([17], [17], 4, 1, 128, 64, BF, True, "heads"),              # one slot's rows, one tile
    ([40, 3, 0, 90], [40, 700, 9, 333], 8, 2, 128, 16, HF, True, "heads"),
    ([40, 3, 0, 90], [40, 700, 9, 333], 8, 2, 128, 16, BF, False, "tokens"),
    ([65, 1], [1300, 96], 8, 2, 64, 32, BF, True, "heads"),      # 260 rows: two blocks of rows, the last of four
    ([64], [257], 8, 2, 64, 128, HF, False, "heads"),            # 256 rows: both slots full
    ([33, 33, 33], [128, 129, 640], 7, 1, 128, 128, BF, True, "tokens"),
    ([200], [200], 4, 2, 128, 64, HF, True, "heads"),            # a prompt of its own keys alone
    ([45] * 20, [45 + 61 * i % 500 for i in range(20)], 4, 4, 64, 64, BF, True, "heads"),
]


@pytest.mark.parametrize("case", MANY, ids=range(len(MANY)))
def test_attention_many_rows(cuda, case):
    counts, lens, Hq, Hk, D, page, dt, causal, layout = case
    rng, g = random.Random(D + page), torch.Generator().manual_seed(len(counts) + page + 1)
    need = [-(-x // page) for x in lens]
    cache = _finite_pool(cuda, sum(need) + 4, Hk, page, D, g, layout)
    rows = _far(_tables(need, sum(need) + 4, rng, max(need) + 1), page)
    q = torch.randn(sum(counts) + 2, Hq + 1, D, generator=g).to(dt).to(cuda)[:, :Hq]
    out = torch.full(q.shape, 5.0, dtype=dt, device=cuda)
    _check(cuda, cache, q, counts, lens, rows, causal, D ** -0.5, out)
    assert bool((out[sum(counts):] == 5.0).all())
    again = cache.attention(q, _cu(counts, cuda), _i32(lens, cuda), _i32(rows, cuda), scale=D ** -0.5, causal=causal)
    assert torch.equal(again[: sum(counts)], out[: sum(counts)])  # no order of blocks shows


@pytest.mark.parametrize("n", [20, 80])  # 40 rows: the slots share them; 160: a slot each
def test_attention_many_rows_edges(cuda, n):
    """What the tests below hold a few rows to: scales of the scores, scales far apart, q of any size, NaN in hidden
    places, pages that are not there, rows that see nothing."""
    from mlx_dspark_b200 import _lib

    g, dev = torch.Generator().manual_seed(n), cuda.index
    cache = _finite_pool(cuda, 40, 1, 16, 64, g, span=0)
    base = torch.randn(n, 2, 64, generator=g)
    q, cu = base.to(BF).to(cuda), _cu([n], cuda)
    rows = _far([list(range(30))], 16)
    for scale in (0.0, -0.2, 3.0):
        _check(cuda, cache, q, [n], [470], rows, True, scale)
    sizes = torch.tensor([1e-38, 1e-20, 1.0, 1e3, 1e-3, 0.0] * n)[:n, None, None]
    _check(cuda, cache, (base * sizes).to(BF).to(cuda), [n], [470], rows, True, 0.125)
    table, ln = _i32(rows, cuda), _i32([470], cuda)
    bad = q.clone()
    bad[1, 0, 5], bad[n - 1, 1, 9] = math.inf, math.nan
    out, fine = (cache.attention(x, cu, ln, table, scale=0.125) for x in (bad, q))
    want = torch.zeros(n, 2, dtype=torch.bool)
    want[1, 0] = want[n - 1, 1] = True
    assert torch.equal(out.isnan().any(-1).cpu(), want) and torch.equal(out[~want.to(cuda)], fine[~want.to(cuda)])
    # NaN codes: behind the last key, and in keys of the rows' own
    clean = fine
    for t in (cache.k, cache.v):
        t.view(torch.uint8)[29, 0, 6:] = 0x7F
    assert torch.equal(cache.attention(q, cu, ln, table, scale=0.125), clean)
    own = 470 - n + 7  # the eighth row's own token
    for t in (cache.v, cache.k):
        old = t[own // 16, 0, own % 16].view(torch.uint8).clone()
        t.view(torch.uint8)[own // 16, 0, own % 16, 10] = 0xFF
        out = cache.attention(q, cu, ln, table, scale=0.125)
        assert torch.equal(out[:7], clean[:7])
        nan = out[7:].isnan()
        if t is cache.v:
            assert bool(nan[..., 10].all()) and int(nan.sum()) == (n - 7) * 2
        else:
            assert bool(nan.all())
        t.view(torch.uint8)[own // 16, 0, own % 16] = old
    # a key of everybody's
    t = cache.v.view(torch.uint8)
    old = t[3, 0, 4].clone()
    t[3, 0, 4, 11] = 0x7F
    nan = cache.attention(q, cu, ln, table, scale=0.125).isnan()
    assert bool(nan[..., 11].all()) and int(nan.sum()) == n * 2
    t[3, 0, 4] = old
    # pages outside the pool and without a positive scale: as if they were not in the table
    short = cache.attention(q, cu, _i32([464], cuda), _i32(_far([list(range(5)) + list(range(6, 30))], 16), cuda), scale=0.2,
                            causal=False)
    assert _lib.device_status(dev) == 0
    for page in (-7, 40, 2 ** 31 - 1):
        r = list(range(30))
        r[5] = page
        out = cache.attention(q, cu, _i32([480], cuda), _i32(_far([r], 16), cuda), scale=0.2, causal=False)
        assert _lib.device_status(dev) != 0 and _lib.device_status(dev) == 0
        # (page 29's last ten tokens hold NaN codes: 480 keys see them)
        assert bool(out.isnan().all())
    for t in (cache.k, cache.v):
        t.view(torch.uint8)[29, 0, 6:] = 0x30
    short = cache.attention(q, cu, _i32([464], cuda), _i32(_far([list(range(5)) + list(range(6, 30))], 16), cuda), scale=0.2,
                            causal=False)
    for page in (-7, 40):
        r = list(range(30))
        r[5] = page
        out = cache.attention(q, cu, _i32([480], cuda), _i32(_far([r], 16), cuda), scale=0.2, causal=False)
        assert torch.allclose(out.float(), short.float(), rtol=2e-2, atol=2e-2) and _lib.device_status(dev) != 0
    for s in (0.0, -1.0, math.nan):
        keep = cache.k_scale[5].clone()
        cache.k_scale[5] = s
        out = cache.attention(q, cu, _i32([480], cuda), table, scale=0.2, causal=False)
        assert torch.allclose(out.float(), short.float(), rtol=2e-2, atol=2e-2)
        cache.k_scale[5] = keep
    # rows that see nothing
    out = cache.attention(q, cu, _i32([n - 9], cuda), table, scale=0.2)
    assert bool((out[:9] == 0).all()) and bool((out[9:] != 0).any(-1).all())
    assert bool((cache.attention(q, cu, _i32([0], cuda), table, scale=0.2) == 0).all())
    none = cache.attention(q, cu, _i32([64], cuda), _i32(_far([[-1] * 4], 16), cuda), scale=0.2)
    assert bool((none == 0).all()) and _lib.device_status(dev) != 0
    # scales 2^80 apart, the largest weights where the values are smallest
    cache.v_scale[:8].copy_(torch.exp2(torch.tensor([[-40.0], [30.0], [0.0], [-40.0], [10.0], [-20.0], [0.0], [-60.0]])))
    for r in ([0, 3, 7, 5], [2, 6, 9], [0, 1, 2], [7]):
        _check(cuda, cache, q, [n], [16 * len(r) - 2], _far([r], 16), False, 0.125)


@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
def test_attention_scales_of_the_scores(cuda, scale):
    g = torch.Generator().manual_seed(9)
    cache = _finite_pool(cuda, 12, 2, 32, 64, g, span=0)
    q = torch.randn(4, 4, 64, generator=g).to(BF).to(cuda)
    _check(cuda, cache, q, [4], [300], [list(range(12))], True, scale)


def test_attention_scales_far_apart(cuda):
    """Pages whose scales differ by 2^80, the largest weights where the values are smallest."""
    g = torch.Generator().manual_seed(10)
    cache = _finite_pool(cuda, 8, 1, 16, 64, g, span=0)
    cache.v_scale.copy_(torch.exp2(torch.tensor([[-40.0], [40.0], [0.0], [-40.0], [10.0], [-20.0], [0.0], [-64.0]])))
    q = torch.randn(3, 2, 64, generator=g).to(HF).to(cuda)
    for rows in ([0, 3, 7, 5], [2, 6], [0, 1, 2], [7]):
        _check(cuda, cache, q, [3], [16 * len(rows) - 2], [rows], True, 0.125)


def test_attention_q_of_any_size(cuda):
    """bf16 rows from the smallest to nearly the largest values, fp16 subnormals; rows with an infinity or NaN are NaN."""
    g = torch.Generator().manual_seed(11)
    cache = _finite_pool(cuda, 8, 1, 16, 64, g, span=0)
    rows, base = [list(range(8))], torch.randn(6, 1, 64, generator=g)
    q = (base * torch.tensor([1e-38, 1e-20, 1.0, 1e3, 1e-3, 0.0])[:, None, None]).to(BF).to(cuda)
    _check(cuda, cache, q, [6], [120], rows, True, 0.125)
    h = (base * torch.tensor([1e-6, 1e-4, 1.0, 8.0, 1e-2, 0.0])[:, None, None]).to(HF).to(cuda)
    _check(cuda, cache, h, [6], [120], rows, True, 0.125)
    for t in (q, h):
        bad = t.clone()
        bad[1, 0, 5], bad[3, 0, 9] = math.inf, math.nan
        out = cache.attention(bad, _cu([6], cuda), _i32([120], cuda), _i32(rows, cuda), scale=0.125)
        assert out.isnan().any(-1)[:, 0].tolist() == [False, True, False, True, False, False]
        fine = cache.attention(t, _cu([6], cuda), _i32([120], cuda), _i32(rows, cuda), scale=0.125)
        assert torch.equal(out[[0, 2, 4, 5]], fine[[0, 2, 4, 5]])


def test_attention_of_rows_that_see_nothing(cuda):
    """Fewer keys than rows, no keys, a negative length: zeros."""
    g = torch.Generator().manual_seed(12)
    cache = _finite_pool(cuda, 6, 2, 16, 128, g)
    q = torch.randn(13, 4, 128, generator=g).to(BF).to(cuda)
    counts, lens = [5, 4, 4], [2, 0, -3]
    out = _check(cuda, cache, q, counts, lens, [[0], [1], [2]], True, 0.1)
    assert bool((out[:3] == 0).all()) and bool((out[3:5] != 0).any()) and bool((out[5:] == 0).all())
    out = cache.attention(q, _cu(counts, cuda), _i32(lens, cuda), _i32([[0], [1], [2]], cuda), scale=0.1, causal=False)
    assert bool((out[:5] != 0).any(-1).all()) and bool((out[5:] == 0).all())


def test_attention_hidden_values_take_no_part(cuda):
    """NaN codes behind the last key and in keys that a row does not see; a row that sees one is NaN."""
    g = torch.Generator().manual_seed(13)
    cache = _finite_pool(cuda, 8, 1, 16, 64, g)
    rows, n, L = [[0, 1, 2, 3, 4]], 6, 70
    q = torch.randn(n, 2, 64, generator=g).to(BF).to(cuda)
    clean = cache.attention(q, _cu([n], cuda), _i32([L], cuda), _i32(rows, cuda), scale=0.1)
    for t in (cache.k, cache.v):
        t.view(torch.uint8)[4, 0, L - 64 :] = 0x7F  # token L and later
        t.view(torch.uint8)[5:] = 0xFF
    assert torch.equal(cache.attention(q, _cu([n], cuda), _i32([L], cuda), _i32(rows, cuda), scale=0.1), clean)
    own = L - n + 3  # the fourth row's own token
    for t in (cache.v, cache.k):
        old = t[own // 16, 0, own % 16].view(torch.uint8).clone()
        t.view(torch.uint8)[own // 16, 0, own % 16, 10] = 0xFF
        out = cache.attention(q, _cu([n], cuda), _i32([L], cuda), _i32(rows, cuda), scale=0.1)
        assert torch.equal(out[:3], clean[:3])
        bad = out[3:].isnan()
        if t is cache.v:
            assert bool(bad[..., 10].all()) and int(bad.sum()) == 3 * 2
            same = torch.ones(64, dtype=torch.bool)
            same[10] = False
            assert torch.equal(out[3:, :, same.to(cuda)], clean[3:, :, same.to(cuda)])
        else:
            assert bool(bad.all())
        t.view(torch.uint8)[own // 16, 0, own % 16] = old


def test_attention_pages_that_are_not_there(cuda):
    """Page ids outside the pool are recorded and not seen, nor are pages whose scale is not positive, nor keys past
    the table."""
    from mlx_dspark_b200 import _lib

    g = torch.Generator().manual_seed(14)
    cache = _finite_pool(cuda, 6, 2, 32, 64, g)
    q = torch.randn(2, 4, 64, generator=g).to(HF).to(cuda)
    cu, dev = _cu([2], cuda), cuda.index
    without = cache.attention(q, cu, _i32([96], cuda), _i32([[0, 2, 3]], cuda), scale=0.2, causal=False)
    assert _lib.device_status(dev) == 0
    for bad in (-1, 6, 2 ** 31 - 1, -2 ** 31):
        out = cache.attention(q, cu, _i32([128], cuda), _i32([[0, bad, 2, 3]], cuda), scale=0.2, causal=False)
        assert _lib.device_status(dev) != 0 and _lib.device_status(dev) == 0
        assert torch.allclose(out.float(), without.float(), rtol=2e-3, atol=2e-3)
    for bad in (0.0, -1.0, math.nan):
        keep = cache.v_scale[1].clone()
        cache.v_scale[1] = bad
        out = cache.attention(q, cu, _i32([128], cuda), _i32([[0, 1, 2, 3]], cuda), scale=0.2, causal=False)
        assert torch.allclose(out.float(), without.float(), rtol=2e-3, atol=2e-3)
        cache.v_scale[1] = keep
    a = cache.attention(q, cu, _i32([400], cuda), _i32([[0, 2, 3]], cuda), scale=0.2, causal=False)
    assert torch.equal(a, without) and _lib.device_status(dev) == 0
    none = cache.attention(q, cu, _i32([64], cuda), _i32([[-1, -1]], cuda), scale=0.2)
    assert bool((none == 0).all()) and _lib.device_status(dev) != 0


def test_attention_far_into_a_large_pool(cuda):
    """Pages past 2^31 bytes of the pool."""
    from mlx_dspark_b200 import paged

    g = torch.Generator().manual_seed(15)
    pages, H, page, D = 20000, 8, 128, 128  # 2.6 GB of keys
    cache = paged.PagedCache.empty(pages, H, page, D, cuda)
    rows = [[19999, 17001, 16384, 3]]
    for i in rows[0]:
        for t in (cache.k, cache.v):
            t.view(torch.uint8)[i] = (64 * torch.randn(H, page, D, generator=g)).clamp(-448, 448).to(E4M3).view(torch.uint8).to(cuda)
    cache.k_scale.fill_(2.0 ** -6)
    cache.v_scale.fill_(2.0 ** -6)
    small = paged.PagedCache(*(t.view(torch.uint8)[rows[0]].view(E4M3) for t in (cache.k, cache.v)),
                             *(t[rows[0]].contiguous() for t in (cache.k_scale, cache.v_scale)))
    q = torch.randn(3, 16, D, generator=g).to(BF).to(cuda)
    args = (_cu([3], cuda), _i32([500], cuda))
    far = cache.attention(q, *args, _i32(rows, cuda), scale=0.1)
    assert torch.equal(far, _check(cuda, small, q, [3], [500], [[0, 1, 2, 3]], True, 0.1))
    x = torch.randn(12, H, D, generator=g).to(BF).to(cuda)
    none = _identity(cuda, D)
    _append_values(cuda, cache, _i32(rows, cuda), 500, x, x, none)
    _append_values(cuda, small, _i32([[0, 1, 2, 3]], cuda), 500, x, x, none)
    assert _same_codes(cache.v[3], small.v[3]) and torch.equal(cache.v_scale[3], small.v_scale[3])


@pytest.mark.parametrize("rows", [1, 40])
def test_attention_long_context(cuda, rows):
    """One request cut over every block, 100,003 keys, against 64 bits on the GPU; twice the same bits."""
    from mlx_dspark_b200 import paged

    H, Hq, D, page, L = 2, 8, 128, 16, 100003
    n_pages = -(-L // page)
    g = torch.Generator(device=cuda).manual_seed(16)
    k, v = ((64 * torch.randn(n_pages, H, page, D, device=cuda, generator=g)).clamp(-448, 448).to(E4M3) for _ in range(2))
    sc = [torch.exp2(torch.randint(-7, -4, (n_pages, H), device=cuda, generator=g).float()) for _ in range(2)]
    cache = paged.PagedCache(k, v, *sc)
    t = torch.randperm(n_pages, device=cuda, generator=g).to(torch.int32)[None]
    q = torch.randn(rows, Hq, D, device=cuda, generator=g).to(HF)
    out = cache.attention(q, _cu([rows], cuda), _i32([L], cuda), t, scale=D ** -0.5)
    assert torch.equal(out, cache.attention(q, _cu([rows], cuda), _i32([L], cuda), t, scale=D ** -0.5))
    kd, vd = ((c.view(torch.uint8)[t[0].long()].view(E4M3).double() * s[t[0].long()].double()[..., None, None])
              .transpose(0, 1).reshape(H, -1, D)[:, :L] for c, s in ((k, sc[0]), (v, sc[1])))
    hidden = torch.ones(rows, L, dtype=torch.bool, device=cuda).tril(L - rows).logical_not()
    for h in range(Hq):
        z = (q[:, h].double() @ kd[h // 4].T * D ** -0.5).masked_fill(hidden, -math.inf)
        p = torch.softmax(z, -1)
        want, absum = p @ vd[h // 4], p @ vd[h // 4].abs()
        vsum = vd[h // 4].abs().sum(0)
        # rounded sums of L terms in many parts: 2^-24 for each addition of a chain of at most L / 32 / 4 + 600
        S = float((q[:, h].double().abs().amax(0) * kd[h // 4].abs().amax(0)).sum()) * D ** -0.5
        eps = 2 * (2.0 ** -20 * S + S * (D + 8) * 2.0 ** -23 + 2.0 ** -22)
        lim = (_half_step(HF, want) + (2.0 ** -11 + 2 * eps + (L / 128 + 600) * 2.0 ** -23) * absum * 1.01 + 2.0 ** -36 * vsum)
        assert bool(((out[:, h].double() - want).abs() <= lim).all())


# ------------------------------------------------------------------------------- scores

LOW = {BF: -2.0 ** 28, FP: -2.0 ** 28, HF: -65504.0}


def _check_scores(cuda, logits, tokens, temp, top, out=None):
    """Sums are fp32: a weight is off by 2^-22 + |log2 weight| 2^-23 (weights below 2^-40 do not matter: 2^-17 of them
    at most), a sum of V terms in strips by (V / 256 + 64) 2^-24; the logarithm by 2^-23 of it; -sum p ln p collects the
    weights' errors times their logarithms, at most 40."""
    from mlx_dspark_b200 import sampling

    R, V = logits.shape
    dev = logits.to(cuda) if not logits.is_cuda else logits
    got = sampling.token_logprobs(dev, _i32(tokens, cuda), temperature=None if temp is None else torch.tensor(temp, device=cuda),
                                  top=top, out=out)
    host = {k: v.cpu().tolist() for k, v in got.items()}
    cpu = logits.cpu()
    rel = 2.0 ** -17 * 2.0 ** -5 + (V / 256 + 64) * 2.0 ** -24 + 2.0 ** -20

    def near(a, b, extra=0.0):
        if math.isinf(b) or math.isinf(a):
            return a == b
        return abs(a - b) <= rel + 2.0 ** -22 * abs(b) + extra

    for r in range(R):
        if not 0 <= tokens[r] < V:
            assert (host["logprob"][r], host["entropy"][r], host["rank"][r]) == (0.0, 0.0, -1)
            if top:
                assert host["top_ids"][r] == [-1] * top and host["top_logprobs"][r] == [-math.inf] * top
            continue
        lp, ent, rank, ids, tl = ref.score(cpu[r], tokens[r], 1.0 if temp is None else temp[r], top, LOW[logits.dtype])
        assert host["rank"][r] == rank, r
        assert near(host["logprob"][r], lp), (r, host["logprob"][r], lp)
        assert near(host["entropy"][r], ent, 40 * rel), (r, host["entropy"][r], ent)
        if top:
            assert host["top_ids"][r] == ids, r
            assert all(near(a, b) for a, b in zip(host["top_logprobs"][r], tl)), r
    return got


@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("R,V,top", [(1, 1, 1), (3, 7, 5), (2, 33, 32), (1, 151936, 20), (5, 4097, 0), (9, 50257, 5),
                                     (700, 515, 32)])
def test_scores(cuda, dt, R, V, top):
    g = torch.Generator().manual_seed(R + V)
    logits = (4 * torch.randn(R, V, generator=g)).to(dt)
    tokens = torch.randint(0, V, (R,), generator=g).tolist()
    for r in range(0, R, 2):
        tokens[r] = int(logits[r].argmax())
    _check_scores(cuda, logits, tokens, None, top)
    temp = (0.3 + 2 * torch.rand(R, generator=g)).tolist()
    temp[R // 2] = 0.0
    _check_scores(cuda, logits, tokens, [float(torch.tensor(t)) for t in temp], top)


@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("shift", range(0, 9))
def test_scores_of_rows_at_any_alignment(cuda, dt, shift):
    """Rows that begin and end off the 16-byte boundaries, the largest values at their ends."""
    g = torch.Generator().manual_seed(shift)
    V, ld = 2051, 2100 + shift
    base = torch.randn(4 * ld + 16, generator=g).to(dt).to(cuda)
    x = base[shift : shift + 4 * ld].view(4, ld)[:, :V]
    x[0, 0], x[1, V - 1], x[2, 1], x[3, V - 2] = 9.0, 9.0, 9.0, 9.0
    x[:, 5 * shift + 3] = 8.0
    _check_scores(cuda, x, [0, V - 1, V - 1, 0], None, 4)


@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("V", [600, 70001])
def test_scores_of_masked_and_extreme_rows(cuda, dt, V):
    g = torch.Generator().manual_seed(V)
    x = torch.randn(12, V, generator=g).to(dt)
    low = torch.finfo(dt).min
    x[0] = -math.inf                      # nothing is left
    x[1] = low                            # the type's lowest value everywhere
    x[2] = math.nan
    x[3] = -math.inf
    x[3, [5, V - 1, 77]] = torch.tensor([1.0, 2.0, 2.0], dtype=dt)  # three are left
    x[4, ::2] = low
    x[4, 1::4] = math.nan
    x[5, 9] = math.inf                    # one takes all
    x[6, [9, 300]] = math.inf
    x[7] = 3.0                            # all equal: the lowest tokens, ln V
    x[8] = torch.linspace(-4, 4, V).to(dt)  # ascending
    x[9] = torch.linspace(4, -4, V).to(dt)
    x[10] = 60000.0 if dt is HF else 1e30
    x[10, 3] = 0.0
    x[11, : V // 2] = 6.0                 # half of them equal at the top
    tokens = [1, 2, 3, 77, 2, 9, 300, V - 1, 0, V - 1, 3, V // 2]
    _check_scores(cuda, x, tokens, None, 8)
    _check_scores(cuda, x, [5, 5, 5, 6, 3, 10, 9, 0, V - 1, 0, 0, 0], [0.5, 1.0, 2.0, 0.01, 100.0, 1e7, 1e-7] + [1.0] * 5, 32)


@pytest.mark.parametrize("V", [8192, 151937])
def test_scores_with_the_largest_values_in_one_strip(cuda, V):
    """All large values where one thread reads them, and every 256th vector equal: more candidates than fit the list."""
    x = torch.zeros(2, V, dtype=BF)
    x[0].view(-1)[: V // 8 * 8].view(-1, 8)[::256] = torch.linspace(1, 5, 8).to(BF)
    x[1, V // 3 :: 3] = 2.0
    _check_scores(cuda, x, [0, 1], None, 32)


def test_scores_of_padded_rows_and_out(cuda):
    from mlx_dspark_b200 import DSparkError, sampling

    g = torch.Generator().manual_seed(1)
    x = torch.randn(6, 999, generator=g).to(HF)
    first = _check_scores(cuda, x, [1, -1, 998, 999, 2 ** 31 - 1, -2 ** 31], None, 3)
    again = _check_scores(cuda, x + 1, [4, -1, -1, 5, 6, 7], None, 3, out=first)
    assert again is first
    y = x[:1].expand(4, 999)  # rows that share their memory
    _check_scores(cuda, y.to(cuda)[:1].expand(4, 999), [0, 1, 2, 3], None, 2)
    with pytest.raises(DSparkError):
        sampling.token_logprobs(x.to(cuda), _i32([0] * 6, cuda), top=2, out=first)
    with pytest.raises(DSparkError):
        sampling.token_logprobs(x.to(cuda), _i32([0] * 6, cuda), out=first)
    with pytest.raises(DSparkError):
        sampling.token_logprobs(x.to(cuda).T, _i32([0] * 999, cuda))
    with pytest.raises(DSparkError):
        sampling.token_logprobs(x.to(cuda), _i32([0] * 5, cuda))
    empty = sampling.token_logprobs(x.to(cuda)[:0], _i32([], cuda), top=2)
    assert empty["top_ids"].shape == (0, 2)


@pytest.mark.parametrize("n", [6, 500])
def test_attention_without_a_scale(cuda, n):
    """scale = 0: every visible key weighs the same, whatever q is (both kernels)."""
    g = torch.Generator().manual_seed(n)
    L, D = 4000, 64
    cache = _finite_pool(cuda, 125, 2, 32, D, g)
    q = (torch.randn(n, 8, D, generator=g) * 1e37).to(BF).to(cuda)
    rows = [list(range(125))]
    args = _cu([n], cuda), _i32([L], cuda), _i32(rows, cuda)
    out = cache.attention(q, *args, scale=0.0)
    assert torch.equal(out, cache.attention(torch.ones_like(q), *args, scale=0.0))
    _check(cuda, cache, torch.ones_like(q), [n], [L], rows, True, 0.0)


def test_append_of_no_rows(cuda):
    from mlx_dspark_b200 import rope

    cache = _pool(cuda, 3, 2, 16, 64, torch.Generator().manual_seed(0))
    q, k = (torch.empty(0, h, 64, dtype=BF, device=cuda) for h in (4, 2))
    keep = cache.k.clone(), cache.k_scale.clone()
    out, now = cache.append(q, k, k, rope.RopeTable(64, device=cuda), _cu([0, 0], cuda), _i32([5, 17], cuda),
                            _i32([[0, 0], [1, 2]], cuda))
    assert out.shape == (0, 4, 64) and now.tolist() == [5, 17]
    assert torch.equal(keep[0].view(torch.uint8), cache.k.view(torch.uint8)) and torch.equal(keep[1], cache.k_scale)
    both = torch.tensor([5, 17, 0], dtype=torch.int32, device=cuda)
    with pytest.raises(Exception, match="len_out"):
        cache.append(q, k, k, rope.RopeTable(64, device=cuda), _cu([0, 0], cuda), both[:2], _i32([[0, 0], [1, 2]], cuda),
                     len_out=both[1:])


# ------------------------------------------------------------------------------- together

def test_refused_calls(cuda):
    from mlx_dspark_b200 import DSparkError, DSparkUnsupported, paged, rope

    cache = paged.PagedCache.empty(4, 2, 16, 64, cuda)
    table = rope.RopeTable(64, device=cuda)
    q, k = (torch.zeros(3, h, 64, dtype=BF, device=cuda) for h in (4, 2))
    cu, ln, pt = _cu([3], cuda), _i32([0], cuda), _i32([[0, 1]], cuda)
    for bad in (dict(q=q[..., :32]), dict(k=k[:2]), dict(v=k[:, :1]), dict(q=q.float(), k=k.float(), v=k.float()),
                dict(k=k.to(HF)), dict(cu=cu.long()), dict(cu=_cu([1, 2], cuda)), dict(ln=_i32([0, 0], cuda)),
                dict(pt=pt.long()), dict(pt=pt[0]), dict(pt=_i32([[0, 1]] * 2, cuda)), dict(len_out=ln),
                dict(row_pos=_i32([0, 1], cuda)), dict(q_out=q[:2]), dict(table=rope.RopeTable(128, device=cuda))):
        a = dict(q=q, k=k, v=k, table=table, cu=cu, ln=ln, pt=pt) | bad
        with pytest.raises(DSparkError):
            cache.append(a["q"], a["k"], a["v"], a["table"], a["cu"], a["ln"], a["pt"],
                         **{x: a[x] for x in ("len_out", "row_pos", "q_out") if x in a})
    for bad in (dict(q=q[:, :3]), dict(q=q.float()), dict(q=q[0]), dict(out=q[:2]), dict(out=q.to(HF)), dict(cu=cu.long()),
                dict(ln=ln.long()), dict(pt=_i32([[0, 1]] * 3, cuda)), dict(q=q.transpose(1, 2))):
        a = dict(q=q, cu=cu, ln=ln, pt=pt, out=None) | bad
        with pytest.raises(DSparkError):
            cache.attention(a["q"], a["cu"], a["ln"], a["pt"], scale=1.0, out=a["out"])
    with pytest.raises(DSparkUnsupported):
        paged.PagedCache(cache.k[..., 8:40], cache.v[..., 8:40], cache.k_scale, cache.v_scale)


def test_rounds_together(cuda):
    """A prompt, then verify rounds with rollback, the scores of what came out: every round against the values that
    the cache holds, in 64 bits; captured and replayed it gives the same bits."""
    from mlx_dspark_b200 import paged, rope, sampling

    rng, g = random.Random(5), torch.Generator().manual_seed(5)
    B, Hq, Hk, D, page, V, width = 3, 8, 2, 64, 16, 1000, 8
    cache = paged.PagedCache.empty(B * width, Hk, page, D, cuda)
    twin = paged.PagedCache.empty(B * width, Hk, page, D, cuda)
    rows = _tables([width] * B, B * width, rng)
    pt, table = _i32(rows, cuda), rope.RopeTable(D, theta=1e4, device=cuda)
    head = torch.randn(Hq * D, V, generator=g).to(BF).to(cuda) * 0.1
    lens = [0] * B
    for counts in ([37, 5, 0], [4, 4, 9], [1, 4, 4], [4, 0, 4], [17, 1, 1]):
        R = sum(counts)
        q, k, v = (torch.randn(R, h, D, generator=g).to(BF).to(cuda) for h in (Hq, Hk, Hk))
        cu, ln = _cu(counts, cuda), _i32(lens, cuda)

        def step(c):
            qr, now = c.append(q, k, v, table, cu, ln, pt)
            o = c.attention(qr, cu, now, pt, scale=D ** -0.5)
            logits = o.flatten(1) @ head
            return qr, now, o, sampling.token_logprobs(logits, logits.argmax(1).to(torch.int32), top=4), logits

        qr, now, o, s, logits = step(cache)
        assert now.tolist() == [a + n for a, n in zip(lens, counts)]
        assert torch.equal(o, _check(cuda, cache, qr, counts, now.tolist(), rows, True, D ** -0.5))
        _check_scores(cuda, logits, logits.argmax(1).tolist(), None, 4)
        assert bool((s["rank"] == 0).all())
        side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(graph, stream=side):
            made = step(twin)
        graph.replay()
        graph.replay()  # (the same append twice: the scales are there already)
        torch.cuda.synchronize()
        assert torch.equal(made[2], o) and all(torch.equal(made[3][x], s[x]) for x in s)
        assert _same_codes(twin.k, cache.k) and torch.equal(twin.v_scale, cache.v_scale)
        # what is rejected is taken back
        lens = [a - (rng.randint(0, n - 1) if n > 1 and a > 5 else 0) for a, n in zip(now.tolist(), counts)]


def test_two_streams(cuda):
    """Calls on two streams at once have workspaces of their own."""
    g = torch.Generator().manual_seed(20)
    cache = _finite_pool(cuda, 80, 8, 32, 128, g)
    rows = _i32([list(range(80))], cuda)
    qs = [torch.randn(n, 32, 128, generator=g).to(BF).to(cuda) for n in (1, 8)]
    cus = [_cu([q.shape[0]], cuda) for q in qs]
    ln = _i32([2500], cuda)
    want = [cache.attention(q, c, ln, rows, scale=0.09) for q, c in zip(qs, cus)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(cache.attention(qs[i], cus[i], ln, rows, scale=0.09))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in got[i])
