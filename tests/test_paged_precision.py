"""How precise the attention over pages is: a bound for each row and key, tight enough that scores or weights of fewer bits, or
parts that are joined a little wrong, fail it.

The scores vary by several units, so that a row's result is made of a few keys: errors do not average out over many. With
a = |scale| sum |q_d k_d|, s the score, m the row's largest and w the normalised weight of a key (all 64 bits) a score is off by at most

    e = ((D + 8) a + 4 |s| + 4 |m| + 64) 2^-23

in units of the natural logarithm: (D + 8) 2^-23 a for the sum of D exact products, whichever way the tensor core cuts its fp32
sums off; 2^-22 |s| for the factor (the scale, log2 e and their product, 2^-24 each); 2^-23 (|s| + |m| + 15) for the multiply-add
with the maximum and its summand; 2^-22 and 2^-22 for exponential and logarithm. A weight is off by e, and in the product with v by half
an fp16 step, 2^-11; the denominator has no fp16 step. L terms add up with (L + 64) 2^-23, joins among them. What fp16 loses of a
weight far below the largest is at most 2^-32 of it a key. The result is rounded to fp16.
"""

from __future__ import annotations

import math
import random

import pytest
import torch
from test_paged_gpu import _cu, _far, _i32, _tables, _with_room

HF = torch.float16
E4M3 = torch.float8_e4m3fn


def _case(n, L, Hq, Hk, D, spread, seed):
    """q [n, Hq, D] fp16, codes [Hk, L, D] of k and v, the scores' scale. Values are code / 64."""
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(n, Hq, D, generator=g).to(HF)
    k, v = ((64 * torch.randn(Hk, L, D, generator=g)).clamp(-448, 448).to(E4M3) for _ in range(2))
    return q, k, v, spread * D ** -0.5


def _exact(q, k, v, scale, causal):
    """The result [n, Hq, D] and its bound without the last rounding; the scores and v for the forms with mistakes."""
    n, Hq, D = q.shape
    Hk, L, _ = k.shape
    qd = q.double().view(n, Hk, Hq // Hk, D).permute(1, 2, 0, 3)           # [Hk, G, n, D]
    kd, vd = k.double()[:, None] / 64, v.double()[:, None] / 64            # [Hk, 1, L, D]
    s = qd @ kd.transpose(2, 3) * scale
    a = qd.abs() @ kd.abs().transpose(2, 3) * abs(scale)
    if causal:
        hidden = torch.ones(n, L, dtype=torch.bool).tril(L - n).logical_not()
        s = s.masked_fill(hidden, -math.inf)
    m = s.amax(-1, keepdim=True)
    w = torch.softmax(s, -1)
    e = ((D + 8) * a + 4 * s.abs().nan_to_num(0.0, 0.0, 0.0) + 4 * m.abs() + 64) * 2.0 ** -23
    out = w @ vd
    lim = (w * (2.0 ** -11 + 1.01 * e + (L + 64) * 2.0 ** -23)) @ vd.abs() + out.abs() * (w * 1.01 * e).sum(-1, keepdim=True) + \
        out.abs() * (L + 64) * 2.0 ** -23 + 2.0 ** -32 * vd.abs().sum(2, keepdim=True)
    back = lambda t: t.permute(2, 0, 1, 3).reshape(n, Hq, D)  # noqa: E731
    return back(out), back(lim), s, vd, back


def _half_step(x):
    return 2.0 ** -11 * x.abs().clamp(min=2.0 ** -14)


def _worst(got, want, lim):
    return float(((got.double() - want).abs() / (lim + _half_step(want))).max())


CASES = [
    # rows, keys, Hq, Hk, D, spread, causal
    (1, 1900, 8, 2, 64, 5.0, True),
    (4, 1301, 8, 2, 128, 5.0, True),
    (30, 700, 4, 1, 64, 4.0, False),
    (90, 1025, 4, 2, 64, 5.0, True),
    (200, 513, 4, 1, 128, 4.0, True),
]


def _joined(s, vd, cut, off):
    """The result of two parts, of the keys before and from `cut` on, the first one's log sum off by `off`."""
    parts = []
    for x, v in ((s[..., :cut], vd[:, :, :cut]), (s[..., cut:], vd[:, :, cut:])):
        lse = torch.logsumexp(x, -1, keepdim=True)
        parts.append((lse, torch.softmax(x, -1).nan_to_num(0.0) @ v))
    (l0, o0), (l1, o1) = parts
    f = torch.sigmoid(l0 + off - l1)
    return o0 * f + o1 * (1 - f)


@pytest.mark.parametrize("case", CASES, ids=range(len(CASES)))
def test_the_bound_tells_right_from_nearly_right(case):
    """Weights in fp16 with scores in fp32 are within the bound; weights in bf16, scores in fp16 (the weights' sum rounded or not),
    two parts joined with a log sum that is off by 2 % are not."""
    n, L, Hq, Hk, D, spread, causal = case
    q, k, v, scale = _case(n, L, Hq, Hk, D, spread, n + L)
    want, lim, s, vd, back = _exact(q, k, v, scale, causal)

    def result(s, weight, total):
        p = torch.exp(s - s.amax(-1, keepdim=True)) * 2.0 ** 7
        x = torch.linspace(1, 0.5, 7).double()[torch.arange(s.shape[2]) % 7][:, None]  # (the maximum in use is any)
        return back((weight(p * x) @ vd) / total(p * x).sum(-1, keepdim=True)).to(HF)

    same, f16, b16 = (lambda t: t), (lambda t: t.to(HF).double()), (lambda t: t.to(torch.bfloat16).double())
    fine = [_worst(result(s, f16, same), want, lim), _worst(result(s.float().double(), f16, same), want, lim)]
    wrong = [_worst(result(s, b16, same), want, lim), _worst(result(s.to(HF).double(), f16, same), want, lim),
             _worst(result(s.to(HF).double(), f16, f16), want, lim), _worst(back(_joined(s, vd, L // 2, 0.02)).to(HF), want, lim)]
    print([round(x, 2) for x in fine + wrong])
    assert max(fine) <= 1 and min(wrong) > 1, (fine, wrong)


# where a call goes: as it is, to clusters of blocks where there are few rows, to shares of a line, to the kernel for many rows
ROOMS = {"tight": lambda rows, page: rows, "clusters": lambda rows, page: _with_room(rows, page, 6000),
         "shares": lambda rows, page: _with_room(rows, page, 40000), "far": _far}


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("room", list(ROOMS))
@pytest.mark.parametrize("case", CASES, ids=range(len(CASES)))
def test_attention_is_within_the_bound(cuda, case, room, page):
    from mlx_dspark_b200 import paged

    n, L, Hq, Hk, D, spread, causal = case
    q, k, v, scale = _case(n, L, Hq, Hk, D, spread, n + L + page)
    want, lim, *_ = _exact(q, k, v, scale, causal)
    need = -(-L // page)
    rows = _tables([need], need + 3, random.Random(L))
    cache = paged.PagedCache.empty(need + 3, Hk, page, D, cuda)
    cache.k_scale.fill_(2.0 ** -6), cache.v_scale.fill_(2.0 ** -6)
    for pool, x in ((cache.k, k), (cache.v, v)):
        x = torch.nn.functional.pad(x.view(torch.uint8), (0, 0, 0, need * page - L))
        pool.view(torch.uint8)[rows[0]] = x.view(Hk, need, page, D).transpose(0, 1).to(cuda)
    out = cache.attention(q.to(cuda), _cu([n], cuda), _i32([L], cuda), _i32(ROOMS[room](rows, page), cuda), scale=scale,
                          causal=causal)
    worst = _worst(out.cpu(), want, lim)
    assert worst <= 1, worst
