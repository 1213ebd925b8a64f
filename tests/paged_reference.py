"""Plain 64-bit forms of the paged 8-bit cache and of token scores, for the tests (torch on the CPU)."""

from __future__ import annotations

import math

import torch

E4M3 = torch.float8_e4m3fn


def nearest(x: torch.Tensor) -> torch.Tensor:
    """The nearest e4m3 value, ties to even, at most 448 (infinities too); NaN stays NaN."""
    step = torch.exp2(torch.frexp(x.abs().clamp(min=2.0 ** -6, max=448.0)).exponent.double() - 4)
    return (torch.round(x / step) * step).clamp(-448, 448)


def scale_of(amax: float) -> float:
    """The smallest power of two, 2^-64 to 2^64, with amax <= 448 * scale."""
    e = -64
    while e < 64 and amax > 448 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def amax(x: torch.Tensor) -> float:
    y = x[torch.isfinite(x)].abs()
    return float(y.max()) if y.numel() else 0.0


def values(codes: torch.Tensor, scale: torch.Tensor, table, n: int) -> torch.Tensor:
    """Tokens 0 .. n - 1 of a request as doubles [H, n, D]; codes [pages, H, page, D] on the CPU."""
    page, H, D = codes.shape[2], codes.shape[1], codes.shape[3]
    t = torch.as_tensor(table[: -(-n // page)], dtype=torch.long)
    x = codes.view(torch.uint8)[t].view(E4M3).double() * scale[t].double()[..., None, None]
    return x.permute(1, 0, 2, 3).reshape(H, -1, D)[:, :n]


def append(codes, scale, table, kv_len, x, spread):
    """Appends x [n, H, D] (double; each value known to +-spread) to one request's pages. Returns what may stand
    in the cache: (lowest codes, highest codes) [pages, H, page, D] as doubles, the lowest and highest scales."""
    lo, hi = codes.double(), codes.double()
    s_lo, s_hi = scale.double(), scale.double()
    page = codes.shape[2]
    for first in sorted({(kv_len + i) // page for i in range(x.shape[0])}):
        pid = table[first]
        at = [i for i in range(x.shape[0]) if (kv_len + i) // page == first]
        begin = max(kv_len - first * page, 0)
        off = [(kv_len + i) % page for i in at]
        for h in range(codes.shape[1]):
            y, d = x[at, h], spread[at, h]
            ends = []
            for sign in (-1, 1):
                s = scale_of(amax((y.abs() + sign * d).clamp(min=0)))
                ends.append(max(s, float(scale[pid, h])) if begin else s)
            s_lo[pid, h], s_hi[pid, h] = ends
            if ends[0] != ends[1]:
                lo[pid, h, off], hi[pid, h, off] = -448.0, 448.0
                continue
            if begin:
                old = nearest(codes[pid, h, :begin].double() * (float(scale[pid, h]) / ends[0]))
                lo[pid, h, :begin] = hi[pid, h, :begin] = old
            lo[pid, h, off], hi[pid, h, off] = nearest((y - d) / ends[0]), nearest((y + d) / ends[0])
    return lo, hi, s_lo, s_hi


def score(row: torch.Tensor, token: int, temperature: float, top: int, low: float):
    """logprob, entropy, rank, ids and logprobs of the alternatives of one row (doubles). low: the largest value
    that masks its token."""
    x = row.double().clone()
    x[torch.isnan(x) | (x <= low)] = -math.inf
    x = x.clamp(max=2.0 ** 28 if row.dtype is not torch.float16 else 65504.0)  # larger ones count as that
    live = x > -math.inf
    order = [int(i) for i in torch.sort(x, descending=True, stable=True).indices if live[int(i)]] if top else []
    V = x.numel()
    if not bool(live.any()):
        return -math.inf, 0.0, -1, [-1] * top, [-math.inf] * top
    if temperature <= 1e-6:
        y = torch.full_like(x, -math.inf)
        y[int(x.argmax())] = 0.0
        ent = 0.0
    else:
        y = torch.log_softmax(x / min(temperature, 1e6), 0)
        p = y.exp()
        ent = float(-(p[live] * y[live]).sum())
    ids = (order + [-1] * top)[:top]
    tl = [float(y[i]) if i >= 0 else -math.inf for i in ids]
    if not bool(live[token]):
        return -math.inf, ent, -1, ids, tl
    before = (x > x[token]) | ((x == x[token]) & (torch.arange(V) < token))
    return float(y[token]), ent, int(before.sum()), ids, tl
