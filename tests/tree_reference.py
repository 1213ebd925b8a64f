"""Plain 64-bit forms of the tree-round operators, for the tests (numpy / torch on the CPU)."""

from __future__ import annotations

import math
import random

import numpy as np
import torch

F32_MAX = float(np.finfo(np.float32).max)


def random_parents(n: int, rng: random.Random, width: int = 3) -> list[int]:
    return [-1] + [rng.randint(max(0, (i - 1) // width - 2), i - 1) for i in range(1, n)]


def ancestors(parent: list[int]) -> list[set[int]]:
    out = []
    for i, p in enumerate(parent):
        out.append({i} | (out[p] if 0 <= p < i else set()))
    return out


def depths(parent: list[int]) -> list[int]:
    out = []
    for i, p in enumerate(parent):
        out.append(out[p] + 1 if 0 <= p < i else 0)
    return out


def words_of(anc: list[set[int]], words: int) -> list[list[int]]:
    rows = []
    for s in anc:
        row = [0] * words
        for j in s:
            if j < 32 * words:
                row[j // 32] |= 1 << (j % 32)
        rows.append([w - (1 << 32) if w >= 1 << 31 else w for w in row])
    return rows


def rope(x, inv_freq, mscale, pos, rot, layout, norm=None, eps=1e-6):
    """x [R, H, D] double, pos [R]."""
    if norm is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * norm
    a = pos.double()[:, None, None] * torch.tensor(inv_freq, dtype=torch.float64)
    c, s = torch.cos(a) * mscale, torch.sin(a) * mscale
    y = x.clone()
    i0 = slice(0, rot // 2) if layout == "half" else slice(0, rot, 2)
    i1 = slice(rot // 2, rot) if layout == "half" else slice(1, rot, 2)
    y[..., i0] = x[..., i0] * c - x[..., i1] * s
    y[..., i1] = x[..., i1] * c + x[..., i0] * s
    return y


def attention(q, k, v, visible, scale):
    """q [n, Hq, D], k / v [Hk, L, D], visible [n, L] bool; all double. Returns the output and the
    bound's weights: sum of p |v| and the sum of |v| over the visible keys. Keys nobody may use
    (masked for a row) never enter its sums."""
    n, hq, d = q.shape
    hk, L = k.shape[0], k.shape[1]
    g = hq // hk
    out = torch.zeros(n, hq, d, dtype=torch.float64)
    absum, vsum = torch.zeros_like(out), torch.zeros_like(out)
    for i in range(n):
        j = torch.nonzero(visible[i]).flatten()
        if not len(j):
            continue
        for h in range(hq):
            s = (k[h // g, j] @ q[i, h]) * scale
            w = torch.softmax(s, 0)
            out[i, h] = w @ v[h // g, j]
            absum[i, h] = w @ v[h // g, j].abs()
            vsum[i, h] = v[h // g, j].abs().sum(0)
    return out, absum, vsum


def probabilities(logits, T):
    """Rows of p = softmax(logits / T) as the accept defines them (double numpy)."""
    l = np.asarray(logits, dtype=np.float64)
    l = np.where(np.isnan(l), -np.inf, np.minimum(l, F32_MAX))
    p = np.zeros_like(l)
    for r in range(l.shape[0]):
        m = l[r].max() if l.shape[1] else -np.inf
        if m == -np.inf:
            continue
        if not T > 0:
            p[r, int(np.argmax(l[r]))] = 1.0
            continue
        e = np.exp((l[r] - m) / T)
        p[r] = e / e.sum()
    return p


def accept(p, ids, parent, u, noise, draft, greedy, margin=1e-5):
    """One request's accept. Returns (path, next, close): close tells that a comparison was decided by
    less than `margin` relative, so that 32-bit arithmetic may decide it the other way."""
    n, close = len(ids), False
    cur, path = 0, [0]
    chain = parent is None
    up = [i - 1 for i in range(n)] if chain else parent
    while True:
        run, nxt, seen = 0.0, None, set()
        for j in range(cur + 1, n):
            if up[j] != cur or ids[j] in seen:
                continue
            seen.add(ids[j])
            px = p[cur, ids[j]] if 0 <= ids[j] < p.shape[1] else 0.0
            if chain:
                q = 1.0 if draft is None or greedy else float(draft[cur, ids[j]])
                a, b = u[cur] * q, px
            else:
                run += px
                a, b = u[cur], run
            if abs(a - b) <= margin * max(abs(a), abs(b)) and a != b:
                close = True
            if a < b:
                nxt = j
                break
        if nxt is None:
            break
        cur = nxt
        path.append(cur)
    w = p[cur].copy()
    if w.sum() == 0:
        return path, -1, close
    if chain and draft is not None and not greedy:
        if cur + 1 < n:
            w = np.maximum(w - draft[cur].astype(np.float64), 0.0)
    else:
        for j in range(cur + 1, n):
            if up[j] == cur and 0 <= ids[j] < len(w):
                w[ids[j]] = 0.0
    if not (w > 0).any():
        w = p[cur].copy()
    with np.errstate(divide="ignore", invalid="ignore"):
        race = np.where(w > 0, w / noise, -1.0)
    top = int(np.argmax(race))
    second = np.partition(race, -2)[-2] if len(race) > 1 else -1.0
    # a residual is a difference: its 32-bit error is relative to p, not to p - q
    slack = margin * (1.0 + p[cur].max() / max(w[top], 1e-300)) if chain and draft is not None else margin
    if second > 0 and race[top] - second <= slack * race[top]:
        close = True
    return path, top, close
