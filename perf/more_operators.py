"""What the operators of a paged 8-bit cache and of token scoring are measured on: cases, inputs, plain forms
and 64-bit values.

A serving round over a paged cache runs three operators beside the projections: rotary positions of q and k
with the append of k and v to pages of 8-bit values that have one scale a page and head (``append``), attention
of packed rows over those pages (``attn``), and the log probabilities of given tokens with the entropy, the rank
and the top alternatives (``score``). Every case is one call of one of them. The plain forms are elementary
torch operations in 32 bits; with ``own`` set, the calls are those of the package.

A page holds ``page`` tokens of every head. The value of a code is e4m3(code) * scale, the scale of a page and
head the smallest power of two (2^-64 to 2^64) with which its largest value is at most 448. An append to a page
that already holds tokens takes the larger of the old and the new scale and rounds the old codes to it.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
E4M3 = torch.float8_e4m3fn


# ------------------------------------------------------------------------------- cases

def listed():
    return [
        # one decoded token of the 32/8-head, head_dim 128 target: latency
        {"name": "append-one-token", "op": "append", "batch": 1, "rows": 1, "ragged": False, "len": 2047, "hq": 32,
         "hk": 8, "d": 128, "rot": 128, "layout": "half", "norm": True, "page": 64, "type": "bf16"},
        # a verify round of 200 users, 1 to 16 rows each, pages of 16 tokens, half of the head rotated
        {"name": "append-verify-batch", "op": "append", "batch": 200, "rows": 16, "ragged": True, "len": 1500,
         "hq": 24, "hk": 8, "d": 128, "rot": 64, "layout": "interleaved", "norm": False, "page": 16, "type": "f16"},
        # a long prompt that goes on in a page with tokens
        {"name": "append-prompt", "op": "append", "batch": 1, "rows": 16389, "ragged": False, "len": 37, "hq": 32,
         "hk": 8, "d": 128, "rot": 128, "layout": "half", "norm": True, "page": 64, "type": "bf16"},
        # plain decoding, one row at 2k of context: latency
        {"name": "attn-one-token", "op": "attn", "batch": 1, "rows": 1, "ragged": False, "len": 2049, "hq": 32,
         "hk": 8, "d": 128, "page": 64, "causal": True, "type": "bf16"},
        # decoding of 96 users with contexts of 256 to 16k, pages of 16 tokens
        {"name": "attn-decode-batch", "op": "attn", "batch": 96, "rows": 1, "ragged": True, "len": 16384, "hq": 32,
         "hk": 8, "d": 128, "page": 16, "causal": True, "type": "bf16"},
        # a verify round: 24 users with blocks of 1 to 16 rows, contexts of 256 to 16k
        {"name": "attn-verify-batch", "op": "attn", "batch": 24, "rows": 16, "ragged": True, "len": 16000, "hq": 32,
         "hk": 8, "d": 128, "page": 64, "causal": True, "type": "f16"},
        # two prompts' chunks at 16k of a 64/8-head target: bound by the matrix products
        {"name": "attn-prompt-chunks", "op": "attn", "batch": 2, "rows": 509, "ragged": False, "len": 16381, "hq": 64,
         "hk": 8, "d": 128, "page": 128, "causal": True, "type": "bf16"},
        # one token of one user with five alternatives: latency
        {"name": "score-one-token", "op": "score", "rows": 1, "vocab": 151936, "top": 5, "temp": False,
         "type": "bf16"},
        # a verify round's rows with the widest list of alternatives, 32-bit logits, another temperature each
        {"name": "score-verify-batch", "op": "score", "rows": 272, "vocab": 151936, "top": 20, "temp": True,
         "type": "f32"},
        # scoring of a text: many rows, no alternatives
        {"name": "score-text", "op": "score", "rows": 2049, "vocab": 151936, "top": 0, "temp": False,
         "type": "bf16"},
        # the log of a serving batch, a vocabulary of odd size
        {"name": "score-serving-batch", "op": "score", "rows": 700, "vocab": 128257, "top": 5, "temp": False,
         "type": "f16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_HEADS = [(32, 8), (64, 8), (8, 8), (16, 2), (24, 8), (20, 4), (12, 4), (7, 1)]


def draw(rng):
    op = rng.choice(["append", "attn", "attn", "score"])
    t = rng.choice(["bf16", "f16"])
    if op == "score":
        rows, vocab = _log(rng, 1, 2000), _log(rng, 500, 260000)
        t = rng.choice(["bf16", "f16", "f32"])
        while rows * vocab * (2 if t == "f32" else 1) > 2049 * 151936:
            rows = rows * 2 // 3
        return {"op": op, "rows": rows, "vocab": vocab, "top": rng.choice([0, 0, 1, 5, 11, 20, 32]),
                "temp": rng.random() < 0.4, "type": t}
    hq, hk = rng.choice(_HEADS)
    d, page = rng.choice([64, 128, 128]), rng.choice([16, 32, 64, 128])
    if op == "append":
        batch = _log(rng, 1, 256)
        rows = _log(rng, 1, max(1, 8000 // batch))
        ln = _log(rng, 1, 30000)
        while batch * (ln + rows) * hk * d > 4e8:
            ln = ln * 2 // 3
        return {"op": op, "batch": batch, "rows": rows, "ragged": rng.random() < 0.6, "len": ln, "hq": hq, "hk": hk,
                "d": d, "rot": rng.choice([d, d, d // 2, d // 4]), "layout": rng.choice(["half", "interleaved"]),
                "norm": rng.random() < 0.5, "page": page, "type": t}
    ln, batch, rows = _log(rng, 1, 32768), _log(rng, 1, 96), _log(rng, 1, 300)
    if rng.random() < 0.4:
        rows = 1
    while 4.0 * batch * rows * hq * ln > 4.0e9 or batch * ln * hk * d > 9e8:
        batch, rows = max(1, batch * 2 // 3), max(1, rows * 2 // 3)
        ln = ln if batch * rows > 1 else ln * 2 // 3
    return {"op": op, "batch": batch, "rows": rows, "ragged": rng.random() < 0.6, "len": max(ln, rows), "hq": hq,
            "hk": hk, "d": d, "page": page, "causal": rng.random() < 0.8, "type": t}


# ------------------------------------------------------------------------------- shapes of a case

def _shape_rng(case):
    """The ragged sizes belong to the case, not to the seed."""
    key = "/".join("%s=%s" % kv for kv in sorted(case.items()) if kv[0] != "name")
    return random.Random(key)


def _counts(case):
    """Rows of each request."""
    r, n = _shape_rng(case), case["rows"]
    if not case["ragged"]:
        return [n] * case["batch"]
    return [n] + [r.randint(1, n) for _ in range(case["batch"] - 1)]


def _lens(case, counts):
    """Keys of each request: before the append, or with the rows for the attention."""
    r = random.Random(_shape_rng(case).random())
    if not case["ragged"]:
        return [case["len"]] * case["batch"]
    lo = min(256, case["len"])
    add = 0 if case["op"] == "append" else 1
    return [case["len"]] + [max(n * add, _log(r, lo, case["len"])) for n in counts[1:]]


def _size(case):
    return 4 if case["type"] == "f32" else 2


def work(case):
    e = _size(case)
    if case["op"] == "score":
        n = case["rows"] * case["vocab"]
        return {"bytes": e * n + case["rows"] * (16 + 8 * case["top"]), "flops": 8 * n}
    n = _counts(case)
    ln = _lens(case, n)
    hq, hk, d, page = case["hq"], case["hk"], case["d"], case["page"]
    R = sum(n)
    if case["op"] == "append":
        pages = sum((x + r - 1) // page - x // page + 1 for r, x in zip(n, ln))
        by = R * d * (2 * e * hq + (e + 1) * 2 * hk) + pages * (4 + 8 * hk)
        return {"bytes": by, "flops": R * d * (6 * hq + 10 * hk)}
    by = sum(2 * x * hk * d + (x + page - 1) // page * (4 + 8 * hk) for x in ln) + 2 * e * R * hq * d
    seen = sum(r * x - (r * (r - 1) // 2 if case["causal"] else 0) for r, x in zip(n, ln))
    return {"bytes": by, "flops": 4 * seen * hq * d}


# ------------------------------------------------------------------------------- inputs

def _pages(case, n, ln, g, dev):
    """A page table in no order and how many pages there are."""
    page = case["page"]
    more = n if case["op"] == "append" else [0] * len(n)
    need = [max(1, -(-(x + r) // page)) for x, r in zip(ln, more)]
    total, width = sum(need) + 3, max(need)
    perm = torch.randperm(total, device=dev, generator=g).to(torch.int32)
    at = torch.tensor([0] + need[:-1], device=dev).cumsum(0)[:, None] + torch.arange(width, device=dev)
    there = torch.arange(width, device=dev)[None] < torch.tensor(need, device=dev)[:, None]
    # places behind a request's last page hold what a table that is used again holds: some other page
    return torch.where(there, perm[at.clamp(max=total - 1)], perm[-1]).contiguous(), total


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    dt = DTYPES[case["type"]]
    i32 = dict(dtype=torch.int32, device=dev)
    s = {"case": case, "op": case["op"]}

    def randn(*shape, dtype=dt):
        return torch.randn(shape, device=dev, generator=g, dtype=torch.float32).to(dtype)

    if case["op"] == "score":
        R, V = case["rows"], case["vocab"]
        logits = torch.randn(R, V, device=dev, generator=g).mul_(3)
        favoured = torch.randint(V, (R, 4), device=dev, generator=g)
        logits.scatter_(1, favoured, 13 + 3 * torch.rand(R, 4, device=dev, generator=g))
        s["logits"] = logits.to(dt)
        # mostly one of the favourites, now and then any token
        any_ = torch.randint(V, (R,), device=dev, generator=g)
        s["tokens"] = torch.where(any_ % 4 == 0, any_, favoured[:, 0]).to(torch.int32)
        s["temp"] = 0.5 + torch.rand(R, device=dev, generator=g) if case["temp"] else None
        return s
    n = _counts(case)
    ln = _lens(case, n)
    R, hq, hk, d, page = sum(n), case["hq"], case["hk"], case["d"], case["page"]
    s["cu"] = torch.tensor([0] + list(torch.tensor(n).cumsum(0).tolist()), **i32)
    s["len"] = torch.tensor(ln, **i32)
    s["table"], total = _pages(case, n, ln, g, dev)

    def pool():
        x = torch.empty(total, hk, page, d, dtype=torch.bfloat16, device=dev).normal_(generator=g)
        return x.mul_(64).clamp_(-448, 448).to(E4M3)

    def scales():
        return torch.exp2(torch.randint(-7, -4, (total, hk), device=dev, generator=g).float())

    s["k"], s["v"], s["ks"], s["vs"] = pool(), pool(), scales(), scales()
    s["rows"], s["max_len"] = max(n), max(ln)
    if case["op"] == "append":
        qkv = randn(R, (hq + 2 * hk) * d)  # the projection's product, split without copies
        s["q"] = qkv[:, : hq * d].view(R, hq, d)
        s["kn"] = qkv[:, hq * d : (hq + hk) * d].view(R, hk, d)
        s["vn"] = qkv[:, (hq + hk) * d :].view(R, hk, d)
        s["wq"] = (1 + 0.1 * randn(d, dtype=torch.float32)).to(dt) if case["norm"] else None
        s["wk"] = (1 + 0.1 * randn(d, dtype=torch.float32)).to(dt) if case["norm"] else None
        i = torch.arange(0, case["rot"], 2, dtype=torch.float64, device=dev)
        s["inv"] = 1e6 ** (-i / case["rot"])
        s["out"] = torch.empty(R, hq, d, dtype=dt, device=dev)
        s["new_len"] = torch.empty_like(s["len"])
        if own:
            from mlx_dspark_b200 import rope
            s["rope"] = rope.RopeTable(d, case["rot"], theta=1e6, layout=case["layout"], device=dev)
    else:
        s["q"] = randn(R, hq, d)
        s["out"] = torch.empty_like(s["q"])
    if own:
        from mlx_dspark_b200 import paged
        s["cache"] = paged.PagedCache(s["k"], s["v"], s["ks"], s["vs"])
    return s


# ------------------------------------------------------------------------------- one pass

def run(s):
    return (_run_own if own else _run_plain)[s["op"]](s)


def _appended(s):
    return {"q": s["out"], "len": s["new_len"], "k": s["k"], "v": s["v"], "k_scale": s["ks"], "v_scale": s["vs"]}


def _own_append(s):
    s["cache"].append(s["q"], s["kn"], s["vn"], s["rope"], s["cu"], s["len"], s["table"], q_norm=s["wq"],
                      k_norm=s["wk"], eps=1e-6, q_out=s["out"], len_out=s["new_len"])
    return _appended(s)


def _own_attn(s):
    return s["cache"].attention(s["q"], s["cu"], s["len"], s["table"], scale=s["case"]["d"] ** -0.5,
                                causal=s["case"]["causal"], out=s["out"])


def _own_score(s):
    from mlx_dspark_b200 import sampling
    return sampling.token_logprobs(s["logits"], s["tokens"], temperature=s["temp"], top=s["case"]["top"])


_run_own = {"append": _own_append, "attn": _own_attn, "score": _own_score}


def _rows(cu, R):
    """Request and place within it of each packed row."""
    r = torch.arange(R, device=cu.device, dtype=torch.int32)
    req = (torch.searchsorted(cu, r, right=True) - 1).long()
    return req, r.long() - cu.long()[req]


def _turned(s, x, w, cos, sin):
    """Rows of heads in fp32, normed and rotated."""
    c = s["case"]
    rot, half = c["rot"], c["rot"] // 2
    x = x.float()
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.float()
    y = x.clone()
    if c["layout"] == "half":
        x0, x1 = x[..., :half], x[..., half:rot]
        y[..., :half] = x0 * cos - x1 * sin
        y[..., half:rot] = x1 * cos + x0 * sin
    else:
        x0, x1 = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2] = x0 * cos - x1 * sin
        y[..., 1:rot:2] = x1 * cos + x0 * sin
    return y


def _plain_append(s):
    c, R, page = s["case"], s["q"].shape[0], s["case"]["page"]
    req, at = _rows(s["cu"], R)
    slot = s["len"].long()[req] + at
    a = slot.double()[:, None, None] * s["inv"]  # in 64 bits: a far position's angle
    cos, sin = torch.cos(a).float(), torch.sin(a).float()
    s["out"].copy_(_turned(s, s["q"], s["wq"], cos, sin))
    s["new_len"].copy_(s["len"] + s["cu"][1:] - s["cu"][:-1])
    pg, off = s["table"].long()[req, slot // page], slot % page
    first = s["table"].long().gather(1, (s["len"].long() // page)[:, None].clamp(max=s["table"].shape[1] - 1))[:, 0]
    begun = s["len"].long() % page  # tokens that each request's first page has
    for x, codes, scale in ((_turned(s, s["kn"], s["wk"], cos, sin), s["k"], s["ks"]),
                            (s["vn"].float(), s["v"], s["vs"])):
        top = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(-1)  # [R, heads]
        most = torch.zeros_like(scale).scatter_reduce_(0, pg[:, None].expand_as(top), top, "amax")
        m, e = torch.frexp(most)
        e = torch.where(most > 0, e - 9 + (m > 0.875).to(e.dtype), torch.full_like(e, -64)).clamp(-64, 64)
        need = torch.exp2(e.float())
        here, old = need[first], scale[first]  # [B, heads]
        kept = torch.where((begun > 0)[:, None], torch.maximum(here, old), here)
        mine = torch.arange(page, device=x.device)[None] < begun[:, None]
        byte = codes.view(torch.uint8)
        have = byte[first]
        again = (have.view(E4M3).float() * (old / kept)[:, :, None, None]).clamp(-448, 448).to(E4M3)
        byte[first] = torch.where(mine[:, None, :, None], again.view(torch.uint8), have)
        scale[pg] = need[pg]
        scale[first] = kept
        byte[pg, :, off] = (x / scale[pg][:, :, None]).clamp(-448, 448).to(E4M3).view(torch.uint8)
    return _appended(s)


def _plain_attn(s):
    c = s["case"]
    B, hk, d, L, N, page = c["batch"], c["hk"], c["d"], s["max_len"], s["rows"], c["page"]
    G, R, dev = c["hq"] // hk, s["q"].shape[0], s["q"].device
    cu, ln = s["cu"].long(), s["len"].long()
    i = torch.arange(N, device=dev)
    row = (cu[:-1, None] + i).clamp(max=R - 1)
    q = s["q"][row].float().view(B, N, hk, G, d).permute(0, 2, 3, 1, 4).reshape(B, hk, G * N, d)
    t = s["table"].long()[:, : -(-L // page)]

    def values(codes, scale):
        x = codes.view(torch.uint8)[t].view(E4M3).float() * scale[t][..., None, None]  # [B, pages, heads, page, d]
        return x.transpose(1, 2).reshape(B, hk, -1, d)[:, :, :L]

    key, n = torch.arange(L, device=dev), cu[1:] - cu[:-1]
    last = ln[:, None] - n[:, None] + i if c["causal"] else (ln - 1)[:, None].expand(B, N)
    seen = (key <= last[..., None]) & (key < ln[:, None, None])  # [B, N, L]
    z = torch.matmul(q, values(s["k"], s["ks"]).transpose(2, 3)).mul_(d ** -0.5).view(B, hk, G, N, L)
    z.masked_fill_(~seen[:, None, None], -math.inf)
    m = z.amax(-1, keepdim=True)
    p = z.sub_(torch.where(torch.isinf(m), torch.zeros_like(m), m)).exp_()
    w = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, hk, G * N, L), values(s["v"], s["vs"])).view(B, hk, G, N, d)
    o = o / torch.where(w == 0, torch.ones_like(w), w)
    req, at = _rows(s["cu"], R)
    s["out"].copy_(o.permute(0, 3, 1, 2, 4).reshape(B, N, hk * G, d)[req, at])
    return s["out"]


def _plain_score(s):
    V, top = s["case"]["vocab"], s["case"]["top"]
    z, tok = s["logits"].float(), s["tokens"].long()[:, None]
    mine = z.gather(1, tok)
    j = torch.arange(V, device=z.device)
    rank = ((z > mine) | ((z == mine) & (j < tok))).sum(1)
    out = {"rank": rank.to(torch.int32)}
    if top:  # the order of the values and, among equal ones, of the tokens in one whole number
        b = z.view(torch.int32).long()
        key = torch.where(b < 0, -2147483648 - b, b) * 2097152 + (V - 1 - j)
        out["top_ids"] = (V - 1 - (key.topk(top, 1).values & 2097151)).to(torch.int32)
    x = z if s["temp"] is None else z / s["temp"][:, None]
    x = x - x.amax(1, keepdim=True)
    e = torch.exp(x)
    total = e.sum(1, keepdim=True)
    lse = torch.log(total)
    out["logprob"] = (x.gather(1, tok) - lse)[:, 0]
    out["entropy"] = (lse - (e * x).sum(1, keepdim=True) / total)[:, 0]
    if top:
        out["top_logprobs"] = x.gather(1, out["top_ids"].long()) - lse
    return out


_run_plain = {"append": _plain_append, "attn": _plain_attn, "score": _plain_score}


# ------------------------------------------------------------------------------- 64 bits

def _nearest_e4m3(x):
    """The nearest value of sign, 4 bits of exponent and 3 of mantissa, ties to even, at most 448."""
    step = torch.exp2(torch.frexp(x.abs().clamp(min=2.0 ** -6)).exponent.double() - 4)
    return (torch.round(x / step) * step).clamp(-448, 448)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "score":
        lp, ent, tl, top = [], [], [], case["top"]
        for r in range(0, case["rows"], 64):
            z = s["logits"][r : r + 64].double()
            order = None
            if top:
                order = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :top]
            if s["temp"] is not None:
                z = z / s["temp"][r : r + 64, None].double()
            y = torch.log_softmax(z, 1)
            lp.append(y.gather(1, s["tokens"][r : r + 64, None].long())[:, 0])
            ent.append(-(y.exp() * y).sum(1))
            if top:
                tl.append(y.gather(1, order))
        out = {"rank": None, "logprob": torch.cat(lp), "entropy": torch.cat(ent)}
        if top:
            out |= {"top_ids": None, "top_logprobs": torch.cat(tl)}
        return out
    n = _counts(case)
    ln, page, hk, d = _lens(case, n), case["page"], case["hk"], case["d"]
    if case["op"] == "attn":
        if sum(4.0 * a * b for a, b in zip(n, ln)) * case["hq"] * d > 5e12:
            return None
        out, r0, G = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), 0, case["hq"] // hk
        for b in range(case["batch"]):
            t = s["table"][b, : -(-ln[b] // page)].long()
            k, v = ((c.view(torch.uint8)[t].view(E4M3).double() * f[t].double()[:, :, None, None]).transpose(0, 1).reshape(hk, -1, d)[:, : ln[b]]
                    for c, f in ((s["k"], s["ks"]), (s["v"], s["vs"])))
            sees = torch.ones(n[b], ln[b], dtype=torch.bool, device="cuda")
            if case["causal"]:
                sees = sees.tril(ln[b] - n[b])
            for h in range(hk):
                q = s["q"][r0 : r0 + n[b], h * G : (h + 1) * G].double().transpose(0, 1)
                w = torch.softmax((q @ k[h].T * d ** -0.5).masked_fill(~sees, -math.inf), -1)
                out[r0 : r0 + n[b], h * G : (h + 1) * G] = (w @ v[h]).transpose(0, 1)
            r0 += n[b]
        return out
    rot, R, dev = case["rot"], sum(n), "cuda"
    slot = torch.tensor([x + i for r, x in zip(n, ln) for i in range(r)], device=dev)
    z = torch.polar(torch.ones(R, 1, rot // 2, device=dev, dtype=torch.float64),
                    slot.double()[:, None, None] * torch.tensor([1e6 ** (-2 * j / rot) for j in range(rot // 2)],
                                                                device=dev, dtype=torch.float64))

    def turned(x, w):
        x = x.double()
        if w is not None:
            x = x / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
        part, rest = x[..., :rot], x[..., rot:]
        if case["layout"] == "half":
            y = torch.complex(part[..., : rot // 2].contiguous(), part[..., rot // 2 :].contiguous()) * z
            return torch.cat([y.real, y.imag, rest], -1)
        y = torch.view_as_complex(part.reshape(*part.shape[:2], rot // 2, 2).contiguous()) * z
        return torch.cat([torch.view_as_real(y).flatten(2), rest], -1)

    # one page after the other is laid out as tokens in order, and rounded as a whole
    out = {"q": turned(s["q"], s["wq"]), "len": None}
    req = [b for b, r in enumerate(n) for _ in range(r)]
    for name, x, codes, scale in (("k", turned(s["kn"], s["wk"]), s["k"], s["ks"]),
                                  ("v", s["vn"].double(), s["v"], s["vs"])):
        codes, scale = codes.double(), scale.double()
        pg = s["table"].long()[torch.tensor(req, device=dev), slot // page]
        ids, where = torch.unique(pg, return_inverse=True)
        fill = torch.zeros(len(ids), hk, page, d, dtype=torch.float64, device=dev)
        fill[where, :, slot % page] = x
        new = torch.zeros(len(ids), page, dtype=torch.bool, device=dev)
        new[where, slot % page] = True
        old = torch.zeros(len(ids), page, dtype=torch.bool, device=dev)
        start = torch.tensor(ln, device=dev)
        first = torch.searchsorted(ids, s["table"].long()[torch.arange(len(ln), device=dev), start // page])
        old[first] = torch.arange(page, device=dev)[None] < (start % page)[:, None]
        need = torch.exp2(torch.ceil(torch.log2(fill.abs().amax((2, 3)) / 448)).clamp(-64, 64))
        need = torch.where(old.any(1)[:, None], torch.maximum(need, scale[ids]), need)
        kept = _nearest_e4m3(codes[ids] * (scale[ids] / need)[:, :, None, None])
        made = _nearest_e4m3(fill / need[:, :, None, None])
        keep = torch.where(old[:, None, :, None], kept, codes[ids])
        codes[ids] = torch.where(new[:, None, :, None], made, keep)
        scale[ids] = need
        out[name], out[name + "_scale"] = codes, scale
    return {k: out[k] for k in ("q", "len", "k", "v", "k_scale", "v_scale")}
