"""What the tree-verify operators are measured on: cases, inputs, plain forms and 64-bit values.

One round of speculative decoding with a drafted tree runs four operators: rotary positions with
the cache append (``rope``), attention of the tree's nodes over the cache (``attn``), verification
of the drafted tokens against the target's probabilities from given random numbers
(``accept``), and keeping the accepted path in the cache (``keep``). Every case is one call of
one of them. The plain forms are elementary torch operations in 32 bits; with ``own`` set, the
calls are those of the package.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ------------------------------------------------------------------------------- cases

def listed():
    return [
        # one decoded token of the 32/8-head, head_dim 128 target: latency
        {"name": "rope-one-token", "op": "rope", "batch": 1, "rows": 1, "hq": 32, "hk": 8, "d": 128,
         "rot": 128, "layout": "half", "scaling": "none", "norm": True, "pos": 2047, "type": "bf16"},
        # a batch of drafted trees on a head_dim 256 target with a rotated quarter of the head
        {"name": "rope-partial-trees", "op": "rope", "batch": 33, "rows": 1013, "hq": 24, "hk": 4,
         "d": 256, "rot": 64, "layout": "interleaved", "scaling": "none", "norm": False, "pos": 16000,
         "type": "f16"},
        # a long prompt's rows far out in a context stretched four times
        {"name": "rope-long-context", "op": "rope", "batch": 1, "rows": 16389, "hq": 32, "hk": 8,
         "d": 128, "rot": 128, "layout": "half", "scaling": "yarn", "norm": False, "pos": 100000,
         "type": "bf16"},
        # plain decoding, one row at 2k of context: latency
        {"name": "attn-one-token", "op": "attn", "batch": 1, "nodes": 1, "len": 2048, "ragged": False,
         "hq": 32, "hk": 8, "d": 128, "type": "bf16"},
        # one user's 61-node tree at 16k of context
        {"name": "attn-tree-16k", "op": "attn", "batch": 1, "nodes": 61, "len": 16411, "ragged": False,
         "hq": 32, "hk": 8, "d": 128, "type": "bf16"},
        # a serving batch: trees of 1 to 48 nodes, contexts of 256 to 16k
        {"name": "attn-serving-batch", "op": "attn", "batch": 64, "nodes": 48, "len": 16384,
         "ragged": True, "hq": 32, "hk": 8, "d": 128, "type": "bf16"},
        # big trees over a 64/8-head target at 32k: bound by the matrix products
        {"name": "attn-big-trees-32k", "op": "attn", "batch": 2, "nodes": 384, "len": 32768,
         "ragged": False, "hq": 64, "hk": 8, "d": 128, "type": "f16"},
        # four drafted tokens found by lookup (no draft distribution), one user: latency
        {"name": "accept-lookup-block", "op": "accept", "batch": 1, "nodes": 5, "ragged": False,
         "vocab": 151936, "tree": False, "draft": False, "type": "bf16"},
        # trees of up to 61 nodes, 16 users, 32-bit logits
        {"name": "accept-trees", "op": "accept", "batch": 16, "nodes": 61, "ragged": True,
         "vocab": 151936, "tree": True, "draft": False, "type": "f32"},
        # the continuous batch: 256 users, blocks of up to 16 rows, a drafter's own distribution
        {"name": "accept-serving-batch", "op": "accept", "batch": 256, "nodes": 16, "ragged": True,
         "vocab": 151936, "tree": False, "draft": True, "type": "bf16"},
        # one user's accepted path in every layer of the 36-layer target
        {"name": "keep-one-user", "op": "keep", "batch": 1, "nodes": 61, "path": 6, "layers": 36,
         "hk": 8, "d": 128, "cap": 2304, "type": "bf16"},
        # the serving batch's accepted paths
        {"name": "keep-serving-batch", "op": "keep", "batch": 64, "nodes": 64, "path": 9, "layers": 36,
         "hk": 8, "d": 128, "cap": 192, "type": "bf16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "attn", "attn", "accept", "accept", "keep"])
    t = rng.choice(["bf16", "f16"])
    if op == "rope":
        d = rng.choice([64, 128, 128, 256])
        rows = _log(rng, 1, 8000)
        hq, hk = rng.choice([(32, 8), (24, 4), (8, 8), (16, 2), (64, 8)])
        return {"op": op, "batch": min(rows, _log(rng, 1, 64)), "rows": rows, "hq": hq, "hk": hk,
                "d": d, "rot": rng.choice([d, d, d // 2, d // 4]),
                "layout": rng.choice(["half", "interleaved"]),
                "scaling": rng.choice(["none", "linear", "ntk", "yarn", "llama3"]),
                "norm": rng.random() < 0.4, "pos": _log(rng, 1, 120000), "type": t}
    if op == "attn":
        hq, hk = rng.choice([(32, 8), (64, 8), (8, 8), (16, 2), (24, 8), (20, 4), (12, 4)])
        ln = _log(rng, 1, 32768)
        batch = _log(rng, 1, 64)
        nodes = _log(rng, 1, 300)
        while 4.0 * batch * nodes * hq * ln > 1.0e11 / 32:
            batch, nodes = max(1, batch * 2 // 3), max(1, nodes * 2 // 3)
        return {"op": op, "batch": batch, "nodes": nodes, "len": max(ln, nodes),
                "ragged": rng.random() < 0.6, "hq": hq, "hk": hk, "d": rng.choice([64, 128, 128]),
                "type": t}
    if op == "accept":
        tree = rng.random() < 0.4
        return {"op": op, "batch": _log(rng, 1, 64), "nodes": _log(rng, 1, 32),
                "ragged": rng.random() < 0.7, "vocab": _log(rng, 500, 152000), "tree": tree,
                "draft": not tree and rng.random() < 0.6, "type": rng.choice(["bf16", "f16", "f32"])}
    nodes = _log(rng, 1, 200)
    return {"op": op, "batch": _log(rng, 1, 32), "nodes": nodes, "path": rng.randint(1, min(nodes, 16)),
            "layers": rng.choice([2, 16, 36, 64]), "hk": rng.choice([2, 4, 8]),
            "d": rng.choice([64, 128, 256]), "cap": nodes + _log(rng, 1, 100), "type": t}


# ------------------------------------------------------------------------------- shapes of a case

def _shape_rng(case):
    """The ragged sizes belong to the case, not to the seed."""
    key = "/".join("%s=%s" % kv for kv in sorted(case.items()) if kv[0] != "name")
    return random.Random(key)


def _counts(case):
    """Rows of each request."""
    r, B = _shape_rng(case), case["batch"]
    if case["op"] == "rope":
        cuts = sorted(r.sample(range(1, case["rows"]), B - 1)) if B > 1 else []
        edges = [0] + cuts + [case["rows"]]
        return [b - a for a, b in zip(edges, edges[1:])]
    if case.get("ragged"):
        return [case["nodes"]] + [r.randint(1, case["nodes"]) for _ in range(B - 1)]
    return [case["nodes"]] * B


def _lens(case, counts):
    """Keys of each request, its tree's nodes among them."""
    r = random.Random(_shape_rng(case).random())
    if not case["ragged"]:
        return [case["len"]] * case["batch"]
    lo = min(256, case["len"])
    return [case["len"]] + [max(n, _log(r, lo, case["len"])) for n in counts[1:]]


def _parents(case, counts):
    """Parent of each node within its request, -1 for the first; a chain's is its neighbour."""
    r, out = random.Random(_shape_rng(case).random() + 1), []
    for n in counts:
        if case["op"] == "accept" and not case["tree"]:
            out.append(list(range(-1, n - 1)))
        else:
            out.append([-1] + [r.randint(max(0, (i - 1) // 3 - 1), (i - 1) // 2) for i in range(1, n)])
    return out


def _paths(case):
    """Ascending nodes of an accepted path, beginning with the first node."""
    r, out = _shape_rng(case), []
    for b in range(case["batch"]):
        n = case["path"] if b == 0 else r.randint(1, case["path"])
        out.append([0] + sorted(r.sample(range(1, case["nodes"]), n - 1)))
    return out


def _anc_words(parents, words):
    """Bits of each node and its ancestors, as rows of 32-bit words."""
    rows = []
    for par in parents:
        bits = []
        for i, p in enumerate(par):
            bits.append((1 << i) | (bits[p] if p >= 0 else 0))
        rows += [[(b >> (32 * w)) & 0xFFFFFFFF for w in range(words)] for b in bits]
    return [[v - (1 << 32) if v >= 1 << 31 else v for v in row] for row in rows]


def _size(case):
    return 4 if case["type"] == "f32" else 2


def work(case):
    e = _size(case)
    if case["op"] == "rope":
        vals = case["rows"] * (case["hq"] + 2 * case["hk"]) * case["d"]
        return {"bytes": 2 * e * vals, "flops": 6 * vals}
    if case["op"] == "attn":
        n = _counts(case)
        ln = _lens(case, n)
        by = sum(2 * e * x * case["hk"] * case["d"] for x in ln)
        by += sum(2 * e * r * case["hq"] * case["d"] for r in n)
        return {"bytes": by, "flops": sum(4 * r * x for r, x in zip(n, ln)) * case["hq"] * case["d"]}
    if case["op"] == "accept":
        par = _parents(case, _counts(case))
        inner = sum(len(set(p) - {-1}) for p in par)
        rows = inner + case["batch"] if inner else case["batch"]
        by = rows * case["vocab"] * e + case["batch"] * case["vocab"] * (4 + (2 if case["draft"] else 0))
        return {"bytes": by, "flops": 4 * rows * case["vocab"]}
    moved = sum(sum(1 for i, x in enumerate(p) if x != i) for p in _paths(case))
    by = 4 * e * moved * case["layers"] * case["hk"] * case["d"]
    return {"bytes": by + 8 * case["batch"] * case["path"], "flops": 0}


# ------------------------------------------------------------------------------- inputs

def _inv_freq(case):
    """Rotary frequencies in 64 bits and the factor on the rotated values."""
    rot, kind, base, f = case["rot"], case["scaling"], 1e6, 4.0
    i = torch.arange(0, rot, 2, dtype=torch.float64)
    if kind == "ntk":
        base = base * f ** (rot / max(rot - 2, 1))
    inv = base ** (-i / rot)
    if kind == "linear":
        return inv / f, 1.0
    if kind == "yarn":
        def at(turns):
            return rot * math.log(32768 / (turns * 2 * math.pi)) / (2 * math.log(base))
        lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
        ramp = ((torch.arange(rot // 2, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        return inv / f * ramp + inv * (1 - ramp), 0.1 * math.log(f) + 1.0
    if kind == "llama3":
        wave, old = 2 * math.pi / inv, 8192.0
        s = ((old / wave - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return (1 - s) * inv / f + s * inv, 1.0
    return inv, 1.0


_SCALING = {"none": None, "linear": {"type": "linear", "factor": 4.0},
            "ntk": {"type": "ntk", "factor": 4.0},
            "yarn": {"type": "yarn", "factor": 4.0, "original_max_position": 32768},
            "llama3": {"type": "llama3", "factor": 4.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
                       "original_max_position": 8192}}


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    dt = DTYPES[case["type"]]
    i32 = dict(dtype=torch.int32, device=dev)
    s = {"case": case, "op": case["op"]}

    def randn(*shape, dtype=dt):
        return torch.randn(shape, device=dev, generator=g, dtype=torch.float32).to(dtype)

    def cu(n):
        return torch.tensor([0] + list(torch.tensor(n).cumsum(0).tolist()), **i32)

    if case["op"] == "rope":
        n, R = _counts(case), case["rows"]
        hq, hk, d = case["hq"], case["hk"], case["d"]
        qkv = randn(R, (hq + 2 * hk) * d)  # the projection's product, split without copies
        s["q"] = qkv[:, : hq * d].view(R, hq, d)
        s["k"] = qkv[:, hq * d : (hq + hk) * d].view(R, hk, d)
        s["v"] = qkv[:, (hq + hk) * d :].view(R, hk, d)
        at = [i for k in n for i in range(k)]
        s["pos"] = torch.tensor([case["pos"] + i for i in at], **i32)
        s["slot"] = torch.tensor([3 + i for i in at], **i32)
        s["req"] = torch.tensor([b for b, k in enumerate(n) for _ in range(k)], **i32)
        cap = max(n) + 8
        s["kc"] = torch.zeros(case["batch"], hk, cap, d, dtype=dt, device=dev)
        s["vc"] = torch.zeros_like(s["kc"])
        s["qn"] = (1 + 0.1 * randn(d, dtype=torch.float32)).to(dt) if case["norm"] else None
        s["kn"] = (1 + 0.1 * randn(d, dtype=torch.float32)).to(dt) if case["norm"] else None
        inv, s["m"] = _inv_freq(case)
        s["inv"] = inv.to(device=dev, dtype=torch.float32)
        s["out"] = torch.empty(R, hq, d, dtype=dt, device=dev)
        if own:
            from mlx_dspark_b200 import rope
            s["table"] = rope.RopeTable(d, case["rot"], theta=1e6, layout=case["layout"],
                                        scaling=_SCALING[case["scaling"]], device=dev)
    elif case["op"] == "attn":
        n = _counts(case)
        ln = _lens(case, n)
        B, cap = case["batch"], max(ln) + 3
        s["q"] = randn(sum(n), case["hq"], case["d"])
        s["kc"] = torch.empty(B, case["hk"], cap, case["d"], dtype=dt, device=dev).normal_(generator=g)
        s["vc"] = torch.empty(B, case["hk"], cap, case["d"], dtype=dt, device=dev).normal_(generator=g)
        s["cu"], s["len"] = cu(n), torch.tensor(ln, **i32)
        s["nodes"], s["max_len"] = max(n), max(ln)
        s["anc"] = torch.tensor(_anc_words(_parents(case, n), (max(n) + 31) // 32), **i32)
        s["out"] = torch.empty_like(s["q"])
    elif case["op"] == "accept":
        n = _counts(case)
        par = _parents(case, n)
        B, R, V = case["batch"], sum(n), case["vocab"]
        s["cu"] = cu(n)
        s["parent"] = torch.tensor([p for x in par for p in x], **i32) if case["tree"] else None
        s["anc"] = torch.tensor(_anc_words(par, (max(n) + 31) // 32), **i32) if case["tree"] else None
        s["nodes"] = max(n)
        req = torch.tensor([b for b, k in enumerate(n) for _ in range(k)], device=dev)
        up = torch.tensor([p for x in par for p in x], device=dev).clamp(min=0) + s["cu"].long()[req]
        logits = 3 * torch.randn(R, V, device=dev, generator=g)
        favoured = torch.randint(V, (R, 4), device=dev, generator=g)
        logits.scatter_(1, favoured, 14 + 2 * torch.rand(R, 4, device=dev, generator=g))
        s["draft"] = None
        if case["draft"]:  # a drafter near the target: its tokens are drawn from its distribution
            q = torch.randn(R, V, device=dev, generator=g).mul_(0.7).add_(logits)
            q = torch.softmax(q, -1).to(torch.bfloat16)
            e = torch.empty(R, V, device=dev).exponential_(generator=g)
            s["draft"] = q
            ids = (q.float() / e).argmax(-1)[up]
        else:  # proposals without a distribution: mostly the target's own favourites
            pick = torch.randint(4, (R,), device=dev, generator=g)
            ids = favoured[up, pick]
        s["ids"] = ids.to(torch.int32)
        s["logits"] = logits.to(dt)
        del logits
        s["u"] = torch.rand(R, device=dev, generator=g)
        s["noise"] = torch.empty(B, V, device=dev).exponential_(generator=g)
        t = 0.5 + torch.rand(B, device=dev, generator=g)
        if B > 2:
            t[1] = 0.0  # a greedy user in the batch
        s["temp"] = t
        s["lens0"] = torch.tensor([1000 + k for k in n], **i32)
        s["lens"] = s["lens0"].clone()
        s["out"] = {"n": torch.empty(B, **i32), "next": torch.empty(B, **i32),
                    "prob": torch.empty(R, device=dev), "path": torch.empty(R, **i32)}
    else:
        p = _paths(case)
        n = [case["nodes"]] * case["batch"]
        s["cu"] = cu(n)
        path = torch.full((case["batch"], case["nodes"]), -1, dtype=torch.int32)
        for b, x in enumerate(p):
            path[b, : len(x)] = torch.tensor(x, dtype=torch.int32)
        s["path"] = path.reshape(-1).to(dev)
        s["n"] = torch.tensor([len(x) - 1 for x in p], **i32)
        base = case["cap"] - case["nodes"]
        s["lens"] = torch.tensor([base + len(x) for x in p], **i32)
        shape = (case["layers"], case["batch"], case["hk"], case["cap"], case["d"])
        s["kc"] = torch.empty(shape, dtype=dt, device=dev).normal_(generator=g)
        s["vc"] = torch.empty(shape, dtype=dt, device=dev).normal_(generator=g)
        s["longest"] = case["path"]
        if own:
            from mlx_dspark_b200 import tree
            s["keeper"] = tree.PathKeeper(list(s["kc"].unbind(0)), list(s["vc"].unbind(0)))
    return s


# ------------------------------------------------------------------------------- one pass

def run(s):
    return (_run_own if own else _run_plain)[s["op"]](s)


def _own_rope(s):
    from mlx_dspark_b200 import rope
    q = rope.rope_append(s["q"], s["k"], s["v"], s["table"], s["pos"], s["kc"], s["vc"], s["slot"],
                         row_req=s["req"], q_norm=s["qn"], k_norm=s["kn"], eps=1e-6, q_out=s["out"])
    return {"q": q, "k_cache": s["kc"], "v_cache": s["vc"]}


def _own_attn(s):
    from mlx_dspark_b200 import tree
    return tree.tree_sdpa(s["q"], s["kc"], s["vc"], s["cu"], s["len"], s["anc"],
                          scale=s["case"]["d"] ** -0.5, max_nodes=s["nodes"], out=s["out"])


def _own_accept(s):
    from mlx_dspark_b200 import sampling
    s["lens"].copy_(s["lens0"])
    r = sampling.sample_accept(s["logits"], s["ids"], s["cu"], s["u"], s["noise"],
                               temperature=s["temp"], draft_probs=s["draft"], parent=s["parent"],
                               max_rows=s["nodes"], lens=s["lens"], out=s["out"])
    return {"n": r["n"], "next": r["next"], "prob": r["prob"], "path": r["path"], "lens": s["lens"]}


def _own_keep(s):
    s["keeper"].keep(s["path"], s["cu"], s["n"], s["lens"])
    return {"k": s["kc"], "v": s["vc"]}


_run_own = {"rope": _own_rope, "attn": _own_attn, "accept": _own_accept, "keep": _own_keep}


def _plain_rope(s):
    c = s["case"]
    rot, half = c["rot"], c["rot"] // 2
    a = s["pos"].float()[:, None, None] * s["inv"]
    cos, sin = torch.cos(a) * s["m"], torch.sin(a) * s["m"]

    def turn(x, w):
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

    s["out"].copy_(turn(s["q"], s["qn"]))
    at = (s["req"].long()[:, None], torch.arange(c["hk"], device=s["q"].device)[None], s["slot"].long()[:, None])
    s["kc"][at] = turn(s["k"], s["kn"]).to(s["kc"].dtype)
    s["vc"][at] = s["v"]
    return {"q": s["out"], "k_cache": s["kc"], "v_cache": s["vc"]}


def _rows(cu, R):
    """Request and place within it of each packed row."""
    r = torch.arange(R, device=cu.device, dtype=torch.int32)
    req = torch.searchsorted(cu, r, right=True) - 1
    return req, r.long() - cu.long()[req]


def _plain_attn(s):
    c = s["case"]
    B, hk, d, L, N = c["batch"], c["hk"], c["d"], s["max_len"], s["nodes"]
    G, R, dev = c["hq"] // hk, s["q"].shape[0], s["q"].device
    cu = s["cu"].long()
    i = torch.arange(N, device=dev)
    row = (cu[:-1, None] + i).clamp(max=R - 1)
    q = s["q"][row].float().view(B, N, hk, G, d).permute(0, 2, 3, 1, 4).reshape(B, hk, G * N, d)
    k, v = s["kc"][:, :, :L].float(), s["vc"][:, :, :L].float()
    first = s["len"].long() - (cu[1:] - cu[:-1])  # keys before the tree
    off = torch.arange(L, device=dev)[None] - first[:, None]
    words = s["anc"][row].long() & 0xFFFFFFFF
    bit = off.clamp(0, N - 1)
    seen = torch.gather(words, 2, (bit >> 5)[:, None].expand(B, N, L)) >> (bit & 31)[:, None] & 1
    seen = (seen.bool() & (off < (cu[1:] - cu[:-1])[:, None])[:, None]) | (off < 0)[:, None]
    z = torch.matmul(q, k.transpose(2, 3)).mul_(d ** -0.5).view(B, hk, G, N, L)
    z.masked_fill_(~seen[:, None, None], -math.inf)
    m = z.amax(-1, keepdim=True)
    p = z.sub_(torch.where(torch.isinf(m), torch.zeros_like(m), m)).exp_()
    t = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, hk, G * N, L), v).view(B, hk, G, N, d) / torch.where(t == 0, torch.ones_like(t), t)
    req, at = _rows(s["cu"], R)
    s["out"].copy_(o.permute(0, 3, 1, 2, 4).reshape(B, N, hk * G, d)[req, at])
    return s["out"]


def _plain_accept(s):
    R, V = s["logits"].shape
    B, N, dev, cu = s["cu"].numel() - 1, s["nodes"], s["logits"].device, s["cu"].long()
    req, at = _rows(s["cu"], R)
    ids, rows = s["ids"].long(), cu[1:] - cu[:-1]
    t = s["temp"][req][:, None]
    z = s["logits"].float()
    m = z.amax(-1, keepdim=True)
    e = torch.exp((z - m) / torch.where(t == 0, torch.ones_like(t), t))
    p = e / e.sum(-1, keepdim=True)
    top = torch.arange(V, device=dev)[None] == z.argmax(-1, keepdim=True)
    p = torch.where(t == 0, top.float(), p)
    del z, e, top
    local = s["parent"].long() if s["parent"] is not None else at - 1
    up = (local.clamp(min=0) + cu[req])
    prob = torch.where(local < 0, torch.ones_like(s["u"]), p[up, ids])
    place = torch.arange(N, device=dev)
    grid = (cu[:-1, None] + place).clamp(max=R - 1)  # [B, N] rows, those beyond the block dropped below
    there = place < rows[:, None]
    s["lens"].copy_(s["lens0"])
    if s["parent"] is None:
        q = torch.ones_like(prob) if s["draft"] is None else s["draft"][up, ids].float()
        q = torch.where(t[:, 0] == 0, torch.ones_like(q), q)
        ok = (s["u"][up] * q < prob) | (local < 0)
        kept = torch.cumprod((ok[grid] & there).long(), 1).bool()
    else:
        lp = torch.where(there, local[grid], -2)
        tok, pr = ids[grid], prob[grid]
        older = (lp[:, :, None] == lp[:, None, :]) & (place[None, :] < place[:, None])  # [B, node, sibling]
        twin = (older & (tok[:, :, None] == tok[:, None, :])).any(-1)
        share = torch.where(twin, torch.zeros_like(pr), pr)
        before = (older * share[:, None, :]).sum(-1)
        u = s["u"][up][grid]
        ok = (~twin & (u >= before) & (u < before + pr)) | (lp == -1)
        w = s["anc"][grid].long() & 0xFFFFFFFF
        above = (torch.gather(w, 2, (place >> 5)[None, None].expand(B, N, N)) >> (place & 31)) & 1
        kept = there & ~((above == 1) & ~ok[:, None, :]).any(-1)
    n = kept.long().sum(1) - 1
    last = torch.where(kept, place, -1).amax(1) + cu[:-1]
    best = p[last]
    rest = best
    if s["draft"] is not None:
        short = (n < rows - 1) & (s["temp"] != 0)
        rest = torch.where(short[:, None], (best - s["draft"][last].float()).clamp(min=0), best)
    elif s["parent"] is not None or R:
        mine = there & (up[grid] == last[:, None]) & (local[grid] >= 0)
        tried = torch.zeros(B, V, device=dev).scatter_add_(1, ids[grid], mine.float()) > 0
        rest = torch.where(tried, torch.zeros_like(best), best)
    rest = torch.where(rest.amax(1, keepdim=True) > 0, rest, best)
    nxt = (rest / s["noise"]).argmax(1)
    order = torch.where(kept, place, N + place).sort(1).values
    path = torch.where(order < N, order, -1)
    o = s["out"]
    o["n"].copy_(n)
    o["next"].copy_(nxt)
    o["prob"].copy_(prob)
    o["path"].copy_(path[req, at])
    s["lens"].sub_((rows - 1 - n).to(torch.int32))
    return {"n": o["n"], "next": o["next"], "prob": o["prob"], "path": o["path"], "lens": s["lens"]}


def _plain_keep(s):
    c = s["case"]
    B, dev, P = c["batch"], s["kc"].device, s["longest"]
    base = (s["lens"] - s["n"] - 1).long()[:, None]
    i = torch.arange(P, device=dev)[None]
    path = s["path"].view(B, -1)[:, :P].long()
    src = base + torch.where(i <= s["n"].long()[:, None], path, i)
    b = torch.arange(B, device=dev)[:, None]
    s["kc"][:, b, :, base + i] = s["kc"][:, b, :, src]
    s["vc"][:, b, :, base + i] = s["vc"][:, b, :, src]
    return {"k": s["kc"], "v": s["vc"]}


_run_plain = {"rope": _plain_rope, "attn": _plain_attn, "accept": _plain_accept, "keep": _plain_keep}


# ------------------------------------------------------------------------------- 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        rot, kind, R = case["rot"], case["scaling"], case["rows"]
        freq, gain = [], 1.0
        for j in range(rot // 2):
            f = 1e6 ** (-2 * j / rot)
            if kind == "linear":
                f /= 4
            elif kind == "ntk":
                f = (1e6 * 4 ** (rot / (rot - 2))) ** (-2 * j / rot)
            elif kind == "yarn":
                first, last = (rot * math.log(32768 / (b * 2 * math.pi)) / (2 * math.log(1e6)) for b in (32, 1))
                first, last = max(math.floor(first), 0), min(math.ceil(last), rot - 1)
                r = min(max((j - first) / max(last - first, 1e-3), 0.0), 1.0)
                f, gain = f * (r / 4 + 1 - r), 0.1 * math.log(4) + 1
            elif kind == "llama3":
                w = 2 * math.pi / f
                if w > 8192:
                    f /= 4
                elif w > 8192 / 4:
                    h = (8192 / w - 1) / 3
                    f = (1 - h) * f / 4 + h * f
            freq.append(f)
        z = torch.polar(torch.full((R, 1, rot // 2), gain, device="cuda", dtype=torch.float64),
                        s["pos"].double()[:, None, None] * torch.tensor(freq, device="cuda", dtype=torch.float64))

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

        kc, vc = s["kc"].double(), s["vc"].double()
        k = turned(s["k"], s["kn"])
        for h in range(case["hk"]):
            kc[s["req"].long(), h, s["slot"].long()] = k[:, h]
            vc[s["req"].long(), h, s["slot"].long()] = s["v"][:, h].double()
        return {"q": turned(s["q"], s["qn"]), "k_cache": kc, "v_cache": vc}
    if case["op"] == "attn":
        n = _counts(case)
        ln, par = _lens(case, n), _parents(case, n)
        if sum(4.0 * a * b for a, b in zip(n, ln)) * case["hq"] * case["d"] > 5e12:
            return None
        out, r0, G = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), 0, case["hq"] // case["hk"]
        for b in range(case["batch"]):
            sees = torch.ones(n[b], ln[b], dtype=torch.bool)
            sees[:, ln[b] - n[b] :] = False
            for i in range(n[b]):
                j = i
                while j >= 0:
                    sees[i, ln[b] - n[b] + j] = True
                    j = par[b][j]
            sees = sees.to("cuda")
            for h in range(case["hk"]):
                q = s["q"][r0 : r0 + n[b], h * G : (h + 1) * G].double().transpose(0, 1)
                z = q @ s["kc"][b, h, : ln[b]].double().T * case["d"] ** -0.5
                w = torch.softmax(z.masked_fill(~sees, -math.inf), -1)
                out[r0 : r0 + n[b], h * G : (h + 1) * G] = (w @ s["vc"][b, h, : ln[b]].double()).transpose(0, 1)
            r0 += n[b]
        return out
    if case["op"] == "accept":
        n = _counts(case)
        prob, r0 = torch.ones(sum(n), dtype=torch.float64, device="cuda"), 0
        for b, par in enumerate(_parents(case, n)):
            lg, t = s["logits"][r0 : r0 + n[b]].double(), float(s["temp"][b])
            if n[b] > 1:
                up = torch.tensor(par[1:], device="cuda")
                tok = s["ids"][r0 + 1 : r0 + n[b]].long()
                if t == 0:
                    prob[r0 + 1 : r0 + n[b]] = (lg.argmax(-1)[up] == tok).double()
                else:
                    prob[r0 + 1 : r0 + n[b]] = torch.log_softmax(lg / t, -1)[up, tok].exp()
            r0 += n[b]
        return {"n": None, "next": None, "prob": prob, "path": None, "lens": None}
    kc, vc, old = s["kc"].double(), s["vc"].double(), s["kc"]
    for b, p in enumerate(_paths(case)):
        at = case["cap"] - case["nodes"]
        for i, x in enumerate(p):
            kc[:, b, :, at + i] = old[:, b, :, at + x].double()
            vc[:, b, :, at + i] = s["vc"][:, b, :, at + x].double()
    return {"k": kc, "v": vc}
