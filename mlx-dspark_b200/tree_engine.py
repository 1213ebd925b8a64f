"""Rounds with drafted trees over a :class:`~.target.Target`'s request slots.

:class:`TreeSpec` is the tree counterpart of :class:`~.batch_engine.SpecBatch` (the reference's tree
rounds, src/mlx_dspark/tree.py, for one request; here any number of slots with trees of any size):
one :meth:`~TreeSpec.step` packs the slots' trees, runs one verify forward over all their nodes, accepts
against the target's probabilities (greedy at temperature 0), keeps the accepted path in every layer's
cache and leaves each slot as plain decoding of the accepted tokens would have. Everything but the
projections of the forward is one of the tree-round operators (:mod:`.rope`, :mod:`.tree`,
:mod:`.sampling`), and nothing in a step waits for the device.
"""

from __future__ import annotations

import ctypes as C

import torch

from . import _lib, sampling, tree
from ._torch import int32, on_device, ptr
from .rope import RopeTable


class TreeSpec:
    """``max_nodes`` bounds the nodes of a slot's tree (its root, the pending token, among them; up to 1024
    in :meth:`step`, the accept's limit); a step holds up to ``target.max_rows`` nodes. ``rope`` replaces
    the target's rotary form (default: its own)."""

    def __init__(self, target, max_nodes: int, *, rope: RopeTable | None = None):
        t, c = target, target.cfg
        self.t, self.max_nodes, self.B = t, int(max_nodes), t.slots
        dev = t.device
        self.rope = rope or RopeTable(c.head_dim, theta=c.rope_theta, device=dev)
        if self.rope.head_dim != c.head_dim:
            raise _lib.DSparkError(_lib.ERR_ARG, f"rope head_dim {self.rope.head_dim}, the target's {c.head_dim}")
        self.lens = torch.zeros(self.B, dtype=torch.int32, device=dev)  # tokens cached per slot
        layers = [("k_cache", []), ("v_cache", [])]
        for name, out in layers:
            for layer in t.layers:
                pool = layer[name]
                out.append(pool.permute(1, 0, 2)[None] if t.position_major else pool)
        self.k_caches, self.v_caches = layers[0][1], layers[1][1]
        self.keeper = tree.PathKeeper(self.k_caches, self.v_caches)
        self.kv_start = None
        if t.position_major:
            self.kv_start = torch.tensor(t._slot_base, dtype=torch.int32, device=dev)
        self.kv_cap = torch.tensor(t.slot_caps, dtype=torch.int32, device=dev)
        R = t.max_rows
        self.qkv = torch.empty((R, (c.n_heads + 2 * c.n_kv_heads) * c.head_dim), dtype=torch.bfloat16, device=dev)
        n = int(_lib.lib.dspark_tree_attn_workspace(self.B, c.n_heads, c.n_kv_heads, c.head_dim, self.max_nodes))
        self.attn_ws = torch.empty(n, dtype=torch.uint8, device=dev)

    def pack(self, cu_rows: torch.Tensor, parent: torch.Tensor | None, n_rows: int) -> dict:
        """:func:`.tree.pack` of a round over the slots as they are, bounded by each slot's capacity."""
        return tree.pack(cu_rows, parent, self.lens, n_rows, self.max_nodes, kv_start=self.kv_start,
                         kv_cap=self.kv_cap)

    def forward(self, ids: torch.Tensor, meta: dict, cu_rows: torch.Tensor,
                logits: torch.Tensor | None = None) -> torch.Tensor:
        """Logits ``[R, vocab]`` of packed nodes ``ids`` (int32 ``[R]``); appends their K/V at the slots
        that ``meta`` (:meth:`pack` of as many rows) gives. ``logits``: bf16, ``R`` rows of the
        vocabulary or more (default: the target's own, which its next forward writes again)."""
        t, c, R = self.t, self.t.cfg, ids.numel()
        if not 1 <= R <= t.max_rows:
            raise _lib.DSparkUnsupported(_lib.ERR_UNSUPPORTED, f"{R} rows (1..{t.max_rows})")
        stream = on_device(ids, cu_rows, logits, *meta.values())
        if logits is not None and (logits.dtype is not torch.bfloat16 or logits.ndim != 2 or logits.shape[0] < R or
                                   logits.shape[1] != c.vocab or logits.stride(1) != 1 or
                                   (R > 1 and logits.stride(0) < c.vocab)):
            raise _lib.DSparkError(_lib.ERR_ARG, f"logits {logits.dtype} {tuple(logits.shape)}: bf16 [{R}, {c.vocab}] "
                                   "with contiguous rows")
        anc = meta["anc"]
        if anc.ndim != 2 or anc.shape[0] != R:
            raise _lib.DSparkError(_lib.ERR_ARG, f"anc {tuple(anc.shape)} for {R} rows")
        cache = self.k_caches[0]
        fwd = _lib.TreeFwd(
            int32("cu_rows", cu_rows, self.B + 1), int32("row_pos", meta["row_pos"], R),
            int32("row_slot", meta["row_slot"], R), int32("row_req", meta["row_req"], R),
            int32("kv_len_new", meta["kv_len_new"], self.B), ptr(self.kv_start), int32("anc", anc),
            self.rope.freq_ptr, ptr(self.qkv), ptr(self.attn_ws), self.attn_ws.numel(), cache.stride(0),
            self.rope.mscale, anc.shape[1], self.max_nodes, self.rope.layout_code,
            self.rope.rotary_dim, cache.shape[2], cache.shape[0])
        out = t.logits if logits is None else logits
        _lib.check(_lib.lib.dspark_tree_forward(
            C.byref(t._model_c), C.byref(t._buf_c), C.byref(fwd), int32("ids", ids), R, self.B, ptr(out),
            out.stride(0), stream))
        return out[:R]

    def step(self, ids: torch.Tensor, cu_rows: torch.Tensor, u: torch.Tensor, noise: torch.Tensor, *,
             parent: torch.Tensor | None = None, temperature: torch.Tensor | None = None,
             draft_probs: torch.Tensor | None = None) -> dict:
        """One round. ``ids`` int32 ``[R]``: every slot's nodes one slot after the other (``cu_rows``
        int32 ``[slots + 1]``; an idle slot has none), the first of them its pending token; ``parent``
        int32 ``[R]`` as in :func:`.tree.pack` (``None``: chains); ``u``, ``noise``, ``temperature``
        (``None``: greedy here, 1 there) and ``draft_probs`` as in :func:`.sampling.sample_accept`. Returns its
        ``n``, ``next``, ``prob`` and ``path``; ``lens`` and the caches move on to the accepted tokens,
        and ``next`` is each slot's new pending token. Nodes past their slot's capacity are neither cached
        nor accepted, and the device status records them; a slot without room for its pending token stays
        as it is and has ``next`` -1."""
        R = ids.numel()
        if temperature is None:
            temperature = torch.zeros(self.B, device=ids.device)
        meta = self.pack(cu_rows, parent, R)
        lens = meta["kv_len_new"]
        logits = self.forward(ids, meta, cu_rows) if R else self.t.logits[:0]  # (every slot idle)
        out = sampling.sample_accept(logits, ids, cu_rows, u, noise, temperature=temperature,
                                     draft_probs=draft_probs, parent=parent, max_rows=self.max_nodes,
                                     row_limit=meta["room"], lens=lens)
        self.keeper.keep(out["path"], cu_rows, out["n"], lens, kv_start=self.kv_start)
        out["lens"] = self.lens.copy_(lens)  # last: a call refused on the way leaves the slots as they were
        return out
