"""Drafted trees: packing, attention over the cache, and keeping the accepted path.

A verify block is a tree of drafted tokens: its root is the pending token, every other node has a
parent before it. Requests are packed as everywhere in the batch engine (``cu_rows``), with any
number of nodes each. :func:`pack` builds the rows' rotary positions, cache slots and ancestor bits on
the device, :func:`tree_sdpa` is the attention of all rows over their request's cache, and
:class:`PathKeeper` moves the accepted path's K/V rows together in every layer, after which the
cache is what the plain decode of the accepted tokens would have left (the reference's tree rounds,
src/mlx_dspark/tree.py, with its 32-node attention in :mod:`.multirow_attn`).
"""

from __future__ import annotations

import torch

from . import _lib
from ._torch import int32, on_device
from .rope import _dtype, _last_contiguous


def anc_words(max_nodes: int) -> int:
    """32-bit words a row of ancestor bits has for trees of up to ``max_nodes`` nodes."""
    return max(1, (int(max_nodes) + 31) // 32)


def pack(cu_rows: torch.Tensor, parent: torch.Tensor | None, kv_len: torch.Tensor, n_rows: int,
         max_nodes: int, out: dict | None = None) -> dict:
    """Device-side metadata of one packed round: ``row_pos`` (cached tokens + depth), ``row_slot``
    (cached tokens + place), ``row_req``, ``anc`` (int32 ``[R, words]`` bit rows of each node and its
    ancestors) and ``kv_len_new``. ``kv_len`` int32 ``[B]``: tokens cached before the round;
    ``parent`` int32 ``[R]``: places within the request, -1 for the root (``None``: chains)."""
    dev, stream = on_device(cu_rows, parent, kv_len)
    R, B = int(n_rows), kv_len.numel()
    int32("cu_rows", cu_rows, B + 1), int32("kv_len", kv_len), int32("parent", parent, R)
    words = anc_words(max_nodes)
    if out is None:
        e = dict(dtype=torch.int32, device=dev)
        out = {"row_pos": torch.empty(R, **e), "row_slot": torch.empty(R, **e),
               "row_req": torch.empty(R, **e), "anc": torch.empty((R, words), **e),
               "kv_len_new": torch.empty(B, **e)}
    else:
        on_device(cu_rows, *out.values())
        for name, n in (("row_pos", R), ("row_slot", R), ("row_req", R), ("anc", R * words),
                        ("kv_len_new", B)):
            int32(name, out[name], n)
    _lib.check(_lib.lib.dspark_tree_pack(
        cu_rows.data_ptr(), None if parent is None else parent.data_ptr(), kv_len.data_ptr(), B, R,
        out["row_pos"].data_ptr(), out["row_slot"].data_ptr(), out["row_req"].data_ptr(),
        out["anc"].data_ptr(), words, out["kv_len_new"].data_ptr(), stream))
    return out


def tree_sdpa(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, cu_rows: torch.Tensor,
              kv_len: torch.Tensor, anc: torch.Tensor | None = None, *, scale: float,
              max_nodes: int, kv_start: torch.Tensor | None = None,
              out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of packed rows ``q [R, Hq, D]`` over the caches ``[B, Hk, cap, D]``: row i of request
    b sees the ``kv_len[b] - rows(b)`` keys before its tree and, of the tree's keys after them, its
    own ancestors by the bits ``anc[i]`` (int32 ``[R, words]``; ``None``: all places up to its own).
    ``kv_len`` int32 ``[B]`` counts the tree's rows too. A position-major pool is passed as one
    batch entry ``[1, Hk, positions, D]`` with ``kv_start`` int32 ``[B]``. ``max_nodes`` bounds the
    rows of a request. Returns ``out [R, Hq, D]``; a row that sees nothing is zero."""
    dev, stream = on_device(q, k_cache, v_cache, cu_rows, kv_len, anc, kv_start, out)
    if q.ndim != 3 or k_cache.ndim != 4 or k_cache.shape != v_cache.shape:
        raise _lib.DSparkError(_lib.ERR_ARG, "tree_sdpa: q [R, Hq, D], caches [B, Hk, cap, D]")
    R, Hq, D = q.shape
    KB, Hk, cap, Dc = k_cache.shape
    B = cu_rows.numel() - 1
    if Dc != D or Hk == 0 or Hq % Hk:
        raise _lib.DSparkError(_lib.ERR_ARG, f"tree_sdpa: q {tuple(q.shape)}, caches {tuple(k_cache.shape)}")
    if out is None:
        out = torch.empty((R, Hq, D), dtype=q.dtype, device=dev)
    elif out.shape != q.shape:
        raise _lib.DSparkError(_lib.ERR_ARG, f"out {tuple(out.shape)} for {tuple(q.shape)}")
    for name, t in (("q", q), ("out", out), ("k_cache", k_cache), ("v_cache", v_cache)):
        _last_contiguous(name, t)
    dt = _dtype(("q", q), ("k_cache", k_cache), ("v_cache", v_cache), ("out", out))
    int32("cu_rows", cu_rows), int32("kv_len", kv_len, B), int32("kv_start", kv_start, B)
    words = 0
    if anc is not None:
        int32("anc", anc)
        if anc.ndim != 2 or anc.shape[0] != R:
            raise _lib.DSparkError(_lib.ERR_ARG, f"anc {tuple(anc.shape)} for {R} rows")
        words = anc.shape[1]
    n = int(_lib.lib.dspark_tree_attn_workspace(B, Hq, Hk, D, max_nodes))
    ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    a = _lib.TreeAttnArgs(
        q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), q.stride()[:2],
        out.stride()[:2], k_cache.stride()[:3], v_cache.stride()[:3], cu_rows.data_ptr(),
        kv_len.data_ptr(), None if kv_start is None else kv_start.data_ptr(),
        None if anc is None else anc.data_ptr(), None if ws is None else ws.data_ptr(), n, scale, dt,
        words, max_nodes, R, B, Hq, Hk, D, cap, KB)
    _lib.check(_lib.lib.dspark_tree_attn(a, stream))
    return out


class PathKeeper:
    """Keeps accepted paths in the caches of all layers of one model: lists of K and V caches
    ``[B, H, cap, D]`` of one shape, type and stride each. The device arrays of their addresses are
    built once; the caches must stay where they are."""

    def __init__(self, k_caches, v_caches):
        ks, vs = list(k_caches), list(v_caches)
        if not ks or len(ks) != len(vs):
            raise _lib.DSparkError(_lib.ERR_ARG, f"{len(ks)} key caches, {len(vs)} value caches")
        for group in (ks, vs):
            for t in group:
                if (t.shape, t.stride(), t.dtype) != (ks[0].shape, group[0].stride(), ks[0].dtype):
                    raise _lib.DSparkError(_lib.ERR_ARG, "the layers' caches differ in shape, type or stride")
                _last_contiguous("cache", t)
                if t.data_ptr() % 16:
                    raise _lib.DSparkUnsupported(_lib.ERR_UNSUPPORTED, "caches must be 16-byte aligned")
        if ks[0].ndim != 4:
            raise _lib.DSparkError(_lib.ERR_ARG, "caches [B, H, cap, D]")
        self.device, _ = on_device(ks[0], *ks, *vs)
        self.k_caches, self.v_caches = ks, vs
        self.batch, self.heads, self.cap, self.dim = ks[0].shape
        self.elem = ks[0].element_size()
        self._kp = torch.tensor([t.data_ptr() for t in ks], dtype=torch.int64, device=self.device)
        self._vp = torch.tensor([t.data_ptr() for t in vs], dtype=torch.int64, device=self.device)
        self._ks, self._vs = (_lib.i64_array(g[0].stride()[:3]) for g in (ks, vs))

    def keep(self, path: torch.Tensor, cu_rows: torch.Tensor, n_accept: torch.Tensor,
             lens: torch.Tensor, *, kv_start: torch.Tensor | None = None) -> None:
        """With ``base = lens[b] - n_accept[b] - 1`` (``lens`` as the accept left it), move cache row
        ``base + path[cu_rows[b] + i]`` to ``base + i`` for ``i <= n_accept[b]``, in every layer."""
        B = n_accept.numel()
        _, stream = on_device(self._kp, path, cu_rows, n_accept, lens, kv_start)
        int32("path", path), int32("cu_rows", cu_rows, B + 1), int32("n_accept", n_accept)
        int32("lens", lens, B), int32("kv_start", kv_start, B)
        _lib.check(_lib.lib.dspark_kv_keep_path(
            self._kp.data_ptr(), self._vp.data_ptr(), len(self.k_caches), self._ks, self._vs,
            path.data_ptr(), cu_rows.data_ptr(), n_accept.data_ptr(), lens.data_ptr(),
            None if kv_start is None else kv_start.data_ptr(), B, self.heads, self.dim, self.elem,
            self.cap, self.batch, stream))
