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

import functools

import torch

from . import _lib
from ._torch import int32, on_device
from .rope import _dtype, _strides

_pack_attn = _lib.packer(_lib.TreeAttnArgs)


@functools.lru_cache(maxsize=4096)
def _workspace(B: int, Hq: int, Hk: int, D: int, max_nodes: int, device: int) -> int:
    return _lib.lib.dspark_tree_attn_workspace(B, Hq, Hk, D, max_nodes)


def anc_words(max_nodes: int) -> int:
    """32-bit words a row of ancestor bits has for trees of up to ``max_nodes`` nodes."""
    return max(1, (int(max_nodes) + 31) // 32)


def pack(cu_rows: torch.Tensor, parent: torch.Tensor | None, kv_len: torch.Tensor, n_rows: int,
         max_nodes: int, kv_start: torch.Tensor | None = None, out: dict | None = None,
         kv_cap: torch.Tensor | None = None) -> dict:
    """Device-side metadata of one packed round: ``row_pos`` (cached tokens + depth), ``row_slot``
    (cached tokens + place), ``row_req``, ``anc`` (int32 ``[R, words]`` bit rows of each node and its
    ancestors) and ``kv_len_new``. ``kv_len`` int32 ``[B]``: tokens cached before the round;
    ``parent`` int32 ``[R]``: places within the request, -1 for the root (``None``: chains).
    With ``kv_start`` (a position-major pool) the slots count from it and ``row_req`` is 0. With ``kv_cap``
    (int32 ``[B]``: positions each request may fill) rows past it have slot -1, and ``room`` (``[B]``)
    tells how many rows fit. Rows behind the last request's are nobody's: position 0, slot and request
    -1, no bits."""
    stream = on_device(cu_rows, parent, kv_len, kv_start, kv_cap)
    R, B = int(n_rows), kv_len.numel()
    words = anc_words(max_nodes)
    if out is None:
        e = dict(dtype=torch.int32, device=cu_rows.device)
        out = {"row_pos": torch.empty(R, **e), "row_slot": torch.empty(R, **e),
               "row_req": torch.empty(R, **e), "anc": torch.empty((R, words), **e),
               "kv_len_new": torch.empty(B, **e)}
        if kv_cap is not None:
            out["room"] = torch.empty(B, **e)
    else:
        on_device(cu_rows, *out.values())
    at = {k: int32(k, out[k], n) for k, n in (("row_pos", R), ("row_slot", R), ("row_req", R),
                                              ("anc", R * words), ("kv_len_new", B))}
    _lib.check(_lib.lib.dspark_tree_pack_capped(
        int32("cu_rows", cu_rows, B + 1), int32("parent", parent, R), int32("kv_len", kv_len),
        int32("kv_start", kv_start, B), int32("kv_cap", kv_cap, B), B, R, at["row_pos"], at["row_slot"],
        at["row_req"], at["anc"], words, at["kv_len_new"], int32("room", out.get("room"), B), stream))
    return out


def tree_sdpa(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, cu_rows: torch.Tensor,
              kv_len: torch.Tensor, anc: torch.Tensor | None = None, *, scale: float,
              max_nodes: int, kv_start: torch.Tensor | None = None,
              out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of packed rows ``q [R, Hq, D]`` over the caches ``[B, Hk, cap, D]``: row i of request
    b sees the ``kv_len[b] - rows(b)`` keys before its tree and, of the tree's keys after them, its
    own ancestors by the bits ``anc[i]`` (int32 ``[R, words]``; ``None``: all places up to its own).
    ``kv_len`` int32 ``[B]`` counts the tree's rows too. A position-major pool is passed as one
    batch entry ``[1, Hk, positions, D]`` with ``kv_start`` int32 ``[B]``. ``max_nodes`` (1 or more) bounds
    the rows of a request. Returns ``out [R, Hq, D]``; a row that sees nothing is zero, a row of no request
    is not written. For up to 32 nodes, as many in every request, :func:`.multirow_attn.multirow_sdpa` with
    ``tree_anc`` is the faster one up to 2k keys (one request, 32/8 heads of 128: 8 to 13 us for 14 to 15)
    and for up to 8 nodes up to 16k; from 16 nodes and 8k keys on this one is (32 nodes over 32k: 39 us
    for 78)."""
    stream = on_device(q, k_cache, v_cache, cu_rows, kv_len, anc, kv_start, out)
    shape, cache = q.shape, k_cache.shape
    if len(shape) != 3 or len(cache) != 4 or v_cache.shape != cache:
        raise _lib.DSparkError(_lib.ERR_ARG, "tree_sdpa: q [R, Hq, D], caches [B, Hk, cap, D]")
    R, Hq, D = shape
    KB, Hk, cap, Dc = cache
    B = cu_rows.numel() - 1
    if Dc != D or Hk == 0 or Hq % Hk:
        raise _lib.DSparkError(_lib.ERR_ARG, f"tree_sdpa: q {tuple(shape)}, caches {tuple(cache)}")
    if out is None:
        out = torch.empty((R, Hq, D), dtype=q.dtype, device=q.device)
    elif out.shape != shape:
        raise _lib.DSparkError(_lib.ERR_ARG, f"out {tuple(out.shape)} for {tuple(shape)}")
    qs, os = _strides("q", q), _strides("out", out)
    ks, vs = _strides("k_cache", k_cache), _strides("v_cache", v_cache)
    dt = _dtype(q, k_cache, v_cache, out)
    words = 0
    if anc is not None:
        if anc.ndim != 2 or anc.shape[0] != R:
            raise _lib.DSparkError(_lib.ERR_ARG, f"anc {tuple(anc.shape)} for {R} rows")
        words = anc.shape[1]
    n = _workspace(B, Hq, Hk, D, max_nodes, q.get_device())
    ws = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
    _lib.check(_lib.lib.dspark_tree_attn(_pack_attn(
        q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), qs[0], qs[1], os[0], os[1],
        ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], int32("cu_rows", cu_rows), int32("kv_len", kv_len, B),
        int32("kv_start", kv_start, B), int32("anc", anc), ws.data_ptr() if n else 0, n, scale, dt, words,
        max_nodes, R, B, Hq, Hk, D, cap, KB), stream))
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
                _strides("cache", t)
                if t.data_ptr() % 16:
                    raise _lib.DSparkUnsupported(_lib.ERR_UNSUPPORTED, "caches must be 16-byte aligned")
        if ks[0].ndim != 4:
            raise _lib.DSparkError(_lib.ERR_ARG, "caches [B, H, cap, D]")
        on_device(ks[0], *ks, *vs)
        self.device = ks[0].device
        self.k_caches, self.v_caches = ks, vs
        self.batch, self.heads, self.cap, self.dim = ks[0].shape
        self.elem = ks[0].element_size()
        self._kp = torch.tensor([t.data_ptr() for t in ks], dtype=torch.int64, device=self.device)
        self._vp = torch.tensor([t.data_ptr() for t in vs], dtype=torch.int64, device=self.device)
        self._kp_ptr, self._vp_ptr = self._kp.data_ptr(), self._vp.data_ptr()
        self._ks, self._vs = (_lib.i64_array(g[0].stride()[:3]) for g in (ks, vs))

    def keep(self, path: torch.Tensor, cu_rows: torch.Tensor, n_accept: torch.Tensor,
             lens: torch.Tensor, *, kv_start: torch.Tensor | None = None) -> None:
        """With ``base = lens[b] - n_accept[b] - 1`` (``lens`` as the accept left it), move cache row
        ``base + path[cu_rows[b] + i]`` to ``base + i`` for ``i <= n_accept[b]``, in every layer."""
        B = n_accept.numel()
        stream = on_device(self._kp, path, cu_rows, n_accept, lens, kv_start)
        if path.numel() == 0:  # no request has rows
            return
        _lib.check(_lib.lib.dspark_kv_keep_path(
            self._kp_ptr, self._vp_ptr, len(self.k_caches), self._ks, self._vs, int32("path", path),
            int32("cu_rows", cu_rows, B + 1), int32("n_accept", n_accept), int32("lens", lens, B),
            int32("kv_start", kv_start, B), B, self.heads, self.dim, self.elem, self.cap, self.batch, stream))
