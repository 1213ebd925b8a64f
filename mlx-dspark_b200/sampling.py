"""Accept of drafted tokens for sampled targets (temperature above zero).

:func:`.batch_engine.accept` is the greedy accept; this is its sampled form, on chains and on trees,
with the random numbers given by the caller, so that a round can be repeated. The emitted tokens have
the target's own distribution whatever was drafted (the reference's lossless sampling,
src/mlx_dspark/sampling.py).
"""

from __future__ import annotations

import torch

from . import _lib
from ._torch import int32, on_device

_DT = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _rows_of(name: str, t: torch.Tensor, rows: int, V: int) -> torch.Tensor:
    if t.ndim != 2 or t.shape[0] != rows or t.shape[1] != V or (V > 1 and t.stride(1) != 1):
        raise _lib.DSparkError(_lib.ERR_ARG, f"{name} {tuple(t.shape)}: [{rows}, {V}] with contiguous rows")
    return t


def _f32(name: str, t: torch.Tensor | None, n: int):
    if t is None:
        return None
    if t.dtype != torch.float32 or t.numel() != n or not t.is_contiguous():
        raise _lib.DSparkError(_lib.ERR_ARG, f"{name} must be {n} contiguous float32 values")
    return t.data_ptr()


def sample_accept(logits: torch.Tensor, ids: torch.Tensor, cu_rows: torch.Tensor, u: torch.Tensor,
                  noise: torch.Tensor, *, temperature: torch.Tensor | None = None,
                  draft_probs: torch.Tensor | None = None, parent: torch.Tensor | None = None,
                  max_rows: int, lens: torch.Tensor | None = None, out: dict | None = None) -> dict:
    """Accept each request's block against ``p = softmax(logits / T)``.

    ``logits [R, V]`` (bf16, fp16 or fp32), ``ids`` int32 ``[R]`` (each block's pending token, then its
    drafts), ``cu_rows`` int32 ``[B + 1]``, ``u`` float32 ``[R]`` uniform in [0, 1), ``noise`` float32
    ``[B, V]`` exponential(1), ``temperature`` float32 ``[B]`` (``None``: 1; 0: greedy).

    * chain (``parent is None``): the draft after row r is accepted iff ``u[r] * q(x) < p_r(x)``;
      ``draft_probs [R, V]``: row r is the distribution that draft was drawn from (``None``: the
      draft was proposed outright, q(x) = 1);
    * tree (``parent`` int32 ``[R]``, places within the request, -1 for the root): a node's children
      are tried in order, accepted is the first whose running sum of ``p_r`` exceeds ``u[r]``.

    The token after the path is drawn by ``argmax(w / noise)``: ``w = max(p - q, 0)`` after a
    rejection with ``draft_probs``, else ``p`` without the tokens just tried. Returns ``n`` (accepted
    drafts), ``next``, ``prob`` (p of each row's token given its parent, 1 for roots) and ``path``
    (kept places of each request in order, then -1); ``lens`` (int32 ``[B]``, tokens cached after the
    verify's append) loses the rejected rows in place. ``max_rows`` (<= 1024) bounds a block."""
    dev, stream = on_device(logits, ids, cu_rows, u, noise, temperature, draft_probs, parent, lens)
    R, B = ids.numel(), cu_rows.numel() - 1
    V = logits.shape[-1]
    _rows_of("logits", logits, R, V), _rows_of("noise", noise, B, V)
    if logits.dtype not in _DT or (draft_probs is not None and draft_probs.dtype not in _DT):
        raise _lib.DSparkUnsupported(_lib.ERR_UNSUPPORTED, f"logits {logits.dtype} (bf16, fp16 or fp32)")
    if noise.dtype != torch.float32:
        raise _lib.DSparkError(_lib.ERR_ARG, f"noise is {noise.dtype}, not float32")
    if draft_probs is not None:
        _rows_of("draft_probs", draft_probs, R, V)
    int32("ids", ids), int32("cu_rows", cu_rows), int32("parent", parent, R), int32("lens", lens, B)
    if out is None:
        e = dict(dtype=torch.int32, device=dev)
        out = {"n": torch.empty(B, **e), "next": torch.empty(B, **e),
               "prob": torch.empty(R, dtype=torch.float32, device=dev), "path": torch.empty(R, **e)}
    else:
        int32("n", out["n"], B), int32("next", out["next"], B), int32("path", out["path"], R)
        on_device(logits, out["n"], out["next"], out["prob"], out["path"])
    n = int(_lib.lib.dspark_sample_workspace(R, B, V))
    ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    a = _lib.SampleArgs(
        logits.data_ptr(), None if draft_probs is None else draft_probs.data_ptr(), logits.stride(0),
        0 if draft_probs is None else draft_probs.stride(0), noise.stride(0), ids.data_ptr(),
        cu_rows.data_ptr(), None if parent is None else parent.data_ptr(), _f32("u", u, R),
        noise.data_ptr(), _f32("temperature", temperature, B), out["n"].data_ptr(),
        out["next"].data_ptr(), _f32("prob", out["prob"], R), out["path"].data_ptr(),
        None if lens is None else lens.data_ptr(), None if ws is None else ws.data_ptr(), n,
        _DT[logits.dtype], 0 if draft_probs is None else _DT[draft_probs.dtype], R, B, V, max_rows)
    _lib.check(_lib.lib.dspark_sample_accept(a, stream))
    out["lens"] = lens
    return out
