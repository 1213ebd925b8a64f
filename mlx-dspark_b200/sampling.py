"""Accept of drafted tokens for sampled targets (temperature above zero).

:func:`.batch_engine.accept` is the greedy accept; this is its sampled form, on chains and on trees,
with the random numbers given by the caller, so that a round can be repeated. The emitted tokens have
the target's own distribution whatever was drafted (the reference's lossless sampling,
src/mlx_dspark/sampling.py).
"""

from __future__ import annotations

import functools

import torch

from . import _lib
from ._torch import int32, on_device

_DT = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


_pack = _lib.packer(_lib.SampleArgs)


@functools.lru_cache(maxsize=4096)
def _workspace(R: int, B: int, V: int, device: int) -> int:
    return _lib.lib.dspark_sample_workspace(R, B, V)


def _rows_of(name: str, t: torch.Tensor, rows: int, V: int) -> int:
    """Row stride of ``t``, checked to be ``[rows, V]`` with contiguous rows."""
    st = t.stride()
    if t.shape != (rows, V) or (V > 1 and st[1] != 1):
        raise _lib.DSparkError(_lib.ERR_ARG, f"{name} {tuple(t.shape)}: [{rows}, {V}] with contiguous rows")
    return st[0]


def _f32(name: str, t: torch.Tensor | None, n: int) -> int:
    if t is None:
        return 0
    if t.dtype is not torch.float32 or t.numel() != n or not t.is_contiguous():
        raise _lib.DSparkError(_lib.ERR_ARG, f"{name} must be {n} contiguous float32 values")
    return t.data_ptr()


def sample_accept(logits: torch.Tensor, ids: torch.Tensor, cu_rows: torch.Tensor, u: torch.Tensor,
                  noise: torch.Tensor, *, temperature: torch.Tensor | None = None,
                  draft_probs: torch.Tensor | None = None, parent: torch.Tensor | None = None,
                  max_rows: int, row_limit: torch.Tensor | None = None, lens: torch.Tensor | None = None,
                  out: dict | None = None) -> dict:
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
    drafts), ``next``, ``prob`` (p of each row's token given its parent, 1 for roots), ``path``
    (kept places of each request in order, then -1) and ``lens`` where it was given; ``out``, a former
    call's result for as many rows and requests, is written again (its workspace too, on one stream).
    ``lens`` (int32 ``[B]``, tokens cached after the verify's append) loses the rejected rows in place.
    ``max_rows`` (<= 1024) bounds a block, ``row_limit`` (int32 ``[B]``) the rows of each that can be
    accepted: the others count as not tried, and a block of which no row can gives n 0, next -1 and
    loses all its rows."""
    given = () if out is None else (out["n"], out["next"], out["prob"], out["path"])
    stream = on_device(logits, ids, cu_rows, u, noise, temperature, draft_probs, parent, row_limit, lens, *given)
    R, B = ids.numel(), cu_rows.numel() - 1
    V = logits.shape[-1]
    ld, ld_noise = _rows_of("logits", logits, R, V), _rows_of("noise", noise, B, V)
    dt, ddt, draft, ld_draft = _DT.get(logits.dtype), 0, 0, 0
    if draft_probs is not None:
        ld_draft = _rows_of("draft_probs", draft_probs, R, V)
        draft, ddt = draft_probs.data_ptr(), _DT.get(draft_probs.dtype)
    if dt is None or ddt is None:
        raise _lib.DSparkUnsupported(_lib.ERR_UNSUPPORTED, "logits and draft_probs: bf16, fp16 or fp32")
    if noise.dtype is not torch.float32:
        raise _lib.DSparkError(_lib.ERR_ARG, f"noise is {noise.dtype}, not float32")
    if out is None:
        e = dict(dtype=torch.int32, device=logits.device)
        out = {"n": torch.empty(B, **e), "next": torch.empty(B, **e),
               "prob": torch.empty(R, dtype=torch.float32, device=logits.device),
               "path": torch.empty(R, **e)}
    n = _workspace(R, B, V, logits.get_device())
    # The workspace goes with the result's `n`, as an attribute: the dictionary holds results alone. A graph has
    # to own what its replays write, a stream what the allocator may hand on in its order.
    kept, ws = getattr(out["n"], "_accept_workspace", (None, None))
    if n and (kept != stream or ws.numel() < n or torch._C._cuda_isCurrentStreamCapturing()):
        ws = torch.empty(n, dtype=torch.uint8, device=logits.device)
        if not torch._C._cuda_isCurrentStreamCapturing():
            out["n"]._accept_workspace = stream, ws
    _lib.check(_lib.lib.dspark_sample_accept_limited(_pack(
        logits.data_ptr(), draft, ld, ld_draft, ld_noise, int32("ids", ids), int32("cu_rows", cu_rows),
        int32("parent", parent, R), _f32("u", u, R), noise.data_ptr(), _f32("temperature", temperature, B),
        int32("n", out["n"], B), int32("next", out["next"], B), _f32("prob", out["prob"], R),
        int32("path", out["path"], R), int32("lens", lens, B), ws.data_ptr() if n else 0, n, dt, ddt, R, B, V,
        max_rows), int32("row_limit", row_limit, B), stream))
    out.pop("lens", None)
    if lens is not None:
        out["lens"] = lens
    return out
