"""Accept of drafted tokens for sampled targets (temperature above zero), and the log probabilities of tokens.

:func:`.batch_engine.accept` is the greedy accept; this is its sampled form, on chains and on trees,
with the random numbers given by the caller, so that a round can be repeated. The emitted tokens have
the target's own distribution whatever was drafted (the reference's lossless sampling,
src/mlx_dspark/sampling.py). :func:`token_logprobs` scores tokens: those that a round emitted, or a given text.
"""

from __future__ import annotations

import functools

import torch

from . import _lib
from ._torch import int32, on_device

_DT = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


_pack = _lib.packer(_lib.SampleArgs)
_pack_score = _lib.packer(_lib.ScoreArgs)


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


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, temperature: torch.Tensor | None = None,
                   top: int = 0, out: dict | None = None) -> dict:
    """Score one token a row against ``p = softmax(logits / T)``.

    ``logits [R, V]`` (bf16, fp16 or fp32, contiguous rows), ``tokens`` int32 ``[R]``, ``temperature`` float32
    ``[R]`` (``None``: 1; 1e-6 or less: greedy, all mass on the first largest logit). Returns ``logprob``
    (``ln p(token)``), ``entropy`` (``-sum p ln p``), ``rank`` (int32: tokens before it by logit, then the lower
    token; 0 is the most likely) and with ``top`` (up to 32) the first tokens of that order, ``top_ids`` and
    ``top_logprobs`` ``[R, top]``; ``out``, a former call's result of as many rows and alternatives, is written again.

    A logit of NaN, -inf, or at most -2^28 (fp16: its lowest value) masks its token: logprob -inf, rank -1, never
    an alternative; where fewer tokens than ``top`` are left, the others' ids are -1 and their logprobs -inf. A row
    whose token is outside the vocabulary (-1: a padded row) is not read: logprob and entropy 0, rank -1, no
    alternatives. Zeros of either sign are one logit.

    Alternatives of a row with more than 512 values at or near the last of them (a constant row, one of few distinct values) are
    found by a pass each: 272 such rows of 151,936 in bf16 take 443 us with 5 and 1703 with 32, others 36 and 40."""
    stream = on_device(logits, tokens, temperature, *(() if out is None else out.values()))
    if logits.ndim != 2:
        raise _lib.DSparkError(_lib.ERR_ARG, f"logits {tuple(logits.shape)}: [R, V]")
    R, V = logits.shape
    top = int(top)
    dt = _DT.get(logits.dtype)
    if dt is None:
        raise _lib.DSparkUnsupported(_lib.ERR_UNSUPPORTED, f"logits of {logits.dtype} (bf16, fp16 or fp32)")
    ld = _rows_of("logits", logits, R, V)
    if not 0 <= top <= 32:
        raise _lib.DSparkUnsupported(_lib.ERR_UNSUPPORTED, f"{top} alternatives (at most 32)")
    if out is None:  # parts of one buffer
        n = R * top
        buf = torch.empty(3 * R + 2 * n, dtype=torch.float32, device=logits.device)
        lp = buf.data_ptr()
        ent, rank, ids, tl = lp + 4 * R, lp + 8 * R, lp + 12 * R, lp + 4 * (3 * R + n)
        x = buf.split_with_sizes((R, R, R, n, n) if top else (R, R, R))
        out = {"logprob": x[0], "entropy": x[1], "rank": x[2].view(torch.int32)}
        if top:
            out["top_ids"], out["top_logprobs"] = x[3].view(torch.int32).view(R, top), x[4].view(R, top)
    else:
        if top and out.get("top_ids") is None or not top and "top_ids" in out:
            raise _lib.DSparkError(_lib.ERR_ARG, f"out of another call: {top} alternatives, {sorted(out)}")
        lp, ent, rank = _f32("logprob", out["logprob"], R), _f32("entropy", out["entropy"], R), int32("rank", out["rank"], R)
        ids = tl = 0
        if top:
            ids, tl = int32("top_ids", out["top_ids"], R * top), _f32("top_logprobs", out["top_logprobs"], R * top)
    _lib.check(_lib.lib.dspark_token_logprobs(_pack_score(
        logits.data_ptr(), ld, int32("tokens", tokens, R), _f32("temperature", temperature, R), lp, ent, rank,
        ids if top else 0, tl if top else 0, dt, R, V, top), stream))
    return out
