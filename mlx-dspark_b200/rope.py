"""Rotary positions of packed rows, with the K/V append of a drafted tree.

The verify forward's fused QKV epilogue rotates Qwen3's way: half layout, a whole head of 128,
unscaled frequencies, and a cache slot that is the position itself. This module is the form for
everything else: interleaved or half layouts, a rotated part of the head, contexts stretched by
linear / NTK / YaRN / Llama-3 scaling, an optional RMS norm of each q / k head before the rotation,
and rows whose rotary position (a tree node's depth) is not their cache slot (its place).

Positions are turned into phases in 64-bit fixed-point turns, so long contexts keep full accuracy
(an fp32 product of position and frequency is off by 4e-3 rad at 100k).
"""

from __future__ import annotations

import math

import torch

from . import _lib
from ._torch import int32, on_device

_DT = {torch.bfloat16: 0, torch.float16: 1}
_LAYOUTS = {"half": _lib.ROPE_HALF, "interleaved": _lib.ROPE_INTERLEAVED}


def inv_freq(rotary_dim: int, theta: float = 1e6, scaling: dict | None = None) -> tuple[list, float]:
    """Frequencies (radians a position) of the ``rotary_dim / 2`` pairs and the factor on the rotated
    values. ``scaling["type"]``:

    * ``None`` / ``"none"``: ``theta^(-2i/rot)``;
    * ``"linear"``: divided by ``factor``;
    * ``"ntk"``: ``theta * factor^(rot/(rot-2))`` as the base;
    * ``"yarn"``: pairs that turn less than ``beta_slow`` (1) times in ``original_max_position`` are
      divided by ``factor``, those above ``beta_fast`` (32) kept, a ramp between; factor on the values
      ``attention_factor`` or ``0.1 ln(factor) + 1``;
    * ``"llama3"``: wavelengths above ``original_max_position / low_freq_factor`` divided by
      ``factor``, below ``.. / high_freq_factor`` kept, blended between.
    """
    sc = scaling or {}
    if sc and "type" not in sc:  # another file's names for it would pass as unscaled
        raise ValueError(f"rope scaling without a type: {sorted(sc)}")
    kind = sc.get("type") or "none"
    n, rot = rotary_dim // 2, rotary_dim
    if kind == "none":
        return [theta ** (-2.0 * i / rot) for i in range(n)], 1.0
    if kind not in ("linear", "ntk", "yarn", "llama3"):
        raise ValueError(f"unknown rope scaling {kind!r}")
    f = float(sc["factor"])
    if not f > 0:
        raise ValueError(f"rope scaling factor {f}")
    base = [theta ** (-2.0 * i / rot) for i in range(n)]
    if kind == "linear":
        return [x / f for x in base], 1.0
    if kind == "ntk":
        if rot <= 2:
            raise ValueError("ntk scaling needs a rotary dim above 2")
        t = theta * f ** (rot / (rot - 2))
        return [t ** (-2.0 * i / rot) for i in range(n)], 1.0
    old = float(sc["original_max_position"])
    if kind == "yarn":
        def pair_of(turns: float) -> float:  # the (real-valued) pair with that many turns in `old`
            return rot * math.log(old / (turns * 2 * math.pi)) / (2 * math.log(theta))

        lo = max(math.floor(pair_of(float(sc.get("beta_fast", 32.0)))), 0)
        hi = min(math.ceil(pair_of(float(sc.get("beta_slow", 1.0)))), rot - 1)
        width = max(hi - lo, 1e-3)
        out = []
        for i, x in enumerate(base):
            r = min(max((i - lo) / width, 0.0), 1.0)
            out.append(x / f * r + x * (1.0 - r))
        m = sc.get("attention_factor")
        if m is None:
            m = 0.1 * math.log(f) + 1.0 if f > 1 else 1.0
        return out, float(m)
    low, high = float(sc["low_freq_factor"]), float(sc["high_freq_factor"])
    out = []
    for x in base:
        s = (old * x / (2 * math.pi) - low) / (high - low)
        s = min(max(s, 0.0), 1.0)
        out.append((1.0 - s) * x / f + s * x)
    return out, 1.0


class RopeTable:
    """The rotary form of one model: layout, rotated part of the head, and its frequencies on the
    device (``freq``: int64 bit patterns of 64-bit fixed-point turns a position)."""

    def __init__(self, head_dim: int, rotary_dim: int | None = None, *, theta: float = 1e6,
                 layout: str = "half", scaling: dict | None = None, device="cuda"):
        rot = int(head_dim if rotary_dim is None else rotary_dim)
        if layout not in _LAYOUTS:
            raise ValueError(f"rope layout {layout!r} (half or interleaved)")
        if head_dim <= 0 or head_dim % 16 or head_dim > 512 or rot <= 0 or rot % 16 or rot > head_dim:
            raise _lib.DSparkUnsupported(
                _lib.ERR_UNSUPPORTED, f"rotary dim {rot} of head_dim {head_dim} (multiples of 16, <= 512)")
        self.head_dim, self.rotary_dim, self.layout = int(head_dim), rot, layout
        self.inv_freq, self.mscale = inv_freq(rot, float(theta), scaling)
        turns = [int(round(x / (2 * math.pi) % 1.0 * 2.0 ** 64)) % 2 ** 64 for x in self.inv_freq]
        self.freq = torch.tensor([t - 2 ** 64 if t >= 2 ** 63 else t for t in turns],
                                 dtype=torch.int64, device=device)
        self.freq_ptr, self.layout_code = self.freq.data_ptr(), _LAYOUTS[layout]


_pack = _lib.packer(_lib.RopeArgs)


def _strides(name: str, t: torch.Tensor) -> tuple:
    """``t``'s strides, the last of them checked to be 1."""
    st = t.stride()
    if st[-1] != 1 and t.shape[-1] > 1:
        raise _lib.DSparkUnsupported(_lib.ERR_UNSUPPORTED, f"{name}: head_dim must be contiguous")
    return st


def _dtype(first: torch.Tensor, *rest: torch.Tensor | None) -> int:
    dt = first.dtype
    for t in rest:
        if t is not None and t.dtype is not dt:
            raise _lib.DSparkUnsupported(_lib.ERR_UNSUPPORTED, f"tensors of {dt} and {t.dtype}")
    code = _DT.get(dt)
    if code is None:
        raise _lib.DSparkUnsupported(_lib.ERR_UNSUPPORTED, f"{dt} (bf16 or fp16)")
    return code


def _norm_weight(name: str, w: torch.Tensor | None, D: int) -> int:
    if w is None:
        return 0
    if w.numel() != D or not w.is_contiguous():
        raise _lib.DSparkError(_lib.ERR_ARG, f"{name} must be a contiguous [{D}]")
    return w.data_ptr()


def rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: RopeTable,
                row_pos: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                row_slot: torch.Tensor, *, row_req: torch.Tensor | None = None,
                q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None,
                eps: float = 1e-6, q_out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotate packed rows ``q [R, Hq, D]`` and ``k [R, Hk, D]`` to ``row_pos`` and write the rotated
    ``k`` and ``v`` to row ``row_slot[r]`` of batch entry ``row_req[r]`` (default 0) of the caches
    ``[B, Hk, cap, D]``. Returns the rotated q (``q_out``, which may be ``q``). All tensors may be
    strided views with head_dim contiguous. ``row_*`` are int32 ``[R]`` on the device; rows outside
    the cache are dropped and recorded in the device status, rows of no request (``row_req`` -1) only
    dropped."""
    stream = on_device(q, k, v, k_cache, v_cache, row_pos, row_slot, row_req, q_norm, k_norm, q_out,
                       table.freq)
    shape, cache = q.shape, k_cache.shape
    if len(shape) != 3 or k.ndim != 3 or len(cache) != 4:
        raise _lib.DSparkError(_lib.ERR_ARG, "rope_append: q / k [R, H, D], caches [B, H, cap, D]")
    R, Hq, D = shape
    B, Hk, cap, Dc = cache
    if k.shape != (R, Hk, D) or v.shape != k.shape or v_cache.shape != cache or Dc != D:
        raise _lib.DSparkError(_lib.ERR_ARG, f"rope_append: q {tuple(shape)}, k {tuple(k.shape)}, "
                               f"v {tuple(v.shape)}, caches {tuple(cache)}")
    if D != table.head_dim:
        raise _lib.DSparkError(_lib.ERR_ARG, f"head_dim {D}, the table's is {table.head_dim}")
    if q_out is None:
        q_out = torch.empty((R, Hq, D), dtype=q.dtype, device=q.device)
    elif q_out.shape != shape:
        raise _lib.DSparkError(_lib.ERR_ARG, f"q_out {tuple(q_out.shape)} for {tuple(shape)}")
    qs, ks, vs, os = _strides("q", q), _strides("k", k), _strides("v", v), _strides("q_out", q_out)
    kc, vc = _strides("k_cache", k_cache), _strides("v_cache", v_cache)
    dt = _dtype(q, k, v, q_out, k_cache, v_cache, q_norm, k_norm)
    _lib.check(_lib.lib.dspark_rope_append(_pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), qs[0], qs[1], ks[0], ks[1], vs[0], vs[1],
        q_out.data_ptr(), os[0], os[1], k_cache.data_ptr(), v_cache.data_ptr(), kc[0], kc[1], kc[2],
        vc[0], vc[1], vc[2], table.freq_ptr, int32("row_pos", row_pos, R), int32("row_slot", row_slot, R),
        int32("row_req", row_req, R), _norm_weight("q_norm", q_norm, D), _norm_weight("k_norm", k_norm, D),
        table.mscale, eps, dt, table.layout_code, R, Hq, Hk, D, table.rotary_dim, cap, B), stream))
    return q_out


def rotate(x: torch.Tensor, table: RopeTable, row_pos: torch.Tensor, *,
           norm: torch.Tensor | None = None, eps: float = 1e-6,
           out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotate packed rows ``x [R, H, D]`` to ``row_pos`` (int32 ``[R]``), no cache; ``out`` may be
    ``x``."""
    stream = on_device(x, row_pos, norm, out, table.freq)
    if x.ndim != 3 or x.shape[2] != table.head_dim:
        raise _lib.DSparkError(_lib.ERR_ARG, f"rotate: {tuple(x.shape)}, head_dim {table.head_dim}")
    R, H, D = x.shape
    if out is None:
        out = torch.empty((R, H, D), dtype=x.dtype, device=x.device)
    elif out.shape != x.shape:
        raise _lib.DSparkError(_lib.ERR_ARG, f"out {tuple(out.shape)} for {tuple(x.shape)}")
    xs, os = _strides("x", x), _strides("out", out)
    dt = _dtype(x, out, norm)
    _lib.check(_lib.lib.dspark_rope_append(_pack(
        x.data_ptr(), 0, 0, xs[0], xs[1], 0, 0, 0, 0, out.data_ptr(), os[0], os[1], 0, 0, 0, 0, 0, 0, 0, 0,
        table.freq_ptr, int32("row_pos", row_pos, R), 0, 0, _norm_weight("norm", norm, D), 0, table.mscale,
        eps, dt, table.layout_code, R, H, 0, D, table.rotary_dim, 0, 0), stream))
    return out
