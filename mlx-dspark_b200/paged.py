"""A paged cache of 8-bit values: append with rotary positions, and attention over the pages.

:class:`PagedCache` is one layer's pool of pages; a page holds 16 to 128 tokens of every head as e4m3 codes with one
scale a page and head. Requests share the pool: row b of an int32 page table ``[B, max_pages]`` names request b's
pages, in any order, and one page may stand in several tables (a shared prefix) as long as nobody appends to it.
Beside the other caches: :class:`.kvcache.BatchCache` and the pools of :class:`.target.Target` keep 16-bit rows in one
stretch a request, :class:`.kvcache.QuantizedKVCache` 4- or 8-bit codes with a scale for every 64 values of a row.

Packed rows are as everywhere in the batch engine (``cu_rows``): blocks of any number of rows, an idle request
none. Rollback is metadata only, as in the other caches: a smaller length, and the next append overwrites the tail.
"""

from __future__ import annotations

import functools

import torch

from . import _lib
from ._torch import int32, on_device
from .rope import RopeTable, _dtype, _norm_weight, _strides

PAGE_SIZES = (16, 32, 64, 128)
HEAD_DIMS = (64, 128)

_pack_append = _lib.packer(_lib.PagedAppendArgs)
_pack_attn = _lib.packer(_lib.PagedAttnArgs)


@functools.lru_cache(maxsize=4096)
def _workspace(R: int, B: int, Hq: int, Hk: int, D: int, device: int) -> int:
    return _lib.lib.dspark_paged_attn_workspace(R, B, Hq, Hk, D)


class PagedCache:
    """One layer's pages: codes ``k`` / ``v`` (``torch.float8_e4m3fn`` ``[pages, heads, page_size, head_dim]``, any
    strides of multiples of 16 with head_dim contiguous) and scales ``k_scale`` / ``v_scale`` (float32
    ``[pages, heads]``): value = code * scale, scales of 2^-64 to 2^64 as :meth:`append` makes them. :meth:`empty`
    makes a pool. :meth:`append` needs pages and scales that share no memory (no expanded ones, ``k`` and ``v`` apart);
    :meth:`attention` reads any."""

    _FIXED = frozenset(("k", "v", "k_scale", "v_scale", "n_pages", "heads", "page_size", "head_dim"))

    def __setattr__(self, name, value):
        # calls pass the addresses and sizes that the pool was made with
        if name in self._FIXED and self.__dict__.get(name, value) is not value:  # (the same one: `cache.k_scale *= 2`)
            raise AttributeError(f"{name} of a PagedCache is fixed: write into its tensors, or make another pool")
        super().__setattr__(name, value)

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor):
        if k.ndim != 4 or v.shape != k.shape or k.dtype is not torch.float8_e4m3fn or v.dtype is not k.dtype:
            raise _lib.DSparkError(_lib.ERR_ARG, f"pages {k.dtype} {tuple(k.shape)}, {v.dtype} {tuple(v.shape)}: "
                                   "float8_e4m3fn [pages, heads, page_size, head_dim]")
        self.n_pages, self.heads, self.page_size, self.head_dim = k.shape
        if self.page_size not in PAGE_SIZES or self.head_dim not in HEAD_DIMS:
            raise _lib.DSparkUnsupported(_lib.ERR_UNSUPPORTED, f"pages of {self.page_size} tokens of head_dim "
                                         f"{self.head_dim} ({PAGE_SIZES}, {HEAD_DIMS})")
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            if t.dtype is not torch.float32 or t.shape != k.shape[:2] or t.stride() != k_scale.stride():
                raise _lib.DSparkError(_lib.ERR_ARG, f"{name} {t.dtype} {tuple(t.shape)}: float32 "
                                       f"{tuple(k.shape[:2])}, both with the same strides")
        on_device(k, v, k_scale, v_scale)
        self._kst, self._vst = _strides("k", k)[:3], _strides("v", v)[:3]
        if any(x % 16 for x in (*self._kst, *self._vst, k.data_ptr(), v.data_ptr())):
            raise _lib.DSparkUnsupported(_lib.ERR_UNSUPPORTED, "the pages' rows must be 16-byte aligned")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self._at = (k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), *k_scale.stride())

    def __reduce__(self):  # a copy is made of its own tensors, whose addresses are others
        return type(self), (self.k, self.v, self.k_scale, self.v_scale)

    @classmethod
    def empty(cls, pages: int, heads: int, page_size: int, head_dim: int, device="cuda") -> "PagedCache":
        """A pool of zeros (scales 1)."""
        k, v = (torch.zeros((pages, heads, page_size, head_dim), dtype=torch.uint8,
                            device=device).view(torch.float8_e4m3fn) for _ in range(2))
        return cls(k, v, *(torch.ones((pages, heads), dtype=torch.float32, device=device) for _ in range(2)))

    def _table(self, page_table: torch.Tensor, B: int) -> tuple[int, int, int]:
        """Address, row stride and width of a page table."""
        if page_table.dtype is not torch.int32 or page_table.ndim != 2 or page_table.shape[0] != B or \
                (page_table.shape[1] > 1 and page_table.stride(1) != 1):
            raise _lib.DSparkError(_lib.ERR_ARG, f"page_table {page_table.dtype} {tuple(page_table.shape)}: int32 "
                                   f"[{B}, pages a request] with contiguous rows")
        return page_table.data_ptr(), page_table.stride(0), page_table.shape[1]

    def append(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: RopeTable, cu_rows: torch.Tensor,
               kv_len: torch.Tensor, page_table: torch.Tensor, *, row_pos: torch.Tensor | None = None,
               q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None, eps: float = 1e-6,
               q_out: torch.Tensor | None = None,
               len_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """Rotate packed rows ``q [R, Hq, D]`` and ``k [R, heads, D]`` and append the rotated ``k`` and ``v`` to their
        requests' pages: row i of request b becomes token ``kv_len[b] + i`` (int32 ``[B]``: tokens cached before). The
        rotary position is ``row_pos`` (int32 ``[R]``) or that token. ``q_norm`` / ``k_norm`` as in
        :func:`.rope.rope_append`. Returns the rotated q (``q_out``, which may be ``q``) and the new lengths
        (``len_out``, apart from ``kv_len`` and the call's other int32 inputs), which :meth:`attention` takes.

        The scale of a page and head is the smallest power of two with which the largest value appended to it is at
        most 448; a page that holds tokens already keeps its scale or raises it, and then its codes are rounded to
        the new one. Rows for which the table has no page (or one outside the pool) are dropped and recorded in the
        device status. Rows behind the last request's are left as they are. One call must not append to a page twice (two
        requests with one page, or a request whose table repeats it).

        How many rows a block takes goes by the call's mean rows a request: a prompt's chunk is appended faster apart from
        decoded tokens (512 rows 6.6 us, 96 tokens 5.8, in one call 36)."""
        stream = on_device(q, k, v, cu_rows, kv_len, page_table, row_pos, q_norm, k_norm, q_out, len_out, table.freq,
                           self.k)
        shape, D = q.shape, self.head_dim
        if len(shape) != 3 or shape[2] != D or k.shape != (shape[0], self.heads, D) or v.shape != k.shape:
            raise _lib.DSparkError(_lib.ERR_ARG, f"append: q {tuple(shape)}, k {tuple(k.shape)}, v {tuple(v.shape)} "
                                   f"for {self.heads} heads of {D}")
        if D != table.head_dim:
            raise _lib.DSparkError(_lib.ERR_ARG, f"head_dim {D}, the rope table's is {table.head_dim}")
        R, Hq, B = shape[0], shape[1], kv_len.numel()
        if q_out is None:
            q_out = torch.empty((R, Hq, D), dtype=q.dtype, device=q.device)
        elif q_out.shape != shape:
            raise _lib.DSparkError(_lib.ERR_ARG, f"q_out {tuple(q_out.shape)} for {tuple(shape)}")
        if len_out is None:
            len_out = torch.empty(B, dtype=torch.int32, device=q.device)
        qs, ks, vs, os = _strides("q", q), _strides("k", k), _strides("v", v), _strides("q_out", q_out)
        dt = _dtype(q, k, v, q_out, q_norm, k_norm)
        tp, ts, width = self._table(page_table, B)
        kp, vp, ksc, vsc, s0, s1 = self._at
        a, b = self._kst, self._vst
        _lib.check(_lib.lib.dspark_paged_append(_pack_append(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], q_out.data_ptr(), os[0],
            os[1], kp, vp, a[0], a[1], a[2], b[0], b[1], b[2], ksc, vsc, s0, s1, table.freq_ptr,
            int32("row_pos", row_pos, R), int32("cu_rows", cu_rows, B + 1), int32("kv_len", kv_len), tp, ts,
            int32("len_out", len_out, B), _norm_weight("q_norm", q_norm, D), _norm_weight("k_norm", k_norm, D),
            table.mscale, eps, dt, table.layout_code, R, B, Hq, self.heads, D, table.rotary_dim, self.page_size,
            self.n_pages, width), stream))
        return q_out, len_out

    def attention(self, q: torch.Tensor, cu_rows: torch.Tensor, kv_len: torch.Tensor, page_table: torch.Tensor, *,
                  scale: float, causal: bool = True, out: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of packed rows ``q [R, Hq, D]`` (bf16 or fp16) over their requests' pages. ``kv_len`` int32 ``[B]``
        counts a request's own rows too; ``causal``: its row i sees keys before ``kv_len[b] - rows(b) + i + 1``, else
        every row all ``kv_len[b]``. Returns ``out [R, Hq, D]``; a row that sees nothing is zero, a row of no request is
        not written. Keys of a page outside the pool are not seen (the device status records them), nor are those
        of a page whose scale is not positive.

        Scores and sums are fp32; the weights are rounded to fp16 for the product with v (fp16 results are off by 2.6e-4 of
        themselves on average where their own rounding alone gives 2.1e-4; bf16 results do not show it).

        The kernel is chosen for the whole call, before the lengths are known, by the mean number of rows a request and by the
        table's width in place of the longest length. So a table no wider than its requests need is fastest (one row over 2049
        keys 8.8 us, in a table of 131,072 tokens 10.7; 16 rows over 4096 keys 17 and 28), and a prompt's chunk apart from
        decoded tokens (96 of them 134 us and 512 rows over 16k keys 150, in one call 672). Neither changes a result but
        for the rounding of its weights."""
        stream = on_device(q, cu_rows, kv_len, page_table, out, self.k)
        shape, D, Hk = q.shape, self.head_dim, self.heads
        if len(shape) != 3 or shape[2] != D or Hk == 0 or shape[1] % Hk or shape[1] == 0:
            raise _lib.DSparkError(_lib.ERR_ARG, f"attention: q {tuple(shape)}, {Hk} heads of {D} in the cache")
        R, Hq, B = shape[0], shape[1], kv_len.numel()
        if out is None:
            out = torch.empty((R, Hq, D), dtype=q.dtype, device=q.device)
        elif out.shape != shape:
            raise _lib.DSparkError(_lib.ERR_ARG, f"out {tuple(out.shape)} for {tuple(shape)}")
        qs, os = _strides("q", q), _strides("out", out)
        dt = _dtype(q, out)
        tp, ts, width = self._table(page_table, B)
        n = _workspace(R, B, Hq, Hk, D, q.get_device())
        ws = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
        kp, vp, ksc, vsc, s0, s1 = self._at
        a, b = self._kst, self._vst
        _lib.check(_lib.lib.dspark_paged_attn(_pack_attn(
            q.data_ptr(), kp, vp, out.data_ptr(), ksc, vsc, qs[0], qs[1], os[0], os[1], a[0], a[1], a[2], b[0], b[1],
            b[2], s0, s1, int32("cu_rows", cu_rows, B + 1), int32("kv_len", kv_len), tp, ts,
            ws.data_ptr() if n else 0, n, scale, dt, int(causal), R, B, Hq, Hk, D, self.page_size, self.n_pages, width),
            stream))
        return out
