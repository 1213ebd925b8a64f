"""The paged 8-bit cache without a GPU: what a call may not be given."""

from __future__ import annotations

import copy
import ctypes as C
import io

import pytest
import torch

import mlx_dspark_b200  # noqa: F401
from mlx_dspark_b200 import _lib, paged


def test_append_refuses_lengths_that_overlap_its_inputs():
    """One block writes len_out while others read kv_len, cu_rows, row_pos and page_table."""
    buf = (C.c_int32 * 256)()
    p = C.cast(buf, C.c_void_p).value
    p += -p % 16
    B, R = 5, 9
    ok = dict(q=p, k=p, v=p, q_out=p, k_pages=p, v_pages=p, k_scale=p, v_scale=p, freq=p, dtype=0, layout=0,
              R=R, B=B, Hq=2, Hk=1, D=64, rot=64, page=16, n_pages=4, max_pages=2, table_stride=3)
    at = dict(kv_len=(p + 256, B), cu_rows=(p + 384, B + 1), row_pos=(p + 512, R), page_table=(p + 640, 4 * 3 + 2))

    def rc(out, **kw):
        args = {**ok, **{k: v[0] for k, v in at.items()}, "len_out": out, **kw}
        return _lib.lib.dspark_paged_append(C.byref(_lib.PagedAppendArgs(**args)), None)

    for name, (first, n) in at.items():
        for out in (first, first + 4 * (n - 1), first - 4 * (B - 1)):
            assert rc(out) == _lib.ERR_ARG and "len_out" in _lib.last_error(), (name, out - first)
        # beside them: refused for the next reason instead, the pages' alignment
        for out in (first + 4 * n, first - 4 * B):
            assert rc(out, k_pages=p + 8) == _lib.ERR_UNSUPPORTED, (name, out - first)
    assert rc(at["row_pos"][0], row_pos=None, k_pages=p + 8) == _lib.ERR_UNSUPPORTED
    assert rc(None, k_pages=p + 8) == _lib.ERR_UNSUPPORTED



def test_append_refuses_pages_that_share_their_memory():
    """Blocks of one launch write pages, heads, keys and values side by side."""
    buf = (C.c_int32 * 256)()
    p = C.cast(buf, C.c_void_p).value
    p += -p % 16
    page = (4096, 1024, 64)
    ok = dict(q=p, k=p, v=p, q_out=p, k_pages=p, v_pages=p + 64, k_scale=p, v_scale=p + 64, kp_strides=page, vp_strides=page,
              scale_strides=(2, 1), freq=p, cu_rows=p, kv_len=p, page_table=p, dtype=0, layout=0, R=1, B=1, Hq=2, Hk=2, D=64,
              rot=64, page=16, n_pages=4, max_pages=2)

    def rc(**kw):
        return _lib.lib.dspark_paged_append(C.byref(_lib.PagedAppendArgs(**{**ok, **kw})), None)

    for bad in (dict(v_pages=p), dict(v_scale=p), dict(kp_strides=(0, 1024, 64)), dict(vp_strides=(4096, 0, 64)),
                dict(kp_strides=(4096, 1024, 0)), dict(scale_strides=(0, 1)), dict(scale_strides=(2, 0))):
        assert rc(**bad) == _lib.ERR_ARG and "share" in _lib.last_error(), bad


def test_a_pools_tensors_and_sizes_are_fixed(monkeypatch):
    """Calls use the addresses and sizes that the pool was made with: another tensor in the place of one of them would leave the
    old one's memory, which may be gone, to be read and written."""
    monkeypatch.setattr(paged, "on_device", lambda *a: 0)
    cache = paged.PagedCache.empty(4, 2, 16, 64, "cpu")
    for name in ("k", "v", "k_scale", "v_scale"):
        with pytest.raises(AttributeError, match=name):
            setattr(cache, name, getattr(cache, name).clone())
    for name in ("n_pages", "heads", "page_size", "head_dim"):
        with pytest.raises(AttributeError, match=name):
            setattr(cache, name, 8)
    cache.k_scale[1] = 2.0  # their values are not
    cache.v_scale.fill_(4.0)
    cache.v_scale *= 2
    cache.owner = "a request"
    cache.owner = None
    assert cache.k_scale[1, 1] == 2.0 and cache.v_scale[0, 0] == 8.0 and cache.n_pages == 4 and cache._at[2] == cache.k_scale.data_ptr()


def test_a_copied_pool_is_its_own(monkeypatch):
    """A deep copy and a loaded pool use their own tensors' addresses, a shallow copy the same ones."""
    monkeypatch.setattr(paged, "on_device", lambda *a: 0)
    k, v = (torch.randint(0, 256, (4, 16, 2, 64), dtype=torch.uint8).view(torch.float8_e4m3fn).permute(0, 2, 1, 3) for _ in range(2))
    cache = paged.PagedCache(k, v, torch.rand(4, 2), torch.rand(4, 2))
    file = io.BytesIO()
    torch.save(cache, file)
    file.seek(0)
    for other in (copy.deepcopy(cache), torch.load(file, weights_only=False), copy.copy(cache)):
        for i, name in enumerate(("k", "v", "k_scale", "v_scale")):
            mine, its = getattr(cache, name), getattr(other, name)
            assert other._at[i] == its.data_ptr() and its.stride() == mine.stride()
            assert torch.equal(its.view(torch.uint8) if i < 2 else its, mine.view(torch.uint8) if i < 2 else mine)
        assert other._at[4:] == cache._at[4:] and other._kst == cache._kst and other.page_size == 16
    assert copy.deepcopy(cache)._at[0] != cache._at[0] and copy.copy(cache)._at == cache._at
