"""Edges of the tree-round operators that need no GPU: refusals."""

from __future__ import annotations

import ctypes as C

import pytest

from mlx_dspark_b200 import _lib, rope


def _aligned():
    buf = (C.c_uint8 * 256)()
    return buf, (C.addressof(buf) + 15) // 16 * 16


def test_workspaces_have_to_be_aligned():
    buf, p = _aligned()
    s3 = (512, 512, 64)
    attn = dict(q=p, k=p, v=p, out=p, cu_rows=p, kv_len=p, anc=p, ws_bytes=1 << 40, scale=1.0, anc_words=1,
                max_rows=4, R=4, B=1, Hq=4, Hk=2, D=64, cap=8, kv_batch=1, q_strides=(256, 64),
                o_strides=(256, 64), k_strides=s3, v_strides=s3)
    accept = dict(logits=p, ids=p, cu_rows=p, u=p, noise=p, n_accept=p, next_tok=p, ws_bytes=1 << 40,
                  ld_logits=100, ld_noise=100, dtype=0, R=4, B=1, V=100, max_rows=4)
    for off in (4, 8):
        assert _lib.lib.dspark_tree_attn(C.byref(_lib.TreeAttnArgs(**attn, workspace=p + off)), None) == _lib.ERR_ARG
        assert "aligned" in _lib.last_error()
        assert _lib.lib.dspark_sample_accept(C.byref(_lib.SampleArgs(**accept, workspace=p + off)), None) == _lib.ERR_ARG
        assert "aligned" in _lib.last_error()


@pytest.mark.parametrize("scaling", [{"factor": 4.0}, {"rope_type": "yarn", "factor": 4.0, "original_max_position": 8192}])
def test_a_scaling_without_a_type_is_not_unscaled(scaling):
    with pytest.raises(ValueError, match="type"):
        rope.inv_freq(64, 1e6, scaling)


def test_unscaled_forms():
    plain = rope.inv_freq(64, 1e6)
    assert all(rope.inv_freq(64, 1e6, s) == plain for s in (None, {}, {"type": None}, {"type": "none"}))
