"""The paged 8-bit cache and token scores without a GPU: refusals, struct layouts, the reference forms."""

from __future__ import annotations

import ctypes as C
import math
import shutil
import subprocess
from pathlib import Path

import paged_reference as ref
import pytest
import torch

import mlx_dspark_b200  # noqa: F401
from mlx_dspark_b200 import DSparkError, DSparkUnsupported, _lib, paged, sampling

ROOT = Path(__file__).resolve().parents[1]
_MIRRORS = {"PagedAppendArgs": "dspark_paged_append_args", "PagedAttnArgs": "dspark_paged_attn_args",
            "ScoreArgs": "dspark_score_args"}


def test_ctypes_mirrors_match_the_header_layout(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not available")
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "dspark.h"', "int main(void) {"]
    want = {}
    for py, c in _MIRRORS.items():
        cls = getattr(_lib, py)
        lines.append(f'  printf("{py} %zu\\n", sizeof({c}));')
        want[py] = C.sizeof(cls)
        for name, _ in cls._fields_:
            lines.append(f'  printf("{py}.{name} %zu\\n", offsetof({c}, {name}));')
            want[f"{py}.{name}"] = getattr(cls, name).offset
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines + ["  return 0;", "}"]) + "\n")
    subprocess.run([gcc, "-std=c11", "-I", str(ROOT / "include"), str(src), "-o", str(tmp_path / "layout")],
                   check=True, capture_output=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout
    assert {k: int(v) for k, v in (line.split() for line in out.splitlines())} == want


def _fake():
    buf = (C.c_uint8 * 64)()
    p = C.cast(buf, C.c_void_p).value
    return p + (-p) % 16


def test_append_refusals():
    p = _fake()
    ok = dict(q=p, k=p, v=p, q_out=p, k_pages=p, v_pages=p, k_scale=p, v_scale=p, freq=p, cu_rows=p, kv_len=p,
              page_table=p, dtype=0, layout=0, R=1, B=1, Hq=2, Hk=1, D=64, rot=64, page=16, n_pages=4, max_pages=2)

    def rc(**kw):
        return _lib.lib.dspark_paged_append(C.byref(_lib.PagedAppendArgs(**{**ok, **kw})), None)

    assert rc(dtype=2) == _lib.ERR_UNSUPPORTED and "dtype" in _lib.last_error()
    assert rc(D=80) == _lib.ERR_UNSUPPORTED and "head_dim" in _lib.last_error()
    for page in (0, 8, 48, 256):
        assert rc(page=page) == _lib.ERR_UNSUPPORTED and "pages of" in _lib.last_error()
    assert rc(rot=24) == _lib.ERR_UNSUPPORTED and rc(rot=80) == _lib.ERR_UNSUPPORTED and rc(rot=0) == _lib.ERR_UNSUPPORTED
    assert rc(layout=2) == _lib.ERR_ARG and rc(R=-1) == _lib.ERR_ARG and rc(Hq=0) == _lib.ERR_ARG
    assert rc(n_pages=-1) == _lib.ERR_ARG and rc(max_pages=-1) == _lib.ERR_ARG
    for name in ("q", "k", "v", "q_out", "k_pages", "v_pages", "k_scale", "v_scale", "freq", "cu_rows", "kv_len", "page_table"):
        assert rc(**{name: None}) == _lib.ERR_ARG, name
    assert rc(k_pages=p + 8) == _lib.ERR_UNSUPPORTED and rc(kp_strides=(64, 64, 8)) == _lib.ERR_UNSUPPORTED
    assert rc(B=0) == _lib.OK
    assert _lib.lib.dspark_paged_append(None, None) == _lib.ERR_ARG


def test_attention_refusals():
    p = _fake()
    ok = dict(q=p, k_pages=p, v_pages=p, out=p, k_scale=p, v_scale=p, cu_rows=p, kv_len=p, page_table=p, workspace=p,
              ws_bytes=1 << 40, scale=1.0, dtype=0, causal=1, R=1, B=1, Hq=2, Hk=1, D=64, page=16, n_pages=4, max_pages=2)

    def rc(**kw):
        return _lib.lib.dspark_paged_attn(C.byref(_lib.PagedAttnArgs(**{**ok, **kw})), None)

    assert rc(dtype=2) == _lib.ERR_UNSUPPORTED and rc(D=256) == _lib.ERR_UNSUPPORTED and rc(page=24) == _lib.ERR_UNSUPPORTED
    assert rc(Hq=3, Hk=2) == _lib.ERR_ARG and rc(R=-1) == _lib.ERR_ARG
    assert rc(max_pages=1 << 30) == _lib.ERR_UNSUPPORTED and rc(R=1 << 30, Hq=8) == _lib.ERR_UNSUPPORTED
    for name in ("q", "out", "cu_rows", "kv_len", "page_table", "k_pages", "v_scale", "workspace"):
        assert rc(**{name: None}) == _lib.ERR_ARG, name
    assert rc(q=p + 4) == _lib.ERR_UNSUPPORTED and rc(q_strides=(12, 8)) == _lib.ERR_UNSUPPORTED
    assert rc(ws_bytes=1) == _lib.ERR_ARG and rc(workspace=p + 8) == _lib.ERR_ARG
    assert rc(R=0) == _lib.OK and rc(B=0) == _lib.OK
    assert _lib.lib.dspark_paged_attn(None, None) == _lib.ERR_ARG
    assert _lib.lib.dspark_paged_attn_workspace(0, 1, 2, 1, 64) == 0
    assert _lib.lib.dspark_paged_attn_workspace(1, 1, 3, 2, 64) == 0


def test_score_refusals():
    p = _fake()
    ok = dict(logits=p, ld=8, tokens=p, logprob=p, entropy=p, rank=p, top_ids=p, top_logprob=p, dtype=0, R=1, V=8, top=2)

    def rc(**kw):
        return _lib.lib.dspark_token_logprobs(C.byref(_lib.ScoreArgs(**{**ok, **kw})), None)

    assert rc(dtype=3) == _lib.ERR_UNSUPPORTED and rc(top=33) == _lib.ERR_UNSUPPORTED and rc(top=-1) == _lib.ERR_ARG
    assert rc(V=0) == _lib.ERR_ARG and rc(R=-1) == _lib.ERR_ARG and rc(R=0) == _lib.OK
    assert rc(logits=p + 1) == _lib.ERR_UNSUPPORTED and rc(dtype=2, logits=p + 2) == _lib.ERR_UNSUPPORTED
    for name in ("logits", "tokens", "logprob", "entropy", "rank", "top_ids", "top_logprob"):
        assert rc(**{name: None}) == _lib.ERR_ARG, name
    assert _lib.lib.dspark_token_logprobs(None, None) == _lib.ERR_ARG


def test_cpu_tensors_and_pools_are_refused():
    k = torch.zeros(4, 2, 16, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    s = torch.ones(4, 2)
    with pytest.raises(DSparkUnsupported):
        paged.PagedCache(k, k.clone(), s, s.clone())
    with pytest.raises(DSparkError):
        paged.PagedCache(k.view(torch.uint8), k, s, s)
    with pytest.raises(DSparkError):
        paged.PagedCache(k, k.clone(), s.double(), s)
    with pytest.raises(DSparkError):
        paged.PagedCache(k, k.clone(), s, torch.ones(2, 4).T)
    odd = torch.zeros(4, 2, 24, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    with pytest.raises(DSparkUnsupported):
        paged.PagedCache(odd, odd, s, s)
    with pytest.raises(DSparkUnsupported):
        sampling.token_logprobs(torch.zeros(1, 8), torch.zeros(1, dtype=torch.int32))


def test_reference_rounding_is_the_types():
    x = torch.cat([torch.linspace(-500, 500, 4001), torch.linspace(-0.05, 0.05, 4001)]).double()
    want = x.clamp(-448, 448).float().to(torch.float8_e4m3fn).double()
    assert torch.equal(ref.nearest(x), want)
    every = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    fine = ~every.isnan()
    assert torch.equal(ref.nearest(every)[fine], every[fine]) and int(fine.sum()) == 254


def test_reference_scale_and_score():
    assert ref.scale_of(448.0) == 1.0 and ref.scale_of(448.5) == 2.0 and ref.scale_of(224.0) == 0.5
    assert ref.scale_of(0.0) == 2.0 ** -64 and ref.scale_of(1e38) == 2.0 ** 64
    lp, ent, rank, ids, tl = ref.score(torch.tensor([1.0, 3.0, -math.inf, 3.0]), 3, 1.0, 4, -2.0 ** 28)
    z = math.exp(1) + 2 * math.exp(3)
    assert rank == 1 and ids == [1, 3, 0, -1] and abs(lp - (3 - math.log(z))) < 1e-12
    p = [math.exp(1) / z, math.exp(3) / z, math.exp(3) / z]
    assert abs(ent + sum(v * math.log(v) for v in p)) < 1e-12 and tl[3] == -math.inf
