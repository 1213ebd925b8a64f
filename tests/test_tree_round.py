"""Tree-round operators without a GPU: refusals, struct layouts, frequencies, the reference forms."""

from __future__ import annotations

import ctypes as C
import math
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch
import tree_reference as ref

import mlx_dspark_b200  # noqa: F401
from mlx_dspark_b200 import DSparkError, DSparkUnsupported, _lib, rope, sampling, tree

ROOT = Path(__file__).resolve().parents[1]
_MIRRORS = {"RopeArgs": "dspark_rope_args", "TreeAttnArgs": "dspark_tree_attn_args",
            "SampleArgs": "dspark_sample_args", "TreeFwd": "dspark_tree_fwd"}


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


def test_packed_arguments_are_the_structs():
    for py in _MIRRORS:
        cls = getattr(_lib, py)
        flat, args = [], {}
        for k, (name, t) in enumerate(cls._fields_):
            if hasattr(t, "_length_"):
                args[name] = tuple(1000 * k + i for i in range(t._length_))
                flat += args[name]
            else:
                args[name] = k + 1
                flat.append(k + 1)
        assert _lib.packer(cls)(*flat) == bytes(cls(**args))


def _fake():
    buf = (C.c_uint8 * 64)()
    return C.cast(buf, C.c_void_p).value


def test_rope_refusals():
    p = _fake()
    ok = dict(q=p, k=p, v=p, q_out=p, k_cache=p, v_cache=p, freq=p, row_pos=p, row_slot=p, dtype=0,
              layout=0, R=1, Hq=2, Hk=1, D=64, rot=64, cap=8, batch=1)

    def rc(**kw):
        return _lib.lib.dspark_rope_append(C.byref(_lib.RopeArgs(**{**ok, **kw})), None)

    assert rc(dtype=2) == _lib.ERR_UNSUPPORTED and "dtype" in _lib.last_error()
    assert rc(D=72) == _lib.ERR_UNSUPPORTED and "head_dim" in _lib.last_error()
    assert rc(rot=24) == _lib.ERR_UNSUPPORTED and rc(rot=80) == _lib.ERR_UNSUPPORTED
    assert rc(layout=5) == _lib.ERR_ARG and rc(q=None) == _lib.ERR_ARG
    assert rc(row_slot=None) == _lib.ERR_ARG and rc(v=None) == _lib.ERR_ARG
    assert rc(R=-1) == _lib.ERR_ARG and rc(cap=0) == _lib.ERR_ARG
    assert rc(R=0) == _lib.OK
    assert _lib.lib.dspark_rope_append(None, None) == _lib.ERR_ARG


def test_tree_attn_refusals():
    p = _fake() // 16 * 16
    s3 = (512, 512, 64)
    ok = dict(q=p, k=p, v=p, out=p, cu_rows=p, kv_len=p, anc=p, workspace=p, ws_bytes=1 << 40, scale=1.0,
              anc_words=1, max_rows=4, R=4, B=1, Hq=4, Hk=2, D=64, cap=8, kv_batch=1, q_strides=(256, 64),
              o_strides=(256, 64), k_strides=s3, v_strides=s3)

    def rc(**kw):
        return _lib.lib.dspark_tree_attn(C.byref(_lib.TreeAttnArgs(**{**ok, **kw})), None)

    assert rc(dtype=2) == _lib.ERR_UNSUPPORTED and "dtype" in _lib.last_error()
    assert rc(D=96) == _lib.ERR_UNSUPPORTED and "head_dim" in _lib.last_error()
    assert rc(Hq=3) == _lib.ERR_ARG and rc(B=2, kv_batch=0) == _lib.ERR_ARG
    assert rc(anc_words=0) == _lib.ERR_ARG and rc(q=None) == _lib.ERR_ARG
    assert rc(R=0) == _lib.OK and rc(B=0) == _lib.OK
    assert _lib.lib.dspark_tree_attn(None, None) == _lib.ERR_ARG


def test_sample_accept_refusals():
    p = _fake()
    ok = dict(logits=p, ids=p, cu_rows=p, u=p, noise=p, n_accept=p, next_tok=p, workspace=p,
              ws_bytes=1 << 40, ld_logits=100, ld_noise=100, dtype=0, R=4, B=1, V=100, max_rows=4)

    def rc(**kw):
        return _lib.lib.dspark_sample_accept(C.byref(_lib.SampleArgs(**{**ok, **kw})), None)

    assert rc(dtype=3) == _lib.ERR_UNSUPPORTED and rc(draft=p, draft_dtype=-1) == _lib.ERR_UNSUPPORTED
    assert rc(draft=p, parent=p) == _lib.ERR_UNSUPPORTED and "draft" in _lib.last_error()
    assert rc(max_rows=1025) == _lib.ERR_UNSUPPORTED and rc(max_rows=0) == _lib.ERR_UNSUPPORTED
    assert rc(V=0) == _lib.ERR_ARG and rc(ld_logits=99) == _lib.ERR_ARG and rc(noise=None) == _lib.ERR_ARG
    assert rc(ws_bytes=0) == _lib.ERR_ARG and "workspace" in _lib.last_error()
    assert rc(B=0) == _lib.OK


def test_keep_path_and_pack_refusals():
    p = _fake()
    s = _lib.i64_array([64, 64, 8])

    def rc(n=1, d=8, es=2, kvb=1, B=1, strides=s):
        return _lib.lib.dspark_kv_keep_path(p, p, n, strides, s, p, p, p, p, None, B, 1, d, es, 8, kvb, None)

    assert rc(d=9) == _lib.ERR_UNSUPPORTED and rc(strides=_lib.i64_array([64, 64, 9])) == _lib.ERR_UNSUPPORTED
    assert rc(B=3, kvb=2) == _lib.ERR_ARG and rc(kvb=0) == _lib.ERR_ARG
    assert rc(n=0) == _lib.OK and rc(B=0) == _lib.OK
    assert _lib.lib.dspark_tree_pack(None, None, p, None, 1, 1, None, None, None, None, 0, None, None) == _lib.ERR_ARG
    assert _lib.lib.dspark_tree_pack(p, None, p, None, 1, 1, None, None, None, p, 0, None, None) == _lib.ERR_ARG


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    c = torch.zeros(1, 2, 8, 64, dtype=torch.bfloat16)
    table = rope.RopeTable(64, device="cpu")
    for call in (lambda: rope.rotate(x, table, i),
                 lambda: rope.rope_append(x, x, x, table, i, c, c, i),
                 lambda: tree.tree_sdpa(x, c, c, i, i, scale=1.0, max_nodes=2),
                 lambda: tree.pack(i, None, i, 2, 2), lambda: tree.PathKeeper([c], [c]),
                 lambda: sampling.sample_accept(x[:, 0].float(), i, i, i.float(), x[:1, 0].float(), max_rows=2)):
        with pytest.raises(DSparkUnsupported):
            call()


def test_rope_tables():
    with pytest.raises(DSparkUnsupported):
        rope.RopeTable(72, device="cpu")
    with pytest.raises(DSparkUnsupported):
        rope.RopeTable(64, 80, device="cpu")
    with pytest.raises(ValueError):
        rope.RopeTable(64, layout="spiral", device="cpu")
    with pytest.raises(ValueError):
        rope.RopeTable(64, scaling={"type": "stretch", "factor": 2}, device="cpu")
    t = rope.RopeTable(64, 32, theta=1e4, device="cpu")
    for i, f in enumerate(t.freq.tolist()):  # fixed point: the fraction of a turn a position
        assert abs((f % 2 ** 64) / 2 ** 64 - 1e4 ** (-2 * i / 32) / (2 * math.pi)) < 1e-15
    for kind, extra in (("yarn", {}), ("llama3", {"low_freq_factor": 1.0, "high_freq_factor": 4.0})):
        inv, m = rope.inv_freq(128, 1e6, {"type": kind, "factor": 4.0, "original_max_position": 8192, **extra})
        plain, _ = rope.inv_freq(128, 1e6)
        assert inv[0] == pytest.approx(plain[0]) and inv[-1] == pytest.approx(plain[-1] / 4)
        assert all(a <= b * (1 + 1e-12) and a >= b / 4 * (1 - 1e-12) for a, b in zip(inv, plain))
        assert m == pytest.approx(0.1 * math.log(4.0) + 1 if kind == "yarn" else 1.0)
    lin, _ = rope.inv_freq(64, 1e4, {"type": "linear", "factor": 2.0})
    assert lin == pytest.approx([x / 2 for x in rope.inv_freq(64, 1e4)[0]])
    ntk, _ = rope.inv_freq(64, 1e4, {"type": "ntk", "factor": 2.0})
    assert ntk[0] == 1.0 and ntk[-1] == pytest.approx(rope.inv_freq(64, 1e4)[0][-1] / 2, rel=1e-9)


def test_reference_accept_is_lossless():
    """The 64-bit form of the accept (what the kernel is held to) emits tokens distributed as p."""
    rng = np.random.default_rng(0)
    V, N = 5, 20000
    logits = rng.standard_normal((3, V))
    p = ref.probabilities(logits, 0.9)
    q = ref.probabilities(rng.standard_normal((3, V)), 1.0)
    for form in ("draft", "tree"):
        count = np.zeros(V)
        for _ in range(N):
            if form == "draft":
                ids, parent, dr = [0, int(rng.choice(V, p=q[0]))], None, q
            else:
                ids, parent, dr = [0, 1, 3], [-1, 0, 0], None
            path, tok, _ = ref.accept(p, ids, parent, rng.random(3), rng.exponential(size=V), dr, False)
            count[ids[path[1]] if len(path) > 1 else tok] += 1
        sd = np.sqrt(p[0] * (1 - p[0]) / N)
        assert (np.abs(count / N - p[0]) <= 5 * sd).all()


def test_shape_checks_of_the_python_surface():
    with pytest.raises(DSparkError):
        sampling._rows_of("logits", torch.zeros(3, 4), 2, 4)
    with pytest.raises(DSparkError):
        sampling._f32("u", torch.zeros(3, dtype=torch.float64), 3)
    assert tree.anc_words(1) == 1 and tree.anc_words(32) == 1 and tree.anc_words(33) == 2
