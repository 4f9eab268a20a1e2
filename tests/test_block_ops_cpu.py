"""The block operators without a GPU: the host path loads and knows its entry points, refuses CPU tensors and wrong types by
name, and the C entry points reject bad arguments before any CUDA call."""

import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def built():
    from tsfast_b200 import _lib, build

    build.build()
    build.build_host()
    return _lib


def test_host_path_binds_every_entry_it_names(built):
    host = built.host()
    assert set(host.entries()) <= set(built.SIGNATURES)
    assert {"b200_gated_fwd", "b200_block_norm_fwd", "b200_quant_linear"} <= set(host.entries())


def test_cpu_tensors_and_types_are_refused(built):
    import tsfast_b200 as b

    x, w = torch.zeros(2, 5, 8), torch.zeros(8)
    calls = [("gated_recurrence", lambda t: b.gated_recurrence(t, t, t, w)),
             ("gated_recurrence_step", lambda t: b.gated_recurrence_step(t[0], t[0], t[0], w, torch.zeros(5, 8))),
             ("gated_norm", lambda t: b.gated_norm(t, t, w)),
             ("residual_norm", lambda t: b.residual_norm(t, t, w))]
    for name, call in calls:
        with pytest.raises(RuntimeError, match=f"b200scan::{name}: .*CUDA"):
            call(x)
        with pytest.raises(RuntimeError, match=f"b200scan::{name}: .*(float32|CUDA)"):
            call(x.double())
    with pytest.raises(RuntimeError, match="b200scan::quantize_weight: .*CUDA"):
        b.quantize_weight(x[0])
    with pytest.raises(RuntimeError, match="b200scan::quant_linear: .*CUDA"):
        b.quant_linear(x.bfloat16(), torch.zeros(4, 8).to(torch.float8_e4m3fn), torch.ones(1, 1))
    with pytest.raises(RuntimeError, match="kind"):
        b.gated_norm(x, x, w, kind="batch")
    with pytest.raises(RuntimeError, match="activation"):
        b.residual_norm(x, x, w, activation="tanh")
    with pytest.raises(RuntimeError, match="post_bias without post_weight"):
        b.residual_norm(x, x, w, post_bias=w)


def test_c_entry_points_reject_bad_arguments(built):
    L = built.lib()
    z, a = ctypes.c_void_p(None), ctypes.c_void_p(1 << 20)  # never dereferenced
    seq = (a, 8, 8)

    def fwd(dtype=2, S=1, L_=4, T=0, D=8, cu=z, x=seq, lam=a, h=a, last=a):
        return L.b200_gated_fwd(dtype, S, L_, T, D, 8.0, cu, 0, *x, *seq, *seq, lam, z, h, last, z, z)

    assert fwd(dtype=1) == 1 and fwd(dtype=9) == 1 and fwd(D=0) == 1 and fwd(S=-1) == 1
    assert fwd(x=(z, 8, 8)) == 1 and fwd(lam=z) == 1 and fwd(h=z) == 1 and fwd(last=z) == 1
    assert fwd(x=(ctypes.c_void_p((1 << 20) + 1), 8, 8)) == 1  # not aligned to an element
    assert fwd(S=0) == 0
    bwd = (2, 1, 4, 0, 8, 8.0, z, 0, *seq, *seq, *seq, a, a, *seq, z, a, a, a, a, z)
    assert L.b200_gated_bwd(*bwd, z, 0, z) == 2 and L.b200_gated_bwd(*bwd, a, 16, z) == 2
    step = lambda dtype=2, B=1, n=4, pitch=8, slots=a, state=a: L.b200_gated_step(  # noqa: E731
        dtype, B, 8, n, 8.0, a, 8, a, 8, a, 8, a, state, pitch, slots, 0, a, z)
    assert step(dtype=1) == 1 and step(pitch=7) == 1 and step(state=z) == 1 and step(B=5, slots=z) == 1 and step(B=0) == 0 and step(B=70000) == 4

    def norm(dtype=0, D=8, kind=0, act=1, eps=1e-6, x=a, res=a, w1=a, b1=z, w2=a, b2=z):
        return L.b200_block_norm_fwd(dtype, 3, D, kind, act, eps, 1, x, 8, z, 0, res, 8, w1, b1, z, w2, b2, a, a, z, z)

    assert norm(dtype=1) == 1 and norm(D=0) == 1 and norm(D=8193) == 4 and norm(kind=2) == 1 and norm(act=3) == 1 and norm(eps=-1.0) == 1
    assert norm(x=z) == 1 and norm(res=z) == 1 and norm(b2=a) == 1 and norm(kind=1, w1=z, b1=a) == 1 and norm(w1=z, w2=z) == 1
    assert norm(eps=float("nan")) == 1
    lin = lambda dtype=2, M=4, K=32, q=a, ldq=32, ldy=16, ws=z, nb=0: L.b200_quant_linear(  # noqa: E731
        dtype, M, 16, K, a, 32, q, ldq, a, z, 0, a, ldy, ws, nb, z)
    assert lin(dtype=0) == 1 and lin(ldq=40) == 1 and lin(ldq=16) == 1 and lin(ldy=15) == 1 and lin(K=0) == 1 and lin(M=0) == 0
    assert lin(q=ctypes.c_void_p((1 << 20) + 8)) == 1 and lin() == 2 and lin(ws=a, nb=100) == 2
    assert L.b200_quant_weight(1, 4, 4, a, 4, a, 4, a, z) == 1 and L.b200_quant_weight(0, 4, 4, a, 4, a, 3, a, z) == 1


@pytest.mark.parametrize("dtype,tag,tile", [(torch.float32, 0, 28), (torch.bfloat16, 2, 28), (torch.float16, 3, 28)])
def test_kept_states_of_the_fake_op_match_the_library(built, dtype, tag, tile):
    """torch.compile plans with the fake op's sizes: they have to be the library's."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    from tsfast_b200 import gated_b200

    L = built.lib()
    with FakeTensorMode():
        for B, steps in ((1, 1), (3, tile), (2, tile + 1), (4, 1000), (2, 0)):
            x = torch.empty(B, steps, 6, dtype=dtype)
            assert gated_b200._gated_op(x, x, x, torch.empty(6), None, None, 8.0)[2].shape[0] == L.b200_gated_chk_rows(tag, B, steps, 0, 0)
        for S, T in ((1, 1), (5, 777), (1, 0)):
            x, cu = torch.empty(T, 6, dtype=dtype), torch.empty(S + 1, dtype=torch.int32)
            assert gated_b200._gated_op(x, x, x, torch.empty(6), None, cu, 8.0)[2].shape[0] == L.b200_gated_chk_rows(tag, S, 0, T, 1)


def test_packed_tiles_never_share_a_slot(built):
    """The slot of a tile is boundary / tile + sequence + tile's number: distinct and inside the buffer for any boundaries."""
    import random

    rng = random.Random(0)
    for tile, tag in ((28, 0), (28, 2)):
        for _ in range(300):
            T = rng.randrange(0, 700)
            cu = sorted(rng.choices(range(T + 1), k=rng.randrange(1, 9)))
            used = [cu[s] // tile + s + k for s in range(len(cu) - 1) for k in range(-(-(cu[s + 1] - cu[s]) // tile))]
            assert len(set(used)) == len(used) and all(u < built.lib().b200_gated_chk_rows(tag, len(cu) - 1, 0, T, 1) for u in used)


def test_norms_without_their_weight_are_refused_on_every_way(built):
    """The custom op checks like the eager call: without a weight it would leave its result unwritten."""
    from tsfast_b200 import norm_b200

    x, w = torch.zeros(3, 8), torch.ones(8)
    with pytest.raises(RuntimeError, match="weight is required"):
        norm_b200._norm_op(x, x, None, w, None, None, None, None, 0, 1, 1e-6)
    with pytest.raises(RuntimeError, match="weight is required"):
        norm_b200._norm_op(x, None, x, None, None, None, None, None, 0, 1, 1e-6)
    with pytest.raises(RuntimeError, match="post_bias without post_weight"):
        norm_b200._norm_op(x, x, None, None, w, None, w, None, 1, 1, 1e-6)
    with pytest.raises(RuntimeError, match="residual is required"):
        norm_b200._norm_op(x, None, None, None, None, None, w, None, 0, 1, 1e-6)


def test_c_entry_points_refuse_pointers_off_their_elements(built):
    """A pointer that is not on its element's boundary (or on 16 bytes, for the statistics) would fault on the device."""
    L = built.lib()
    z, base = ctypes.c_void_p(None), 1 << 20  # never dereferenced
    at = lambda off=0: ctypes.c_void_p(base + off)  # noqa: E731

    def norm_fwd(dtype=2, pf32=1, **off):
        o = lambda n: at(off.get(n, 0))  # noqa: E731
        return L.b200_block_norm_fwd(dtype, 3, 8, 1, 1, 1e-6, pf32, o("x"), 8, o("gate"), 8, o("residual"), 8, o("w1"), o("b1"), o("scale"), o("w2"),
                                     o("b2"), o("y"), o("residual_out"), o("stats"), z)

    def norm_bwd(dtype=2, pf32=1, **off):
        o = lambda n: at(off.get(n, 0))  # noqa: E731
        return L.b200_block_norm_bwd(dtype, 3, 8, 1, 1, 1e-6, pf32, o("gy"), 8, o("gres"), 8, o("x"), 8, o("gate"), 8, o("residual"), 8, o("w1"), o("b1"),
                                     o("scale"), o("w2"), o("b2"), o("stats"), o("gx"), o("ggate"), o("gresidual"), o("gw1"), o("gb1"), o("gscale"),
                                     o("gw2"), o("gb2"), at(), 1 << 30, z)

    rows, params = ("x", "gate", "residual"), ("w1", "b1", "scale", "w2", "b2")
    for name in (*rows, "y", "residual_out"):
        assert norm_fwd(**{name: 1}) == 1 and norm_fwd(dtype=0, **{name: 2}) == 1, name
    for name in (*rows, "gy", "gres", "gx", "ggate", "gresidual"):
        assert norm_bwd(**{name: 1}) == 1 and norm_bwd(dtype=0, **{name: 2}) == 1, name
    for name in params:
        assert norm_fwd(**{name: 2}) == 1 and norm_fwd(pf32=0, **{name: 1}) == 1 and norm_bwd(**{name: 2}) == 1, name
    for name in ("gw1", "gb1", "gscale", "gw2", "gb2"):
        assert norm_bwd(**{name: 2}) == 1 and norm_bwd(pf32=0, **{name: 1}) == 1, name
    for off in (4, 8):
        assert norm_fwd(stats=off) == 1 and norm_bwd(stats=off) == 1

    seq = (at(), 8, 8)

    def fwd(cu=z, cu64=0, **off):
        o = lambda n: at(off.get(n, 0))  # noqa: E731
        return L.b200_gated_fwd(2, 1, 4, 4, 8, 8.0, cu, cu64, *seq, *seq, *seq, o("lam"), o("h0"), o("h"), o("last"), o("chk"), z)

    for name in ("lam", "h0", "last", "chk"):
        assert fwd(**{name: 2}) == 1, name
    assert fwd(h=1) == 1 and fwd(cu=at(2)) == 1 and fwd(cu=at(4), cu64=1) == 1

    def bwd(cu=z, cu64=0, **off):
        o = lambda n: at(off.get(n, 0))  # noqa: E731
        return L.b200_gated_bwd(2, 1, 4, 4, 8, 8.0, cu, cu64, *seq, *seq, *seq, o("lam"), o("chk"), *seq, o("glast"), o("gx"), o("gr"), o("gi"), o("glam"),
                                o("gh0"), at(), 1 << 30, z)

    for name in ("lam", "chk", "glast", "glam", "gh0"):
        assert bwd(**{name: 2}) == 1, name
    assert bwd(gr=1) == 1 and bwd(cu=at(2)) == 1 and bwd(cu=at(4), cu64=1) == 1

    def step(slots64=0, **off):
        o = lambda n: at(off.get(n, 0))  # noqa: E731
        return L.b200_gated_step(2, 1, 8, 4, 8.0, o("x"), 8, o("r"), 8, o("i"), 8, o("lam"), o("state"), 8, o("slots"), slots64, o("h"), z)

    assert step(x=1) == step(h=1) == step(lam=2) == step(state=2) == step(slots=2) == step(slots64=1, slots=4) == 1

    def lin(bias_f32=1, **off):
        o = lambda n: at(off.get(n, 0))  # noqa: E731
        return L.b200_quant_linear(2, 4, 16, 32, o("x"), 32, o("q"), 32, o("scale"), o("bias"), bias_f32, o("y"), 16, at(), 1 << 30, z)

    assert lin(x=1) == lin(y=1) == lin(scale=2) == lin(bias=2) == lin(bias_f32=0, bias=1) == 1
    weight = lambda dtype=0, w=0, scale=0: L.b200_quant_weight(dtype, 4, 4, at(w), 4, at(), 4, at(scale), z)  # noqa: E731
    assert weight(w=2) == weight(dtype=2, w=1) == weight(scale=2) == 1


def test_host_path_is_built_again_for_another_torch(built, monkeypatch, tmp_path):
    import shutil

    from tsfast_b200 import build

    copy = tmp_path / build.HOST_LIB.name
    shutil.copy2(build.HOST_LIB, copy)
    monkeypatch.setattr(build, "HOST_LIB", copy)
    runs = []

    class Done:
        returncode = 0

    monkeypatch.setattr(build.subprocess, "run", lambda cmd, **kw: runs.append(cmd) or Done)
    assert build.host_is_current()
    build.build_host()
    assert not runs
    monkeypatch.setattr(torch, "__version__", "2.0.0")
    assert not build.host_is_current()
    build.build_host()
    assert len(runs) == 1 and any("torch 2.0.0" in a for a in runs[0])
    monkeypatch.setattr(built, "_HOST", None)
    with pytest.raises(RuntimeError, match="another torch"):
        built.host()
