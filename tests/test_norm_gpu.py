"""The block norms (norm_b200) against their definition in float64, values and gradients.

Tolerances, as max|a-b| / max|b| per tensor: 1e-5 in float32 (row sums of at most 8192 terms and approximate exponentials
and reciprocals within a few 2^-23, as in the other norm's test), plus half a unit in the last place (eps / 2) of
the value where a result is rounded to 16 bits.  Parameter gradients, sums over the rows, repeat bit for bit.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def norm(v, w, b, kind, eps):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v / torch.sqrt(v.square().mean(-1, keepdim=True) + eps) * w
    return v if b is None else v + b


def act(g, name):
    return g * torch.sigmoid(g) if name == "silu" else torch.sigmoid(g) if name == "sigmoid" else torch.ones_like(g)


def define(v, residual, kind, activation, eps):
    """(y,) of the gated norm or (y, r) of the residual norm, from a dict of float64 tensors (None where absent)."""
    m = v["x"]
    w, b = ("post_weight", "post_bias") if residual else ("weight", "bias")
    if v[w] is not None:
        m = norm(m, v[w], v[b], kind, eps)
    if v["gate"] is not None:
        m = m * act(v["gate"], activation)
    if not residual:
        return (m,)
    r = v["residual"] + (m if v["scale"] is None else v["scale"] * m)
    return norm(r, v["weight"], v["bias"], kind, eps), r


def close(got, want, dt, what, tol=1e-5, slack=1e-30):
    got, want = got.detach().double(), want.detach().double()
    assert got.shape == want.shape, what
    if not want.numel():
        return
    tol += 0 if dt == torch.float32 else torch.finfo(dt).eps / 2
    err, top = (got - want).abs().max().item(), want.abs().max().item()
    assert err <= tol * top + slack, f"{what}: {err} of {top}"


def make(shape, dt, pdt, names, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    t = dict.fromkeys(("x", "residual", "gate", "post_weight", "post_bias", "scale", "weight", "bias"))
    for n in names:
        rows = n in ("x", "residual", "gate")
        v = rand(*shape) * 2 + 0.5 if rows else rand(shape[-1]) * 0.3 + (0.0 if "bias" in n else 0.7)
        t[n] = v.to(dt if rows else pdt).requires_grad_()
    return t, rand


def call(t, residual, **kw):
    import tsfast_b200 as b

    if not residual:
        return (b.gated_norm(t["x"], t["gate"], t["weight"], t["bias"], **kw),)
    return b.residual_norm(t["x"], t["residual"], t["weight"], t["bias"], gate=t["gate"], scale=t["scale"], post_weight=t["post_weight"],
                           post_bias=t["post_bias"], **kw)


def cancelled(v, residual, kind, activation, eps, ups):
    """What rounding may leave of a gradient that cancels.  A norm's gradient is rstd (g w - mean - hat mean(g w hat)),
    which in a row of one or two features is a small difference of terms of size T = rstd |g w|: four float32 roundings of
    each term (the product, hat twice over, the sum) leave up to 8 * 2^-24 T whatever the difference is.  The terms of
    the inner norm come out of the outer one times |scale act w|; sums add them over the rows."""
    top = lambda t: 1.0 if t is None else t.abs().max().item()  # noqa: E731
    spread = lambda t: (1 / torch.sqrt((t - t.mean(-1, keepdim=True) if kind == "layer" else t).square().mean(-1) + eps)).max().item()  # noqa: E731
    T = top(ups[0])
    gate = 1.0 if v["gate"] is None else act(v["gate"], activation).abs().max().item()
    if residual:
        T = T * top(v["weight"]) * spread(define(v, True, kind, activation, eps)[1].detach()) + top(ups[1])
    inner = v["post_weight" if residual else "weight"]
    T = max(T, T * top(v["scale"]) * max(gate, 1.0) * top(inner) * spread(v["x"].detach()))
    return 8 * 2.0**-24 * T * v["x"].numel() / v["x"].shape[-1]


def compare(shape, dt, pdt, names, residual, kind, activation, seed=0, eps=1e-5):
    t, rand = make(shape, dt, pdt, names, seed)
    outs = call(t, residual, kind=kind, eps=eps, activation=activation)
    ups = [rand(*shape).to(dt) for _ in outs]
    leaves = [t[n] for n in names]
    grads = torch.autograd.grad(outs, leaves, ups)
    v = {n: None if x is None else x.detach().double().requires_grad_() for n, x in t.items()}
    want = define(v, residual, kind, activation, eps)
    wgrads = torch.autograd.grad(want, [v[n] for n in names], [u.double() for u in ups], allow_unused=True, materialize_grads=True)
    for k, (a, w) in enumerate(zip(outs, want)):
        close(a, w, dt, f"out {k} {shape} {names}")
    slack = cancelled(v, residual, kind, activation, eps, ups) if shape[-1] <= 2 else 1e-30
    for n, a, w in zip(names, grads, wgrads):
        assert a.dtype == t[n].dtype
        close(a, w, a.dtype, f"grad {n} {shape} {names} {kind}", 2e-5, slack)
    again = torch.autograd.grad(call(t, residual, kind=kind, eps=eps, activation=activation), leaves, ups)
    assert all(torch.equal(p, q) for p, q in zip(grads, again))
    with torch.no_grad():
        plain = call(t, residual, kind=kind, eps=eps, activation=activation)
    assert all(torch.equal(p, q) for p, q in zip(outs, plain))


SHAPES = [(1, 1), (3, 2), (5, 31), (2, 3, 128), (70, 130), (9, 256), (4, 257), (300, 512), (33, 1000), (17, 1003), (5, 2048), (7, 4096),
          (3, 4098), (4, 8192), (2, 8191)]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("shape", SHAPES)
def test_all_parts(shape, kind, dt):
    # a row of one feature has no variance: its mean norm is 0 / sqrt(eps), whose slope is what rounding makes of it
    if shape[-1] == 1 and kind == "layer":
        shape = (shape[0], 5)
    bias = ["bias"] if kind == "layer" else []
    compare(shape, dt, dt, ["x", "gate", "weight"] + bias, False, kind, "silu", seed=sum(shape))
    compare(shape, dt, dt, ["x", "residual", "gate", "post_weight", "scale", "weight"] + bias + (["post_bias"] if bias else []), True, kind,
            "silu", seed=sum(shape) + 1)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("activation", ["silu", "sigmoid", None])
@pytest.mark.parametrize("width", [96, 700])
def test_parts_left_out(width, activation, dt):
    shape = (41, width)
    for kind in ("rms", "layer"):
        compare(shape, dt, torch.float32, ["x", "weight"], False, kind, activation)
        compare(shape, dt, torch.float32, ["x", "gate", "weight"], False, kind, activation)
        for extra in ([], ["gate"], ["scale"], ["post_weight"], ["gate", "scale"], ["gate", "post_weight"], ["post_weight", "scale"]):
            compare(shape, dt, torch.float32, ["x", "residual", "weight"] + extra, True, kind, activation)
    compare(shape, dt, dt, ["x", "residual", "weight", "bias", "post_weight"], True, "layer", activation)


@pytest.mark.parametrize("dt", DTYPES)
def test_many_rows_sum_in_order(dt):
    compare((20011, 64), dt, torch.float32, ["x", "residual", "gate", "post_weight", "scale", "weight"], True, "rms", "silu")
    compare((3001, 640), dt, torch.float32, ["x", "gate", "weight", "bias"], False, "layer", "sigmoid")


@pytest.mark.parametrize("D,off", [(64, 0), (63, 1), (260, 4), (1000, 2)])
def test_strided_rows_give_what_dense_ones_give(D, off):
    """Rows that do not start on a boundary are added up in another order, so their results may round the other way: one
    unit in the last place (eps) of the largest value."""
    import tsfast_b200 as b

    wide = torch.randn(50, 3 * D + off + 3, device="cuda", dtype=torch.bfloat16)
    x, res, gate = (wide[:, off + k * D : off + (k + 1) * D].requires_grad_() for k in range(3))
    w = torch.randn(D, device="cuda", dtype=torch.bfloat16)
    dense = [t.detach().clone().contiguous().requires_grad_() for t in (x, res, gate)]
    got = b.residual_norm(x, res, w, gate=gate, post_weight=w)
    want = b.residual_norm(dense[0], dense[1], w, gate=dense[2], post_weight=w)
    up = torch.randn(D, 50, device="cuda", dtype=torch.bfloat16).T  # column stride 50
    gg = torch.autograd.grad(got, (x, res, gate), (up, up[:1].expand(50, D)))
    wg = torch.autograd.grad(want, dense, (up.contiguous(), up[:1].expand(50, D).contiguous()))
    for p, q in zip((*got, *gg), (*want, *wg)):
        close(p, q, torch.float32, f"{D} at {off}", torch.finfo(torch.bfloat16).eps)


def test_only_one_result_is_used():
    import tsfast_b200 as b

    x, res, w = (torch.randn(s, device="cuda", requires_grad=True) for s in ((6, 40), (6, 40), (40,)))
    y, r = b.residual_norm(x, res, w)
    gx, gres = torch.autograd.grad(r.sum(), (x, res), retain_graph=True)
    assert torch.equal(gx, torch.ones_like(x)) and torch.equal(gres, torch.ones_like(x))
    gx, gres, gw = torch.autograd.grad(y.sum(), (x, res, w), retain_graph=True)
    (y.sum() + 0 * r.sum()).backward()
    assert torch.equal(x.grad, gx) and torch.equal(res.grad, gres) and torch.equal(w.grad, gw)
    x.grad.zero_()  # the two gradients do not share their memory
    assert torch.equal(res.grad, gres) and res.grad.abs().sum() > 0


def test_values_far_out():
    """A NaN or an infinity stays in its row; a row of zeros gives zeros; a large mean costs the variance nothing."""
    import tsfast_b200 as b

    x = torch.randn(6, 300, device="cuda")
    w = torch.rand(300, device="cuda") + 0.5
    x[1, 7], x[3, 9], x[4] = float("nan"), float("inf"), 0
    y = b.gated_norm(x, None, w)
    assert torch.isnan(y[1]).all() and torch.isnan(y[3, 9]) and (y[4] == 0).all() and torch.isfinite(y[[0, 2, 4, 5]]).all()
    far = torch.randn(4, 512, device="cuda") + 1000
    close(b.gated_norm(far, None, torch.ones(512, device="cuda"), kind="layer"), norm(far.double(), 1.0, None, "layer", 1e-6), torch.float32,
          "large mean", 1e-4)  # 1000 in float32 is known to 3e-5, the deviations are about 1


def test_no_rows():
    import tsfast_b200 as b

    x = torch.randn(0, 64, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    y, r = b.residual_norm(x, x, w, scale=w)
    gw = torch.autograd.grad(y.sum() + r.sum(), w)[0]
    assert y.shape == r.shape == (0, 64) and (gw == 0).all()


def test_replays_from_a_graph():
    import tsfast_b200 as b

    x, res, gate = (torch.randn(70, 640, device="cuda", dtype=torch.bfloat16, requires_grad=True) for _ in range(3))
    w = torch.randn(640, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    up = torch.randn(70, 640, device="cuda", dtype=torch.bfloat16)

    def passing():
        outs = b.residual_norm(x, res, w, gate=gate, scale=w, post_weight=w)
        return (*outs, *torch.autograd.grad(outs, (x, res, gate, w), (up, up)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            want = [t.detach().clone() for t in passing()]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = passing()
    for _ in range(2):
        graph.replay()
        assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_opcheck_and_compile():
    import tsfast_b200 as b
    from tsfast_b200 import norm_b200 as nb

    x, res, gate = (torch.randn(9, 24, device="cuda", requires_grad=True) for _ in range(3))
    w = torch.randn(24, device="cuda", requires_grad=True)
    utils = ("test_schema", "test_faketensor", "test_autograd_registration")
    torch.library.opcheck(nb._norm_op, (x, res, gate, w, None, w, w, None, 0, 1, 1e-6), test_utils=utils)
    torch.library.opcheck(nb._norm_op, (x, None, gate, w, w, None, None, None, 1, 2, 1e-6), test_utils=utils)

    def seam(x, res, gate, w):
        y, r = b.residual_norm(x, res, w, gate=gate, scale=w)
        return (y * r).sum()

    args = (x, res, gate, w)
    eager = torch.autograd.grad(seam(*args), args)
    compiled = torch.autograd.grad(torch.compile(seam, fullgraph=True, backend="aot_eager")(*args), args)
    assert all(torch.equal(p, q) for p, q in zip(eager, compiled))


@pytest.mark.parametrize("activation", ["sigmoid", "silu"])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("width", [24, 200, 1003])
def test_gradient_of_a_gate_at_every_opening(width, dt, activation):
    """Value by value: the gate's gradient has the logistic function's slope s (1 - s), whose second factor goes to nothing where the gate is
    open. u = 2^-24; s and 1 - s, the function of the other sign, are each within 1.5 |g| u and 8 u, the norm and the products
    within 32 u; SiLU's slope s + g s (1 - s) adds terms of up to |g|."""
    import tsfast_b200 as b

    g = torch.tensor([-60.0, -20, -12, -8, -2, 0, 2, 5, 8, 10, 12, 14, 15, 16, 18, 20, 40, 60], device="cuda")
    gate = g.to(dt)[:, None].expand(-1, width).contiguous().requires_grad_()
    x = (torch.rand(len(g), width, device="cuda", generator=torch.Generator(device="cuda").manual_seed(width)) + 0.5).to(dt)
    w, up = torch.ones(width, device="cuda", dtype=dt), torch.ones_like(x)
    (got,) = torch.autograd.grad(b.gated_norm(x, gate, w, activation=activation), gate, up)
    v, x64 = gate.detach().double(), x.double()
    s, shut = torch.sigmoid(v), torch.sigmoid(-v)
    slope = s * shut if activation == "sigmoid" else s * (1 + v * shut)
    want = x64 / torch.sqrt(x64.square().mean(-1, keepdim=True) + 1e-6) * slope
    rel = (4 * v.abs() + 64) * 2.0**-24 + (0 if dt == torch.float32 else torch.finfo(dt).eps / 2 * (1 + 2.0**-7))
    err = (got.double() - want).abs() / (rel * want.abs())
    assert (err <= 1).all(), f"gate {v.flatten()[err.argmax()]}: {got.flatten()[err.argmax()]} for {want.flatten()[err.argmax()]}"
