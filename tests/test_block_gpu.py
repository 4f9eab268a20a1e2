"""The block operators run together, as a gated recurrent block uses them, and what they refuse.

The block: y, r = residual_norm(x, r); (u, a, i, z) = y W_in; h = gated_recurrence(u, a, i); o = gated_norm(h, z) W_out; and
so on to the next.  In float32 the whole training pass is compared with float64 end to end: every operator is within
2e-5 of the largest value and the two products and two norms between them multiply that by the norms' gain and the weights'
(about one by construction), so 1e-4 per tensor.  Serving is compared with itself: a prompt followed by single tokens
gives what the whole sequence gives, up to the roundings of bfloat16 along the block.
"""

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu


def weights(D, N, dt, seed=0, layers=2):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    out = []
    for _ in range(layers):
        base = torch.rand(N, device="cuda", generator=g) * 0.2 + 0.79
        out.append({"norm": (1 + 0.1 * rand(D)).to(dt), "in": (rand(4 * N, D) / D**0.5).to(dt), "lam": torch.log(torch.expm1(-torch.log(base) / 8)),
                    "gated": (1 + 0.1 * rand(N)).to(dt), "out": (rand(D, N) / N**0.5).to(dt), "scale": (0.5 + 0.1 * rand(D)).to(dt)})
    return out, rand


def forward(layers, x, cu=None, states=None):
    """``layers`` blocks over ``x [..., D]``; returns the last residual sum and the final states."""
    import tsfast_b200 as b

    delta, r, last = torch.zeros_like(x), x, []
    for k, w in enumerate(layers):
        y, r = b.residual_norm(delta, r, w["norm"], scale=w["scale"])
        N = w["lam"].shape[0]
        u, a, i, z = (y @ w["in"].T).split(N, dim=-1)
        h, s = b.gated_recurrence(u, a, i, w["lam"], None if states is None else states[k], cu_seqlens=cu)
        delta = b.gated_norm(h, z, w["gated"]) @ w["out"].T
        last.append(s)
    return r + delta, last


def reference(layers, x, bounds):
    def rms(v, w):
        return v / torch.sqrt(v.square().mean(-1, keepdim=True) + 1e-6) * w

    delta, r = torch.zeros_like(x), x
    for w in layers:
        r = r + w["scale"] * delta
        y = rms(r, w["norm"])
        N = w["lam"].shape[0]
        u, a, i, z = (y @ w["in"].T).split(N, dim=-1)
        log_a = -8 * F.softplus(w["lam"]) * torch.sigmoid(a)
        rows = []
        for s in range(len(bounds) - 1):
            h = torch.zeros_like(u[0])
            for t in range(bounds[s], bounds[s + 1]):
                h = torch.exp(log_a[t]) * h + torch.sqrt(-torch.expm1(2 * log_a[t])) * torch.sigmoid(i[t]) * u[t]
                rows.append(h)
        h = torch.stack(rows)
        delta = rms(h, w["gated"]) * z * torch.sigmoid(z) @ w["out"].T
    return r + delta


@pytest.mark.parametrize("D,N", [(48, 96), (130, 70)])
def test_training_pass_of_two_blocks(D, N):
    layers, rand = weights(D, N, torch.float32)
    bounds = [0, 30, 31, 95]
    x, up = rand(bounds[-1], D), rand(bounds[-1], D)
    x.requires_grad_()
    params = [t.requires_grad_() for w in layers for t in w.values()]
    out, _ = forward(layers, x, torch.tensor(bounds, device="cuda", dtype=torch.int32))
    grads = torch.autograd.grad(out, [x, *params], up)
    x64 = x.detach().double().requires_grad_()
    layers64 = [{k: t.detach().double().requires_grad_() for k, t in w.items()} for w in layers]
    want = reference(layers64, x64, bounds)
    wgrads = torch.autograd.grad(want, [x64, *(t for w in layers64 for t in w.values())], up.double())
    for a, w in zip((out, *grads), (want, *wgrads)):
        assert (a.double() - w).abs().max().item() <= 1e-4 * w.abs().max().item()  # (the first scale multiplies zeros)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_prompt_then_tokens(dt):
    """A batch of prompts read in together, then token by token with a captured graph over a padded batch."""
    import tsfast_b200 as b

    D, N, B, L, T = 64, 128, 3, 40, 6
    layers, rand = weights(D, N, dt, seed=1)
    x = rand(B, L + T, D).to(dt)
    with torch.no_grad():
        whole, _ = forward(layers, x)
        _, last = forward(layers, x[:, :L])
        slots = torch.tensor([5, -1, 0, 3], device="cuda", dtype=torch.int32)  # row 1 is empty
        rows = [0, 2, 3]
        caches = [torch.zeros(7, N, device="cuda") for _ in layers]
        for c, s in zip(caches, last):
            c[slots[rows].long()] = s
        token = torch.zeros(4, D, device="cuda", dtype=dt)

        def step():
            delta, r = torch.zeros_like(token), token
            for w, c in zip(layers, caches):
                y, r = b.residual_norm(delta, r, w["norm"], scale=w["scale"])
                u, a, i, z = (y @ w["in"].T).split(N, dim=-1)
                delta = b.gated_norm(b.gated_recurrence_step(u, a, i, w["lam"], c, slots), z, w["gated"]) @ w["out"].T
            return r + delta

        start = [c.clone() for c in caches]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for c, s in zip(caches, start):
            c.copy_(s)
        for t in range(L, L + T):
            token[rows] = x[:, t]
            graph.replay()
            want = whole[:, t].double()
            # float32: as above; bfloat16: about eight roundings of 2^-9 on the way through either path, of values no larger
            # than the largest here
            tol = 1e-4 if dt == torch.float32 else 16 * 2.0**-9
            assert (out[rows].double() - want).abs().max().item() < tol * want.abs().max().item()
    for c in caches:
        assert (c[[1, 2, 4, 6]] == 0).all()


def test_quantised_projections_of_a_block():
    """The same block with its projections in 8 bits equals the block with the weights and inputs those bits stand for."""
    import tsfast_b200 as b

    D, N = 256, 384
    layers, rand = weights(D, N, torch.bfloat16, seed=2, layers=1)
    w = layers[0]
    x = rand(50, D).bfloat16()
    with torch.no_grad():
        q_in, q_out = b.quantize_weight(w["in"]), b.quantize_weight(w["out"])
        y, r = b.residual_norm(x, x, w["norm"])
        mixed = b.quant_linear(y, *q_in)
        u, a, i, z = mixed.split(N, dim=-1)
        h, _ = b.gated_recurrence(u, a, i, w["lam"])
        out = b.quant_linear(b.gated_norm(h, z, w["gated"]), *q_out)
        plain = (y.float() @ w["in"].float().T)
        # e4m3 carries 2^-4 of a value: a sum of 256 independent products of two such roundings is off by about
        # 2^-4 sqrt(2/3) of its standard deviation, and 6 of those are never reached
        assert (mixed.float() - plain).std() < 2.0**-4 * plain.std() and torch.isfinite(out).all()
        assert out.shape == (50, D)


def test_refusals():
    import tsfast_b200 as b

    x = torch.zeros(2, 5, 8, device="cuda")
    lam, cache = torch.zeros(8, device="cuda"), torch.zeros(4, 8, device="cuda")
    no = lambda text: pytest.raises(RuntimeError, match=text)  # noqa: E731
    with no("r is .* like x"):
        b.gated_recurrence(x, x[..., :4], x, lam)
    with no("i is .* like x"):
        b.gated_recurrence(x, x, x.half(), lam)
    with no("lam is"):
        b.gated_recurrence(x, x, x, lam.half())
    with no("lam is"):
        b.gated_recurrence(x, x, x, lam[:4])
    with no("h0 is"):
        b.gated_recurrence(x, x, x, lam, torch.zeros(3, 8, device="cuda"))
    with no("h0 is"):
        b.gated_recurrence(x, x, x, lam, torch.zeros(2, 8, device="cuda").half())
    with no("c=0"):
        b.gated_recurrence(x, x, x, lam, c=0)
    with no("expected 2 axes"):
        b.gated_recurrence(x, x, x, lam, cu_seqlens=torch.tensor([0, 5], device="cuda"))
    with no("cu_seqlens is"):
        b.gated_recurrence(x[0], x[0], x[0], lam, cu_seqlens=torch.tensor([0.0, 5.0], device="cuda"))
    with no("cu_seqlens is"):
        b.gated_recurrence(x[0], x[0], x[0], lam, cu_seqlens=torch.tensor([0, 5]))
    with no("at least one boundary"):
        b.gated_recurrence(x[0], x[0], x[0], lam, cu_seqlens=torch.zeros(0, dtype=torch.int32, device="cuda"))
    with no("at least one channel"):
        b.gated_recurrence(x[..., :0], x[..., :0], x[..., :0], lam[:0])
    with no("expected at least"):
        b.gated_recurrence(lam, lam, lam, lam)
    t = x[:, 0]
    with no("state is"):
        b.gated_recurrence_step(t, t, t, lam, cache.half())
    with no("updated in place"):
        b.gated_recurrence_step(t, t, t, lam, torch.zeros(8, 4, device="cuda").T)
    with no("updated in place"):
        b.gated_recurrence_step(t, t, t, lam, cache[:1].expand(4, 8))
    with no("slots for"):
        b.gated_recurrence_step(t, t, t, lam, cache, torch.zeros(3, dtype=torch.int32, device="cuda"))
    with no("without slots"):
        b.gated_recurrence_step(t, t, t, lam, cache[:1])
    with no("no gradient"):
        b.gated_recurrence_step(t.clone().requires_grad_(), t, t, lam, cache)
    w = torch.ones(8, device="cuda")
    with no("residual is .* like x"):
        b.residual_norm(x, x[:1], w)
    with no("gate is .* like x"):
        b.gated_norm(x, x.half(), w)
    with no("weight is"):
        b.gated_norm(x, x, w[:4])
    with no("post_weight is .*float16"):
        b.residual_norm(x.bfloat16(), x.bfloat16(), w.bfloat16(), post_weight=w.half())
    with no("while other parameters"):
        b.residual_norm(x.bfloat16(), x.bfloat16(), w, scale=w.bfloat16())
    with no("RMS norm has none"):
        b.gated_norm(x, x, w, w)
    with no("the kernel takes 1 to 8192"):
        b.gated_norm(torch.zeros(1, 8200, device="cuda"), None, torch.ones(8200, device="cuda"))
    with no("eps="):
        b.gated_norm(x, x, w, eps=-1.0)
    with no("weight is required"):
        b.gated_norm(x, x, None)
    q, s = b.quantize_weight(torch.randn(16, 8, device="cuda"))
    with no("expected bfloat16 or float16"):
        b.quant_linear(x, q, s)
    with no("q is"):
        b.quant_linear(x.half(), q[:, :4], s)
    with no("q is"):
        b.quant_linear(x.half(), q.float(), s)
    with no("scale is"):
        b.quant_linear(x.half(), q, s.half())
    with no("bias is"):
        b.quant_linear(x.half(), q, s, torch.zeros(16, device="cuda").bfloat16())
    with no("w is"):
        b.quantize_weight(torch.zeros(4, 0, device="cuda"))


def test_second_derivatives_are_refused():
    import tsfast_b200 as b

    x = torch.randn(1, 6, 4, device="cuda", requires_grad=True)
    lam = torch.zeros(4, device="cuda", requires_grad=True)
    h, _ = b.gated_recurrence(x, x, x, lam)
    (g,) = torch.autograd.grad(h.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(g.sum(), x)
    (g,) = torch.autograd.grad(b.gated_norm(x, x, lam + 1).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(g.sum(), x)


def test_boundaries_that_are_wrong_stay_in_bounds():
    """Decreasing boundaries and ones past the buffer give some values, touch nothing else and leave right sequences right."""
    import tsfast_b200 as b

    T, D = 40, 20
    pool = torch.full((3 * T, D), 5.0, device="cuda")
    x = pool[T : 2 * T].normal_()
    lam = torch.zeros(D, device="cuda")
    right, _ = b.gated_recurrence(x, x, x, lam, cu_seqlens=torch.tensor([0, 10, 30], device="cuda"))
    for bounds in ([0, 10, 1000], [0, 10, 5], [-7, 10, 30], [0, 10, 2**40]):
        h, last = b.gated_recurrence(x, x, x, lam, cu_seqlens=torch.tensor(bounds, device="cuda"))
        if bounds[0] == 0:
            assert torch.equal(h[:5], right[:5])
        assert torch.isfinite(last).all()
    assert (pool[:T] == 5).all() and (pool[2 * T :] == 5).all()


def test_error_words_read_zero():
    import tsfast_b200 as b
    from tsfast_b200 import _lib

    x = torch.randn(1, 5000, 64, device="cuda").half()  # several CTAs per chain
    with torch.no_grad():
        b.gated_recurrence(x, x, x, torch.zeros(64, device="cuda"))
        b.quant_linear(x, *b.quantize_weight(torch.randn(640, 64, device="cuda")))
    assert _lib.lib().b200_block_status(_lib.stream_ptr(x.device)) == 0
    b.track_status(True)
    try:
        b.check_status()
    finally:
        b.track_status(False)


def test_quantised_block_against_what_the_bits_stand_for():
    """Both projections of the 8-bit block, each against float64 products of the quantised rows that go in and the weights that the
    bits stand for: the second's rows are what the recurrence and the gated norm made of the first's results."""
    import tsfast_b200 as b
    from test_quant_gpu import check

    D, N = 256, 384
    layers, rand = weights(D, N, torch.bfloat16, seed=2, layers=1)
    w = layers[0]
    x = rand(50, D).bfloat16()
    with torch.no_grad():
        q_in, q_out = b.quantize_weight(w["in"]), b.quantize_weight(w["out"])
        y, _ = b.residual_norm(x, x, w["norm"])
        mixed = b.quant_linear(y, *q_in)
        u, a, i, z = mixed.split(N, dim=-1)
        h, _ = b.gated_recurrence(u, a, i, w["lam"], cu_seqlens=torch.tensor([0, 20, 50], device="cuda"))
        inner = b.gated_norm(h, z, w["gated"])
        check(y, *q_in, None, mixed)
        check(inner, *q_out, None, b.quant_linear(inner, *q_out))
