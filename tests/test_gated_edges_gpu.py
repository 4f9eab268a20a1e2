"""The ends of the block operators' ranges, value by value.

Where the other tests compare with a tensor's largest value, these compare every value with its own float64 one, at gates that are
nearly open or shut and at decays from almost one to almost nothing.  Tolerances count in u = 2^-24.  A gate's logistic function
is 1 / (1 + 2^t) with t = -x log2(e): rounding t and the constant costs 1.5 |x| u relative, the exponential and
the reciprocal 6 u, and so it is for 1 minus the gate, which is the function of -x.  softplus is within 8 u, the square root and its
reciprocal within 4 u, the decay's polynomial within 2 u, and a decay e^l carries l's relative error times |l|.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
TINY = 2.0**-126  # where float32 begins to lose digits


def near(got, want, rel, what, slack=TINY):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    assert got.shape == want.shape, what
    err = (got - want).abs()
    bound = rel.cpu() * want.abs() + slack if torch.is_tensor(rel) else rel * want.abs() + slack
    worst = torch.where(torch.isfinite(err), err / bound, torch.full_like(err, float("inf"))).flatten().argmax()
    assert (err <= bound).all(), f"{what}: {got.flatten()[worst]} for {want.flatten()[worst]}, {err.flatten()[worst] / bound.flatten()[worst]} of the bound"


def one_step(r, i, lam, x, gh, dt, h0=None):
    """One step per sequence of the batch, rows of the gates against columns of lam: the operator's and the definition's results.
    Without an h0 every gradient of x, r and i is a plain product: nothing cancels but what the operator makes cancel."""
    import tsfast_b200 as b

    D = lam.numel()
    wide = lambda v: v.to(dt).cuda()[:, None, None].expand(-1, 1, D).contiguous().requires_grad_()  # noqa: E731
    leaves = [wide(x), wide(r), wide(i), lam.float().cuda().requires_grad_()]
    state = torch.full((r.numel(), D), 0.0 if h0 is None else h0, device="cuda").requires_grad_()
    h, last = b.gated_recurrence(*leaves, state)
    up = wide(gh).detach()
    got = (h, last, *torch.autograd.grad((h, last), [*leaves, state], (up, torch.zeros_like(last))))
    x, r, i, lam, state, up = (t.detach().double().requires_grad_() for t in (*leaves, state, up))
    rho, shut, iota, shut_i = torch.sigmoid(r), torch.sigmoid(-r), torch.sigmoid(i), torch.sigmoid(-i)
    sp = torch.nn.functional.softplus(lam, threshold=700)
    l = -8 * sp * rho
    a, beta = torch.exp(l), torch.sqrt(-torch.expm1(2 * l))
    before = state[:, None]
    gl = up * (a * before - a * a / beta * iota * x)
    out = a * before + beta * iota * x
    return got, dict(h=out, last=out[:, 0], gx=up * beta * iota, gr=gl * l * shut, gi=up * beta * iota * x * shut_i,
                     glam=(gl * -8 * rho * torch.sigmoid(lam)).sum((0, 1)), gh0=(up * a)[:, 0], l=l, r=r, i=i, lam=lam)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
def test_gradient_of_r_at_every_gate_and_rate(dt):
    """gr has the factors l and 1 - rho.  The rates go down to where c softplus(lam) is subnormal and to nothing; sums of relative
    errors: 1.5 |r| u for rho and for 1 - rho, of which only one is not next to 1, half of it again for beta, and the constants above."""
    r = torch.tensor([-60.0, -20, -8, -2, 0, 2, 5, 8, 10, 12, 14, 15, 16, 18, 20, 40, 60])
    lam = torch.tensor([-120.0, -104, -103, -100, -95, -92, -91, -90, -60, -20, -8, -5, -2.5])
    got, want = one_step(r, torch.zeros_like(r), lam, torch.ones_like(r), torch.ones_like(r), dt)
    rel = (2.5 * want["r"].abs() + 64) * U + (0 if dt == torch.float32 else torch.finfo(dt).eps / 2 * (1 + 2.0**-7))
    # float16 steps by 2^-24 below 2^-14.  beta loses digits where beta^2 comes near the smallest normal number: gr's values there
    # are about beta / 2, 1e-19 and less
    slack = 2.0**-62 if dt != torch.float16 else 2.0**-25
    near(got[3], want["gr"].expand_as(got[3]), rel, "gr", slack)
    assert all(torch.isfinite(t).all() for t in got)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_gradient_of_i_at_every_gate(dt):
    """gi has the factor 1 - iota: the relative error is the gates' (1.5 |i| u, once) and that of the constants."""
    i = torch.tensor([-60.0, -20, -8, -2, 0, 2, 5, 8, 10, 12, 14, 15, 16, 18, 20, 40, 60])
    got, want = one_step(torch.zeros_like(i), i, torch.tensor([-20.0, -8, -5, -2.5]), torch.ones_like(i), torch.ones_like(i), dt)
    rel = (2 * want["i"].abs() + 64) * U + (0 if dt == torch.float32 else torch.finfo(dt).eps / 2 * (1 + 2.0**-7))
    near(got[4], want["gi"].expand_as(got[4]), rel, "gi")


def test_gradient_of_lam_where_its_sigmoid_and_softplus_end():
    """glam is a sum times sigmoid(lam) / softplus(lam), which tends to 1. A large state brings the gradient of a channel that
    hardly decays into sight: c softplus(lam) is subnormal from lam = -85.3 on, with 10 bits left at -96, so 2^-10."""
    r = torch.tensor([-1.0, 0, 1, 2])
    lam = torch.tensor([-96.0, -92, -90, -89, -88.5, -87, -80, -30, -17.5, -16.5, -10, -5])
    got, want = one_step(r, torch.zeros_like(r), lam, torch.zeros_like(r), torch.ones_like(r), torch.float32, 1e15)
    near(got[5], want["glam"], torch.where(want["lam"] < -85, 2.0**-10, 512 * U), "glam")


def decays():
    r = torch.tensor([-30.0, -10, -4, -1, 0, 0.5, 1, 2, 4, 8, 30])
    lam = torch.tensor([-30.0, -8, -4, -2, -1, 0, 0.5, 1, 1.5, 2, 3, 4, 6, 8, 10, 12, 20, 60, 300])
    return r, lam


def decay_bound(want):
    """The relative error of e^l: |l| times l's own (the gate's and softplus's), and a few u for the exponential."""
    return want["l"].abs() * (1.5 * want["r"].abs() + 20) * U + 8 * U


def test_decays_of_every_size():
    """A state and no input: h is the decay, and so is the gradient of h0, down to where float32 ends."""
    r, lam = decays()
    got, want = one_step(r, torch.zeros_like(r), lam, torch.zeros_like(r), torch.ones_like(r), torch.float32, 1.0)
    bound = decay_bound(want)
    near(got[0], want["h"].expand_as(got[0]), bound, "h")
    near(got[1], want["last"], bound[:, 0], "last")
    near(got[6], want["gh0"], bound[:, 0], "gh0")


def test_decays_of_every_size_in_a_step():
    import tsfast_b200 as b

    r, lam = decays()
    _, want = one_step(r, torch.zeros_like(r), lam, torch.zeros_like(r), torch.ones_like(r), torch.float32, 1.0)
    rows = r.cuda()[:, None].expand(-1, lam.numel()).contiguous()
    state = torch.ones_like(rows)
    h = b.gated_recurrence_step(torch.zeros_like(rows), rows, rows, lam.cuda(), state)
    near(h, want["last"], decay_bound(want)[:, 0], "h")
    assert torch.equal(h, state)


@pytest.mark.parametrize("packed", [False, True])
def test_layers_that_forget(packed):
    """Decays from 0.999 down to 1e-4 in one warp of channels, and no value that cancels: every term is positive, so every state is
    within the sum of its steps' errors. The same for the adjoint's carry (gh0) of a positive upstream gradient."""
    import tsfast_b200 as b
    from test_gated_gpu import definition

    L, D = 61, 96
    g = torch.Generator(device="cuda").manual_seed(11)
    rand = lambda *s: torch.rand(*s, device="cuda", generator=g)  # noqa: E731
    base = torch.logspace(-4, -0.0004345, D, device="cuda", dtype=torch.float64)
    lam = torch.log(torch.expm1(-torch.log(base) / 8)).float().requires_grad_()
    x, r, i = (rand(L, D).requires_grad_(), (6 * rand(L, D) - 3).requires_grad_(), (6 * rand(L, D) - 3).requires_grad_())
    h0, gh, gl = (10 + rand(1, D)).requires_grad_(), torch.zeros(L, D, device="cuda"), rand(1, D)
    gh[20:] = rand(L - 20, D)
    if packed:
        h, last = b.gated_recurrence(x, r, i, lam, h0, cu_seqlens=torch.tensor([0, L], device="cuda"))
    else:
        h, last = (t[0] if k == 0 else t for k, t in enumerate(b.gated_recurrence(x[None], r[None], i[None], lam, h0)))
    gh0 = torch.autograd.grad((h, last), h0, (gh, gl))[0]
    want, want_last, *grads = definition(x, r, i, lam, h0, [0, L], 8.0, gh, gl)
    # a step's decay has |l| (1.5 * 3 + 20) u + 8 u, |l| up to 9.3 * 0.96, that is 220 u where the decay is about 1e-4 and the
    # state forgets the step at once; what is remembered for long has |l| below 1: at most 33 u a step, 61 steps, and 220 u for one more
    near(h, want, (61 * 33 + 220) * U, "h")
    near(last, want_last, (61 * 33 + 220) * U, "last")
    # gh0 is a product of twenty decays and more: the sum of their |l| counts, l's error alone being (4.5 + 20) u of it
    total = (8 * torch.nn.functional.softplus(lam.detach().double()) * torch.sigmoid(r.detach().double())[:21].sum(0))[None]
    near(gh0, grads[4], (total * 25 + 21 * 8 + 61 * 33 + 220) * U, "gh0")


def test_channels_that_hardly_change():
    """beta = sqrt(1 - a^2) of a channel with a rate near the end of float32: beta^2 may lose the smallest normal number, 2^-126,
    and beta half of that relative to beta^2 (1.6e-34 at lam = -79, that is 4e-5)."""
    r = torch.tensor([-1.0, 0, 1])
    lam = torch.tensor([-79.0, -75, -70, -60])
    got, want = one_step(r, torch.zeros_like(r), lam, torch.ones_like(r), torch.ones_like(r), torch.float32)
    beta2 = -torch.expm1(2 * want["l"])
    near(got[2], want["gx"].expand_as(got[2]), 72 * U + TINY / beta2 / 2, "gx")
    near(got[0], want["h"].expand_as(got[0]), 72 * U, "h")


# one CTA per chain, clusters of several, packed sequences, either width of a lane
@pytest.mark.parametrize("dt,S,L,D,mute", [(torch.float32, 2, 100, 30, 0), (torch.bfloat16, 300, 60, 256, 1), (torch.float32, 1, 3000, 64, 3),
                                           (torch.bfloat16, 8, 2000, 1024, 2), (torch.bfloat16, 1, 2000, 40, 0)])
def test_a_wait_that_runs_out_is_reported(dt, S, L, D, mute):
    """A step whose result is kept back (the probe's mute step): the waits for it give up, the launch ends and the error word says so,
    once; what came before is right, and so is the next call."""
    import tsfast_b200 as b
    from tsfast_b200 import _lib

    lib = _lib.lib()
    g = torch.Generator(device="cuda").manual_seed(L)
    x, r, i = (torch.randn(S, L, D, device="cuda", generator=g).to(dt) for _ in range(3))
    lam = torch.randn(D, device="cuda", generator=g) - 5
    stream = _lib.stream_ptr(x.device)
    with torch.no_grad():
        want, last = b.gated_recurrence(x, r, i, lam)
    assert lib.b200_block_status(stream) == 0
    tag = {torch.float32: 0, torch.bfloat16: 2}[dt]

    def probe(mute):
        h, end = torch.zeros_like(want), torch.zeros_like(last)
        assert lib.b200_gated_probe(mute, tag, S, L, 0, D, 8.0, None, 0, *(a for t in (x, r, i) for a in (_lib.ptr(t), L * D, D)), _lib.ptr(lam),
                                    None, _lib.ptr(h), _lib.ptr(end), None, stream) == 0
        return h, end

    assert all(torch.equal(a, w) for a, w in zip(probe(-1), (want, last))) and lib.b200_block_status(stream) == 0
    h, _ = probe(mute)
    assert lib.b200_block_status(stream) == 5  # B200_ERR_TIMEOUT
    assert lib.b200_block_status(stream) == 0
    assert torch.equal(h[:, : 28 * mute], want[:, : 28 * mute])  # (later values are whatever shared memory held: the last call's, even)
    with torch.no_grad():
        again, last_again = b.gated_recurrence(x, r, i, lam)
    assert torch.equal(again, want) and torch.equal(last_again, last) and lib.b200_block_status(stream) == 0
