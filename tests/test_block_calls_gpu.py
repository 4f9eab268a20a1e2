"""What the block operators' host path does beside a plain eager call: calls that are recorded or interpreted (a tracer, a
dispatch mode, fake tensors), derivatives that do not exist, tensors of inference mode, constants that float32 does not hold.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu


def tensors(dt=torch.float32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x, r, i = (torch.randn(2, 37, 24, device="cuda", generator=g).to(dt) for _ in range(3))
    lam = torch.randn(24, device="cuda", generator=g) - 3
    w = torch.rand(24, device="cuda", generator=g).to(dt) + 0.5
    return x, r, i, lam, w


def calls(q=None):
    """Every operator as a function of (x, r, i, lam, w), tensors of [2, 37, 24]."""
    import tsfast_b200 as b

    q = q or b.quantize_weight(torch.randn(40, 24, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)))
    cu = torch.tensor([0, 30, 74], device="cuda")

    def step(x, r, i, lam, w):
        state = torch.ones(37, 24, device="cuda") * lam
        return b.gated_recurrence_step(x[0], r[0], i[0], lam, state), state

    return {"recurrence": lambda x, r, i, lam, w: b.gated_recurrence(x, r, i, lam),
            "recurrence 4-d": lambda x, r, i, lam, w: b.gated_recurrence(x[None], r[None], i[None], lam, lam.expand(1, 2, 24)),
            "recurrence packed": lambda x, r, i, lam, w: b.gated_recurrence(x.reshape(74, 24), r.reshape(74, 24), i.reshape(74, 24), lam, cu_seqlens=cu),
            "step": step,
            "gated_norm": lambda x, r, i, lam, w: b.gated_norm(x, r, w),
            "residual_norm": lambda x, r, i, lam, w: b.residual_norm(x, i, w, gate=r, scale=w),
            "quant_linear": lambda x, r, i, lam, w: b.quant_linear(x.half(), *q),
            "quantize_weight": lambda x, r, i, lam, w: tuple(t.float() for t in b.quantize_weight(x[0]))}


NAMES = ["recurrence", "recurrence 4-d", "recurrence packed", "step", "gated_norm", "residual_norm", "quant_linear", "quantize_weight"]


def flat(out):
    return [out] if torch.is_tensor(out) else list(out)


@pytest.mark.parametrize("name", NAMES)
def test_a_traced_call_runs_the_operator(name):
    f = calls()[name]
    with torch.no_grad():
        traced = torch.jit.trace(f, tensors(), check_trace=False)
        assert "b200scan::" in str(traced.graph)
        for seed in (0, 5):
            args = tensors(seed=seed)
            junk = [torch.full((2, 37, 24), 7.0, device="cuda") for _ in range(8)]  # what an uninitialised result would show
            del junk
            for a, w in zip(flat(traced(*args)), flat(f(*args)), strict=True):
                assert torch.equal(a, w)


@pytest.mark.parametrize("name", NAMES)
def test_a_dispatch_mode_sees_the_call(name):
    from torch.utils._python_dispatch import TorchDispatchMode

    class Log(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    seen, f, args = [], calls()[name], tensors()
    with torch.no_grad():
        want = f(*args)
        with Log():
            got = f(*args)
    assert any(s.startswith("b200scan") for s in seen), seen
    assert all(torch.equal(a, w) for a, w in zip(flat(got), flat(want), strict=True))


def test_gradients_under_a_dispatch_mode():
    from torch.utils._python_dispatch import TorchDispatchMode

    class Pass(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    for name in ("recurrence", "gated_norm", "residual_norm"):
        f = calls()[name]

        def grads():
            leaves = [t.requires_grad_() for t in tensors()]
            return torch.autograd.grad(sum(o.square().sum() for o in flat(f(*leaves))), leaves, allow_unused=True, materialize_grads=True)

        want = grads()
        with Pass():
            got = grads()
        assert all(torch.equal(a, w) for a, w in zip(got, want, strict=True))


@pytest.mark.parametrize("name", NAMES)
def test_make_fx_records_the_operator(name):
    from torch.fx.experimental.proxy_tensor import make_fx

    f, args = calls()[name], tensors()
    with torch.no_grad():
        module = make_fx(f)(*args)
        assert "b200scan" in module.code
        for a, w in zip(flat(module(*args)), flat(f(*args)), strict=True):
            assert torch.equal(a, w)


def test_fake_tensors_give_fake_results():
    import tsfast_b200 as b
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode(), torch.no_grad():
        x, lam, w = torch.empty(2, 37, 24, device="cuda"), torch.empty(24, device="cuda"), torch.empty(24, device="cuda")
        h, last = b.gated_recurrence(x, x, x, lam)
        assert h.shape == x.shape and last.shape == (2, 24) and last.dtype == torch.float32
        h, last = b.gated_recurrence(x[:, :0], x[:, :0], x[:, :0], lam)
        assert h.shape == (2, 0, 24)
        h, last = b.gated_recurrence(x[None, :, :0], x[None, :, :0], x[None, :, :0], lam)
        assert h.shape == (1, 2, 0, 24) and last.shape == (1, 2, 24)
        assert b.gated_recurrence_step(x[0], x[0], x[0], lam, torch.empty(50, 24, device="cuda")).shape == (37, 24)
        assert b.gated_norm(x, x, w).shape == x.shape
        y, r = b.residual_norm(x, x, w)
        assert y.shape == r.shape == x.shape
        q, scale = b.quantize_weight(torch.empty(300, 200, device="cuda"))
        assert q.shape == (300, 200) and q.stride(0) == 256 and scale.shape == (3, 2) and q.dtype == torch.float8_e4m3fn
        assert b.quant_linear(torch.empty(2, 3, 200, device="cuda").half(), q, scale).shape == (2, 3, 300)


def test_opcheck_of_the_weight():
    from tsfast_b200 import quant_b200

    for shape in ((300, 200), (1, 128)):
        torch.library.opcheck(quant_b200._weight_op, (torch.randn(*shape, device="cuda"),), test_utils=("test_faketensor",))


def test_second_derivatives_by_every_operand_are_refused():
    """Gradients depend on the upstream gradients and on h0 too: asking for those derivatives raises as for the others, with
    allow_unused as well, and so does the forward derivative that is made of two backward passes."""
    import tsfast_b200 as b

    x, r, i, lam, w = (t.requires_grad_() for t in tensors())
    h0 = torch.randn(2, 24, device="cuda", requires_grad=True)
    up, up_last = torch.randn(2, 37, 24, device="cuda", requires_grad=True), torch.randn(2, 24, device="cuda", requires_grad=True)
    outs = b.gated_recurrence(x, r, i, lam, h0)
    grads = torch.autograd.grad(outs, (x, r, i, lam, h0), (up, up_last), create_graph=True)
    for g in grads:
        for by in (up, up_last, h0, x, r, i, lam):
            with pytest.raises(RuntimeError, match="no second derivative"):
                torch.autograd.grad(g.sum(), by, retain_graph=True, allow_unused=True)
    seam = b.residual_norm(x, i, w, gate=r)
    for g in torch.autograd.grad(seam, (x, i, r, w), (up, up), create_graph=True):
        for by in (up, x, i, r, w):
            with pytest.raises(RuntimeError, match="no second derivative"):
                torch.autograd.grad(g.sum(), by, retain_graph=True, allow_unused=True)
    for f in (lambda t: b.gated_recurrence(t, r.detach(), i.detach(), lam.detach())[0], lambda t: b.gated_norm(t, r.detach(), w.detach())):
        with pytest.raises(RuntimeError, match="no second derivative"):
            torch.autograd.functional.jvp(f, x.detach(), torch.ones_like(x))


def test_the_start_may_be_overwritten_before_the_backward_pass():
    """h0 is not kept for it: a cache may be used as h0 and go on."""
    import tsfast_b200 as b

    x, r, i, lam, _ = (t.requires_grad_() for t in tensors())
    h0 = torch.randn(2, 24, device="cuda")
    want = torch.autograd.grad(b.gated_recurrence(x, r, i, lam, h0)[0].sum(), (x, lam))
    cache = h0.clone()
    h, last = b.gated_recurrence(x, r, i, lam, cache)
    cache.copy_(last.detach())
    assert all(torch.equal(a, b_) for a, b_ in zip(torch.autograd.grad(h.sum(), (x, lam)), want))


@pytest.mark.parametrize("name", [n for n in NAMES if n != "quantize_weight"])
def test_forward_derivatives_are_refused(name):
    """Not dropped: a dual tensor raises, and so does a tensor inside a transform of torch.func."""
    import torch.autograd.forward_ad as fw

    f, args = calls()[name], tensors()
    with torch.no_grad():
        with fw.dual_level():
            for k in range(5):
                dual = [fw.make_dual(t, torch.ones_like(t)) if j == k else t for j, t in enumerate(args)]
                if any(a is not b for a, b in zip(dual, args)) and uses(name, k):
                    with pytest.raises(RuntimeError, match="forward-mode"):
                        f(*dual)
        if uses(name, 0):
            with pytest.raises(RuntimeError, match="torch.func"):
                torch.func.jvp(lambda x: f(x, *args[1:]), (args[0],), (torch.ones_like(args[0]),))
            with pytest.raises(RuntimeError, match="torch.func"):
                torch.vmap(lambda x: f(x, *args[1:]))(torch.stack([args[0], args[0]]))


def uses(name, k):
    return k in {"gated_norm": (0, 1, 4), "residual_norm": (0, 1, 2, 4), "quant_linear": (0,)}.get(name, (0, 1, 2, 3))


def test_constants_that_float32_does_not_hold_are_refused():
    import tsfast_b200 as b

    x, r, i, lam, w = tensors()
    for c in (1e-60, 1e39, float("inf"), float("nan"), -1.0):
        with pytest.raises(RuntimeError, match="c="):
            b.gated_recurrence(x, r, i, lam, c=c)
        with pytest.raises(RuntimeError, match="c="):
            b.gated_recurrence_step(x[0], r[0], i[0], lam, torch.zeros(37, 24, device="cuda"), c=c)
    for eps in (1e39, float("inf"), float("nan")):
        with pytest.raises(RuntimeError, match="eps="):
            b.gated_norm(x, r, w, eps=eps)
        with pytest.raises(RuntimeError, match="eps="):
            b.residual_norm(x, r, w, eps=eps)


def test_a_cache_of_inference_mode():
    """It may be updated inside that mode only, as for every operator that updates a tensor; a refused call leaves it as it was."""
    import tsfast_b200 as b

    x, r, i, lam, _ = tensors()
    with torch.inference_mode():
        state = torch.zeros(37, 24, device="cuda")
        b.gated_recurrence_step(x[0], r[0], i[0], lam, state)
        kept = state.clone()
    with torch.no_grad(), pytest.raises(RuntimeError, match="nference"):
        b.gated_recurrence_step(x[0], r[0], i[0], lam, state)
    with torch.inference_mode():
        assert torch.equal(state, kept) and state.abs().sum() > 0


def test_compiled_calls_refuse_what_eager_ones_refuse():
    """A norm without its weight would return memory that nothing wrote."""
    import tsfast_b200 as b

    x, r, i, lam, w = tensors()
    compiled = lambda f: torch.compile(f, backend="aot_eager")  # noqa: E731
    with torch.no_grad():
        with pytest.raises(Exception, match="weight is required"):
            compiled(lambda x, r, w: b.residual_norm(x, r, None, post_weight=w))(x, r, w)
        with pytest.raises(Exception, match="weight is required"):
            compiled(lambda x, r: b.gated_norm(x, r, None))(x, r)
        with pytest.raises(Exception, match="post_bias without post_weight"):
            compiled(lambda x, r, w: b.residual_norm(x, r, w, post_bias=w, kind="layer"))(x, r, w)
        with pytest.raises(Exception, match="residual is required"):
            compiled(lambda x, w: b.residual_norm(x, None, w))(x, w)
        wide = x.reshape(2, 1, 37, 24)
        with pytest.raises(Exception, match="r is"):
            compiled(lambda x, r, lam: b.gated_recurrence(x, r, x, lam))(wide, wide.transpose(0, 1).contiguous(), lam)
        with pytest.raises(Exception, match="h0 is"):
            compiled(lambda x, lam, h: b.gated_recurrence(x, x, x, lam, h))(wide, lam, torch.zeros(1, 2, 24, device="cuda"))
        h, last = compiled(lambda x, lam: b.gated_recurrence(x, x, x, lam))(wide[:, :, :0], lam)
        assert h.shape == (2, 1, 0, 24) and (last == 0).all()


def checkpointed(f, *leaves):
    from torch.utils.checkpoint import checkpoint

    out = checkpoint(f, *leaves, use_reentrant=False)
    return torch.autograd.grad(sum(o.square().sum() for o in flat(out)), leaves, allow_unused=True, materialize_grads=True)


@pytest.mark.parametrize("name", ["recurrence", "recurrence 4-d", "recurrence packed", "gated_norm", "residual_norm"])
def test_checkpointed_calls(name):
    """Recomputation ends with an exception from inside the last operator that keeps a tensor: it has to come through as it is."""
    f = calls()[name]
    leaves = [t.requires_grad_() for t in tensors()]
    want = torch.autograd.grad(sum(o.square().sum() for o in flat(f(*leaves))), leaves, allow_unused=True, materialize_grads=True)
    assert all(torch.equal(a, w) for a, w in zip(checkpointed(f, *leaves), want, strict=True))


@pytest.mark.parametrize("name", ["recurrence", "gated_norm", "residual_norm"])
def test_an_exception_of_a_hook_keeps_its_type(name):
    class Mine(Exception):
        pass

    def pack(t):
        raise Mine("from the hook")

    f, leaves = calls()[name], [t.requires_grad_() for t in tensors()]
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t), pytest.raises(Mine, match="from the hook"):
        f(*leaves)


def test_a_compiled_program_quantises_its_weight():
    import tsfast_b200 as b

    def f(w, x):
        q, scale = b.quantize_weight(w)
        return b.quant_linear(x, q, scale), q.float(), scale

    w, x = torch.randn(150, 200, device="cuda"), torch.randn(9, 200, device="cuda").bfloat16()
    with torch.no_grad():
        for a, want in zip(torch.compile(f, fullgraph=True, backend="aot_eager")(w, x), f(w, x), strict=True):
            assert torch.equal(a, want)
