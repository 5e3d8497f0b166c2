"""The sequence and 8-bit operators under whatever watches or replaces torch's operators: fake tensors, make_fx, torch.jit.trace,
torch.func, forward-mode derivatives, checkpointing. A traced function holds the operators themselves and gives an eager
call's results, bit for bit."""
import pytest
import torch
import torch.autograd.forward_ad as fw
from torch._subclasses.fake_tensor import FakeTensor, FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

import metal_linalg_torch as mlt

OPS = torch.ops.metal_linalg


def rule_inputs(device="cuda", b=1, t=70, h=1, hv=2, dk=32, dv=48, seed=0):
    if device == "fake":
        r = lambda *s, dtype=torch.float32: torch.empty(s, dtype=dtype, device="cuda")  # noqa: E731
    else:
        gen = torch.Generator().manual_seed(seed)
        r = lambda *s, dtype=torch.float32: (0.2 * torch.randn(*s, generator=gen)).to(device, dtype)  # noqa: E731
    bf16 = torch.bfloat16
    return [r(b, t, h, dk, dtype=bf16), r(b, t, h, dk, dtype=bf16), r(b, t, hv, dv, dtype=bf16), -r(b, t, hv).abs(), r(b, t, hv).abs(),
            r(b, hv, dk, dv)]


def maps(device="cuda"):
    if device == "fake":
        return torch.empty(40, 64, device="cuda"), torch.empty(24, 64, device="cuda")
    gen = torch.Generator().manual_seed(1)
    return torch.randn(40, 64, generator=gen).to(device), torch.randn(24, 64, generator=gen).to(device)


def rule(q, k, v, g, beta, s):
    return mlt.gated_delta_rule(q, k, v, g, beta, initial_state=s)


def step(q, k, v, g, beta, s):
    return mlt.gated_delta_step(q[:, :1], k[:, :1], v[:, :1], g[:, :1], beta[:, :1], s), s


def product(x, w):
    return mlt.matmul_fp8(*mlt.quantize_fp8(x), *mlt.quantize_fp8(w, block=(128, 128)))


# function, inputs, the operators that a trace of it has to hold
CASES = {
    "rule": (rule, rule_inputs, {OPS.gated_delta_rule}),
    "step": (step, rule_inputs, {OPS.gated_delta_step}),
    "product": (product, maps, {OPS.quantize_fp8, OPS.matmul_fp8}),
    "linear": (mlt.linear_fp8, maps, {OPS.linear_fp8}),
}
case = pytest.mark.parametrize("case", CASES)


def held(graph):
    return {n.target.overloadpacket for n in graph.graph.nodes if n.op == "call_function" and hasattr(n.target, "overloadpacket")}


# ---------------------------------------------------------------------------
# Without a GPU
# ---------------------------------------------------------------------------

@case
def test_fake_tensors_give_shapes(case):
    f, make, _ = CASES[case]
    with FakeTensorMode():
        outs = f(*make("fake"))
    outs = outs if isinstance(outs, tuple) else (outs,)
    assert all(isinstance(x, FakeTensor) and x.device.type == "cuda" for x in outs)
    want = {"rule": [(1, 70, 2, 48), (1, 2, 32, 48)], "step": [(1, 1, 2, 48), (1, 2, 32, 48)], "product": [(40, 24)], "linear": [(40, 24)]}
    assert [tuple(x.shape) for x in outs] == want[case]


@case
def test_fake_tensors_behind_their_mode(case):
    """A tensor subclass, no mode in effect."""
    f, make, _ = CASES[case]
    with FakeTensorMode():
        args = make("fake")
    outs = f(*args)
    assert isinstance(outs[0] if isinstance(outs, tuple) else outs, FakeTensor)


@pytest.mark.parametrize("pre_dispatch", [False, True])
@case
def test_make_fx_of_fake_tensors(case, pre_dispatch):
    f, make, ops = CASES[case]
    with FakeTensorMode():
        graph = make_fx(f, pre_dispatch=pre_dispatch)(*make("fake"))
    assert ops <= held(graph)


def test_forward_mode_is_refused():
    meta = lambda *s: torch.empty(*s, device="meta")  # noqa: E731
    args = [meta(1, 5, 1, 8), meta(1, 5, 1, 8), meta(1, 5, 2, 8), meta(1, 5, 2), meta(1, 5, 2), meta(1, 2, 8, 8)]
    for name, call, i in (("gated_delta_rule", rule, 0), ("gated_delta_rule", rule, 5), ("gated_delta_rule", rule, 3), ("gated_delta_step", step, 2),
                          ("gated_delta_step", step, 5)):
        with fw.dual_level():
            call(*args)
            with pytest.raises(RuntimeError, match=f"{name}: forward-mode"):
                call(*(fw.make_dual(x, torch.empty_like(x)) if j == i else x for j, x in enumerate(args)))
    x, w = meta(4, 16), meta(3, 16)
    for call, name in ((mlt.linear_fp8, "linear_fp8"), (product, "quantize_fp8")):
        with fw.dual_level(), pytest.raises(RuntimeError, match=f"{name}: forward-mode"):
            call(x, fw.make_dual(w, torch.empty_like(w)))
        with pytest.raises(RuntimeError, match=f"{name}: forward-mode"):
            torch.func.jvp(lambda y: call(y, w), (x,), (torch.empty_like(x),))


# ---------------------------------------------------------------------------
# On the GPU: what was traced computes what an eager call does
# ---------------------------------------------------------------------------

def fresh(args):
    return [x.clone() for x in args]


def same(got, want):
    got, want = (x if isinstance(x, (tuple, list)) else (x,) for x in (got, want))
    assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["real", "fake", "symbolic"])
@case
def test_make_fx(case, mode):
    f, make, ops = CASES[case]
    graph = make_fx(f, tracing_mode=mode)(*make())
    assert ops <= held(graph)
    other = [-x if x.dim() == 2 else x * 0.5 for x in make()]
    same(graph(*fresh(other)), f(*fresh(other)))


@pytest.mark.gpu
def test_make_fx_of_gradients():
    def rule_grads(*args):
        leaves = [x.detach().requires_grad_() for x in args]
        o, s = rule(*leaves)
        return torch.autograd.grad((o, s), leaves, (torch.ones_like(o), torch.ones_like(s)))

    def linear_grads(*args):
        leaves = [x.detach().requires_grad_() for x in args]
        y = mlt.linear_fp8(*leaves)
        return torch.autograd.grad(y, leaves, torch.ones_like(y))

    for mode in ("real", "fake"):
        assert {OPS.gated_delta_rule, OPS.gated_delta_rule_backward} <= held(make_fx(rule_grads, tracing_mode=mode)(*rule_inputs()))
        assert {OPS.linear_fp8, OPS.quantize_fp8, OPS.matmul_fp8} <= held(make_fx(linear_grads, tracing_mode=mode)(*maps()))


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["rule", "step", "product", "linear"])
def test_jit_trace(name):
    f, make, _ = CASES[name]
    traced = torch.jit.trace(f, tuple(make()), check_trace=False)
    other = [-x if x.dim() == 2 else x * 0.5 for x in make()]
    same(traced(*fresh(other)), f(*fresh(other)))


@pytest.mark.gpu
def test_checkpointed():
    """Activations computed again in the backward pass: what the forward saved is asked for once."""
    from torch.utils.checkpoint import checkpoint
    for f, args in ((rule, rule_inputs()), (mlt.linear_fp8, maps())):
        leaves = [x.requires_grad_() for x in args]
        total = lambda outs: sum(x.float().square().sum() for x in (outs if isinstance(outs, tuple) else (outs,)))  # noqa: E731
        want = torch.autograd.grad(total(f(*leaves)), leaves)
        same(torch.autograd.grad(total(checkpoint(f, *leaves, use_reentrant=False)), leaves), want)


@pytest.mark.gpu
def test_functionalized():
    """The step changes its pool, which torch.func.functionalize refuses of custom operators; the others pass through it."""
    for f, args in ((rule, rule_inputs()), (product, maps()), (mlt.linear_fp8, maps())):
        same(torch.func.functionalize(f)(*args), f(*args))
    with pytest.raises(RuntimeError, match="gated_delta_step"):
        torch.func.functionalize(step)(*rule_inputs())
