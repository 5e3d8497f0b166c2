"""The gated delta rule against its recurrence in 64 bits, token by token.

Tolerances. With keys of length at most 1, beta in (0, 1) and decays at most 1 every token's map is a contraction, so an
error made in a token is not amplified by those behind it, and a result's relative error (2-norm) is that of the few
products it passes through: parts dropped in a product of split operands are at most 2^-22 of it, float32 sums of up to
128 terms 128 * 2^-24 at worst and about sqrt(128) * 2^-24 = 2.9 * 2^-22 / 4 as a rule. Five products lie between an input and an output,
eleven between an output's gradient and an input's: 5 * (1 + 0.8) rounds to F32 = 16 * 2^-22 forward and 2.5 times that backward. A result
of a shorter type adds one rounding, half a step: finfo(t).eps / 2.
"""
import math

import pytest
import torch

import metal_linalg_torch as mlt
from metal_linalg_torch import _lib

F32 = 16 * 2.0 ** -22
GRAD = 2.5 * F32


def tolerance(dtype, grad=False):
    short = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    return short + (GRAD if grad else F32)


def inputs(b, t, h, hv, dk, dv, dtype, seed=0, device="cuda", n=None, gate=0.5):
    gen = torch.Generator().manual_seed(seed)
    unit = lambda x: x / x.norm(dim=-1, keepdim=True).clamp_min(1e-6)  # noqa: E731
    q = unit(torch.randn(b, t, h, dk, generator=gen)).to(dtype)
    k = unit(torch.randn(b, t, h, dk, generator=gen) + 0.3).to(dtype)
    v = torch.randn(b, t, hv, dv, generator=gen).to(dtype)
    g = -gate * torch.rand(b, t, hv, generator=gen) ** 3
    beta = torch.rand(b, t, hv, generator=gen)
    s0 = 0.3 * torch.randn(b if n is None else n, hv, dk, dv, generator=gen)
    return [x.to(device) for x in (q, k, v, g, beta, s0)]


def recurrence(q, k, v, g, beta, s, scale=None):
    """In float64 on the CPU, one sequence a batch row."""
    q, k, v, g, beta, s = (x.to("cpu", torch.float64) for x in (q, k, v, g, beta, s))
    up = v.shape[2] // q.shape[2]
    q, k = q.repeat_interleave(up, 2), k.repeat_interleave(up, 2)
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    out = []
    for t in range(q.shape[1]):
        s = s * g[:, t].exp()[..., None, None]
        d = beta[:, t, :, None] * (v[:, t] - (k[:, t, :, :, None] * s).sum(-2))
        s = s + k[:, t, :, :, None] * d[..., None, :]
        out.append(scale * (q[:, t, :, :, None] * s).sum(-2))
    return torch.stack(out, 1) if out else v, s


def near(got, want, tol, what=""):
    want = want.to("cpu", torch.float64)
    got = got.detach().to("cpu", torch.float64)
    assert got.shape == want.shape, what
    off = (got - want).norm().item()
    assert off <= tol * want.norm().item() + 1e-30, f"{what}: off by {off / max(want.norm().item(), 1e-300):.3g}, allowed {tol:.3g}"


SHAPES = [
    # B, T, H, HV, Dk, Dv
    (1, 1, 1, 1, 1, 1), (2, 1, 1, 2, 16, 16), (1, 63, 2, 2, 64, 64), (1, 64, 1, 1, 128, 128), (2, 65, 2, 4, 128, 128),
    (1, 130, 1, 3, 17, 24), (1, 200, 2, 2, 71, 200), (3, 129, 1, 2, 128, 256), (1, 257, 3, 3, 96, 40), (1, 150, 1, 1, 65, 1),
]
TYPES = [torch.bfloat16, torch.float16, torch.float32]


# ---------------------------------------------------------------------------
# Refusals (no GPU needed: shapes, types and places are checked before any pointer is used)
# ---------------------------------------------------------------------------

def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="meta")


def fine():
    return dict(q=meta(1, 5, 2, 16), k=meta(1, 5, 2, 16), v=meta(1, 5, 4, 8), g=meta(1, 5, 4, dtype=torch.float32),
                beta=meta(1, 5, 4, dtype=torch.float32))


def test_meta_gives_shapes():
    o, s = mlt.gated_delta_rule(**fine())
    assert o.shape == (1, 5, 4, 8) and o.dtype == torch.bfloat16
    assert s.shape == (1, 4, 16, 8) and s.dtype == torch.float32
    cu = torch.zeros(4, dtype=torch.int32, device="meta")
    assert mlt.gated_delta_rule(**fine(), cu_seqlens=cu)[1].shape == (3, 4, 16, 8)
    assert mlt.gated_delta_step(**fine(), state=meta(3, 4, 16, 8, dtype=torch.float32)).shape == (1, 5, 4, 8)


@pytest.mark.parametrize("change, error", [
    (dict(q=meta(1, 5, 2, 16, dtype=torch.float64), k=meta(1, 5, 2, 16, dtype=torch.float64)), TypeError),
    (dict(k=meta(1, 5, 2, 16, dtype=torch.float16)), TypeError),
    (dict(g=meta(1, 5, 4, dtype=torch.int32)), TypeError),
    (dict(k=meta(1, 4, 2, 16)), ValueError),
    (dict(v=meta(1, 5, 3, 8), g=meta(1, 5, 3), beta=meta(1, 5, 3)), ValueError),
    (dict(v=meta(1, 5, 8)), ValueError),
    (dict(g=meta(1, 5, 2)), ValueError),
    (dict(q=meta(1, 5, 2, 129), k=meta(1, 5, 2, 129)), ValueError),
    (dict(v=meta(1, 5, 4, 257)), ValueError),
    (dict(initial_state=meta(1, 4, 16, 8)), TypeError),
    (dict(initial_state=meta(2, 4, 16, 8, dtype=torch.float32)), ValueError),
    (dict(cu_seqlens=meta(3, dtype=torch.float32)), TypeError),
    (dict(cu_seqlens=meta(1, dtype=torch.int32)), ValueError),
    (dict(cu_seqlens=torch.zeros(3, dtype=torch.int32)), ValueError),
    (dict(g=None), TypeError),
])
def test_rule_refuses(change, error):
    with pytest.raises(error, match="gated_delta_rule"):
        mlt.gated_delta_rule(**{**fine(), **change})


def test_rule_refuses_a_batch_of_ragged_rows_and_the_cpu():
    two = {n: x.expand(2, *x.shape[1:]) for n, x in fine().items()}
    with pytest.raises(ValueError, match="B must be 1"):
        mlt.gated_delta_rule(**two, cu_seqlens=meta(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="no CPU path"):
        mlt.gated_delta_rule(*(torch.zeros(x.shape, dtype=x.dtype) for x in fine().values()))


@pytest.mark.parametrize("change, error", [
    (dict(state=meta(1, 4, 16, 8)), TypeError),
    (dict(state=meta(1, 4, 8, 16, dtype=torch.float32)), ValueError),
    (dict(state=meta(1, 4, 8, 16, dtype=torch.float32).mT), ValueError),
    (dict(state=meta(0, 4, 16, 8, dtype=torch.float32)), ValueError),
    (dict(slots=meta(2, dtype=torch.int32)), ValueError),
    (dict(slots=meta(1, dtype=torch.float32)), TypeError),
    (dict(state=meta(1, 4, 16, 8, dtype=torch.float32).requires_grad_()), RuntimeError),
])
def test_step_refuses(change, error):
    with pytest.raises(error, match="gated_delta_step"):
        mlt.gated_delta_step(**{**fine(), "state": meta(1, 4, 16, 8, dtype=torch.float32), **change})


def test_c_entries_refuse_without_a_gpu():
    """Sizes are refused before any pointer is looked at, host pointers before any launch."""
    from metal_linalg_torch._delta import _PROBLEM
    lib = _lib.lib

    def problem(b=1, t=4, h=1, hv=1, dk=8, dv=8, seqs=0, dtype=0, index=4, ptr=0, device=-1):
        return _PROBLEM.pack(b, t, h, hv, dk, dv, seqs, dtype, index, 1.0, device, 0, *[ptr] * 7, *[0] * 15)

    size = lib.metal_linalg_gated_delta_rule_workspace_bytes
    assert size(problem(), 0) > 0 and size(problem(), 1) > size(problem(), 0)
    for bad in (problem(dk=129), problem(dv=257), problem(dk=0), problem(h=0), problem(h=2, hv=3), problem(dtype=3), problem(b=2, seqs=2),
                problem(b=70000), problem(t=1 << 30)):
        assert size(bad, 0) == 0 and _lib.last_error()
        assert lib.metal_linalg_gated_delta_rule(bad, None, None, None, 0) == _lib.INVALID_ARGUMENT
    assert size(None, 0) == 0
    assert lib.metal_linalg_gated_delta_rule(None, None, None, None, 0) == _lib.INVALID_ARGUMENT
    assert lib.metal_linalg_gated_delta_rule(problem(), None, None, None, 0) == _lib.INVALID_ARGUMENT and "q is NULL" in _lib.last_error()
    import numpy as np
    host = np.zeros(64, np.float32)
    assert lib.metal_linalg_gated_delta_rule(problem(ptr=host.ctypes.data), None, None, None, 0) == _lib.INVALID_ARGUMENT
    assert "device pointer" in _lib.last_error()
    assert lib.metal_linalg_gated_delta_step(problem(ptr=host.ctypes.data), host.ctypes.data, host.ctypes.data, 64, 1, None) == _lib.INVALID_ARGUMENT
    assert lib.metal_linalg_gated_delta_rule(problem(device=-2), None, None, None, 0) == _lib.INVALID_ARGUMENT
    assert lib.metal_linalg_gated_delta_rule(problem(t=0), None, None, None, 0) == _lib.OK       # nothing to do, nowhere to put it
    with mlt.CpuOnly():
        assert lib.metal_linalg_gated_delta_rule(problem(), None, None, None, 0) == _lib.RUNTIME_ERROR


def test_workspaces_of_more_than_64_bits_are_refused():
    """A size that ran over would be one that a caller's workspace seems to have."""
    from metal_linalg_torch._delta import _PROBLEM
    size = lambda b, t, hv, seqs=0: _lib.lib.metal_linalg_gated_delta_rule_workspace_bytes(  # noqa: E731
        _PROBLEM.pack(b, t, hv, hv, 128, 256, seqs, 0, 4, 1.0, -1, 0, *[0] * 7, *[0] * 15), 1)
    for bad in ((65535, 1 << 19, 65535), (1, (1 << 30) - 1, 65535), (1, (1 << 30) - 1, 65535, 65535), (65535, 1 << 12, 2048)):
        assert size(*bad) == 0 and "too many tokens" in _lib.last_error()
    chunk = size(1, 128, 1) - size(1, 64, 1)
    assert size(1, 1 << 24, 64) == chunk * (1 << 18) * 64 and size(65535, 64, 1) == chunk * 65535


# ---------------------------------------------------------------------------
# Values
# ---------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_rule(shape, dtype):
    q, k, v, g, beta, s0 = inputs(*shape, dtype)
    o, s = mlt.gated_delta_rule(q, k, v, g, beta, initial_state=s0)
    want_o, want_s = recurrence(q, k, v, g, beta, s0)
    assert o.dtype == dtype and s.dtype == torch.float32
    near(o, want_o, tolerance(dtype), "o")
    near(s, want_s, F32, "state")
    o2, s2 = mlt.gated_delta_rule(q, k, v, g, beta)                        # from zero
    want_o, want_s = recurrence(q, k, v, g, beta, torch.zeros_like(s0))
    near(o2, want_o, tolerance(dtype), "o from zero")
    near(s2, want_s, F32, "state from zero")


@pytest.mark.gpu
@pytest.mark.parametrize("heads, batch", [(1, 1), (10, 1), (20, 2), (40, 2)])
def test_rule_whatever_shares_a_chain(heads, batch):
    """Few chains (four warps to one), more (two), many (one) give the same result, and the same bits twice."""
    args = inputs(batch, 140, heads, heads, 128, 128, torch.bfloat16, seed=heads)
    o, s = mlt.gated_delta_rule(*args[:5], initial_state=args[5])
    want_o, want_s = recurrence(*args)
    near(o, want_o, tolerance(torch.bfloat16))
    near(s, want_s, F32)
    again = mlt.gated_delta_rule(*args[:5], initial_state=args[5])
    assert torch.equal(o, again[0]) and torch.equal(s, again[1])


def ragged(lens, h, hv, dk, dv, dtype, seed=0, tail=0):
    total = sum(lens) + tail
    q, k, v, g, beta, s0 = inputs(1, total, h, hv, dk, dv, dtype, seed=seed, n=len(lens))
    cu = torch.tensor([0] + lens).cumsum(0)
    return (q, k, v, g, beta, s0), cu


LENS = [[5], [64, 64], [0, 1, 63, 0, 65, 130, 0], [200, 3], [1] * 40, [0], [0, 0, 7]]


@pytest.mark.gpu
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("lens", LENS, ids=str)
def test_ragged(lens, index):
    (q, k, v, g, beta, s0), cu = ragged(lens, 2, 4, 64, 48, torch.bfloat16, seed=len(lens), tail=70)
    o, s = mlt.gated_delta_rule(q, k, v, g, beta, initial_state=s0, cu_seqlens=cu.to("cuda", index))
    for i, (a, b) in enumerate(zip(cu.tolist(), cu.tolist()[1:])):
        part = [x[:, a:b] for x in (q, k, v, g, beta)]
        want_o, want_s = recurrence(*part, s0[i:i + 1])
        near(o[:, a:b], want_o, tolerance(torch.bfloat16), f"sequence {i}")
        near(s[i:i + 1], want_s, F32, f"state {i}")
        if a == b:
            assert torch.equal(s[i], s0[i])
    assert not o[:, int(cu[-1]):].any()


@pytest.mark.gpu
def test_ragged_more_sequences_than_a_block_counts():
    lens = [(7 * i) % 5 for i in range(600)]
    (q, k, v, g, beta, s0), cu = ragged(lens, 1, 1, 16, 16, torch.float32)
    o, s = mlt.gated_delta_rule(q, k, v, g, beta, initial_state=s0, cu_seqlens=cu.cuda())
    longest = max(lens)
    at = (cu[:-1, None] + torch.arange(longest)).clamp(max=q.shape[1] - 1)
    there = torch.arange(longest) < torch.tensor(lens)[:, None]
    spread = [x[0].cpu()[at] for x in (q, k, v, g, beta)]
    for i in (1, 3, 4):                                     # k, g, beta: zero behind a sequence's end
        spread[i] = spread[i] * there.reshape(*there.shape, *[1] * (spread[i].dim() - 2))
    want_o, want_s = recurrence(*spread, s0)
    near(s, want_s, F32)
    near(o[0].cpu(), want_o[there], F32)


@pytest.mark.gpu
def test_bad_bounds_stay_inside():
    """cu_seqlens that fall, overlap or leave the tokens are the caller's mistake; the kernels stay inside their buffers
    (checked by what lies around them: every output is the call's own, and finite)."""
    (q, k, v, g, beta, s0), _ = ragged([100, 100, 100], 1, 1, 32, 32, torch.float32)
    for bounds in ([0, 300, 0, 300], [50, 40, 30, 20], [-7, 100, 5000, 300], [0, 2 ** 31 - 1, 0, 2 ** 31 - 1]):
        o, s = mlt.gated_delta_rule(q, k, v, g, beta, initial_state=s0, cu_seqlens=torch.tensor(bounds, dtype=torch.int32).cuda())
        assert o.shape == v.shape and s.isfinite().all()


@pytest.mark.gpu
def test_no_tokens():
    q, k, v, g, beta, s0 = inputs(2, 0, 1, 2, 16, 24, torch.bfloat16)
    o, s = mlt.gated_delta_rule(q, k, v, g, beta, initial_state=s0)
    assert o.shape == (2, 0, 2, 24) and torch.equal(s, s0)
    o, s = mlt.gated_delta_rule(q, k, v, g, beta)
    assert not s.any()


@pytest.mark.gpu
def test_gates_that_close_and_rows_that_add_nothing():
    """-inf and very negative gates clear the state and keep the decays behind them exact; beta 0 leaves it as it is."""
    q, k, v, g, beta, s0 = inputs(1, 200, 1, 2, 64, 32, torch.float32, seed=3)
    g[0, 70, 0] = -math.inf
    g[0, 10, 1] = -3e4
    g[0, 90:95, 1] = -500.0
    beta[0, 100:130] = 0.0
    o, s = mlt.gated_delta_rule(q, k, v, g, beta, initial_state=s0)
    want_o, want_s = recurrence(q, k, v, g, beta, s0)
    near(o, want_o, F32)
    near(s, want_s, F32)
    # a gate of -inf in the last token leaves that token alone in the state
    g[0, -1] = -math.inf
    _, s = mlt.gated_delta_rule(q, k, v, g, beta, initial_state=s0)
    want = k[0, -1].double().cpu()[..., None] * (beta[0, -1].double().cpu()[:, None] * v[0, -1].double().cpu())[:, None]
    near(s[0], want, F32)


@pytest.mark.gpu
def test_what_is_not_finite_stays_in_its_sequence_and_head():
    q, k, v, g, beta, s0 = inputs(2, 100, 2, 2, 32, 32, torch.float32)
    clean = mlt.gated_delta_rule(q, k, v, g, beta, initial_state=s0)
    v[0, 50, 1, 3] = math.nan
    k[1, 20, 0, 0] = math.inf
    o, s = mlt.gated_delta_rule(q, k, v, g, beta, initial_state=s0)
    for b, h in ((0, 0), (1, 1)):
        assert torch.equal(o[b, :, h], clean[0][b, :, h]) and torch.equal(s[b, h], clean[1][b, h])
    assert o[0, 50, 1, 3].isnan() and not s[1, 0].isfinite().any()
    assert torch.equal(o[0, :, 1, 16:], clean[0][0, :, 1, 16:])            # columns are independent


@pytest.mark.gpu
def test_strides_and_alignment():
    b, t, h, d = 2, 100, 2, 64
    base = torch.randn(b, t, 3, h, d, device="cuda", dtype=torch.bfloat16) * 0.2      # one projection's output, cut up
    q, k, v = base.unbind(2)
    g = -torch.rand(b, h, t, device="cuda").transpose(1, 2)
    beta = torch.rand(b, t, 2 * h, device="cuda")[..., ::2]
    s0 = torch.randn(b, h, d, d, device="cuda").mT
    want = mlt.gated_delta_rule(*(x.contiguous() for x in (q, k, v, g, beta)), initial_state=s0.contiguous())
    got = mlt.gated_delta_rule(q, k, v, g, beta, initial_state=s0)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # rows that start off 16 bytes, and a last dimension that is not contiguous
    wide = torch.zeros(b, t, h, d + 3, device="cuda", dtype=torch.bfloat16)
    wide[..., 1:d + 1] = q
    turned = k.transpose(-1, -2).contiguous().transpose(-1, -2)
    got = mlt.gated_delta_rule(wide[..., 1:d + 1], turned, v, g, beta, initial_state=s0)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # a head's keys broadcast over the batch
    shared = k[:1].expand(b, -1, -1, -1)
    got = mlt.gated_delta_rule(q, shared, v, g, beta)
    want = mlt.gated_delta_rule(q, shared.contiguous(), v, g, beta)
    assert torch.equal(got[0], want[0])


@pytest.mark.gpu
def test_gates_in_short_types_and_a_scale():
    q, k, v, g, beta, s0 = inputs(1, 70, 1, 1, 32, 32, torch.bfloat16)
    o, s = mlt.gated_delta_rule(q, k, v, g.bfloat16(), beta.half(), scale=0.7, initial_state=s0)
    want_o, want_s = recurrence(q, k, v, g.bfloat16(), beta.half(), s0, scale=0.7)
    near(o, want_o, tolerance(torch.bfloat16))
    near(s, want_s, F32)


# ---------------------------------------------------------------------------
# Gradients
# ---------------------------------------------------------------------------

NAMES = ("q", "k", "v", "g", "beta", "initial_state")


def wanted_grads(args, d_o, d_s):
    leaves = [x.detach().to("cpu", torch.float64).requires_grad_() for x in args]
    o, s = recurrence(*leaves)
    return torch.autograd.grad((o, s), leaves, (d_o.to("cpu", torch.float64), d_s.to("cpu", torch.float64)), allow_unused=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_gradients(shape, dtype):
    args = inputs(*shape, dtype, seed=11)
    leaves = [x.detach().requires_grad_() for x in args]
    o, s = mlt.gated_delta_rule(*leaves[:5], initial_state=leaves[5])
    gen = torch.Generator(device="cuda").manual_seed(5)
    d_o = torch.randn(o.shape, device="cuda", generator=gen).to(dtype)
    d_s = 0.3 * torch.randn(s.shape, device="cuda", generator=gen)
    got = torch.autograd.grad((o, s), leaves, (d_o, d_s))
    want = wanted_grads(args, d_o, d_s)
    for name, x, y in zip(NAMES, got, want):
        assert x.dtype == (dtype if name in "qkv" else torch.float32)
        near(x, y, tolerance(x.dtype, grad=True), name)


@pytest.mark.gpu
@pytest.mark.parametrize("heads, batch", [(10, 1), (20, 2), (40, 2)])
def test_gradients_whatever_shares_a_chain(heads, batch):
    args = inputs(batch, 130, heads, heads, 128, 128, torch.bfloat16, seed=heads)
    leaves = [x.detach().requires_grad_() for x in args]
    o, s = mlt.gated_delta_rule(*leaves[:5], initial_state=leaves[5])
    d_o, d_s = torch.randn_like(o), torch.randn_like(s)
    got = torch.autograd.grad((o, s), leaves, (d_o, d_s), retain_graph=True)
    for name, x, y in zip(NAMES, got, wanted_grads(args, d_o, d_s)):
        near(x, y, tolerance(x.dtype, grad=True), name)
    again = torch.autograd.grad((o, s), leaves, (d_o, d_s))
    assert all(torch.equal(x, y) for x, y in zip(got, again))


@pytest.mark.gpu
@pytest.mark.parametrize("lens", LENS, ids=str)
def test_gradients_ragged(lens):
    args, cu = ragged(lens, 1, 2, 64, 48, torch.float32, seed=len(lens), tail=66)
    leaves = [x.detach().requires_grad_() for x in args]
    o, s = mlt.gated_delta_rule(*leaves[:5], initial_state=leaves[5], cu_seqlens=cu.cuda())
    d_o, d_s = torch.randn_like(o), torch.randn_like(s)
    got = torch.autograd.grad((o, s), leaves, (d_o, d_s))
    for i, (a, b) in enumerate(zip(cu.tolist(), cu.tolist()[1:])):
        part = [x[:, a:b] for x in args[:5]] + [args[5][i:i + 1]]
        want = wanted_grads(part, d_o[:, a:b], d_s[i:i + 1])
        for name, x, y in zip(NAMES, got, want):
            if y is not None:
                near(x[i:i + 1] if name == "initial_state" else x[:, a:b], y, GRAD, f"{name} of sequence {i}")
    for x in got[:5]:
        assert not x[:, int(cu[-1]):].any()


@pytest.mark.gpu
def test_gradients_of_one_result_and_without_a_state():
    args = inputs(1, 90, 1, 1, 48, 32, torch.float32)
    zero = torch.zeros_like(args[5])
    for use_o, use_s in ((True, False), (False, True)):
        leaves = [x.detach().requires_grad_() for x in args[:5]]
        o, s = mlt.gated_delta_rule(*leaves)
        d_o, d_s = torch.randn_like(o), torch.randn_like(s)
        outs = [x for x, use in ((o, use_o), (s, use_s)) if use]
        got = torch.autograd.grad(outs, leaves, [x for x, use in ((d_o, use_o), (d_s, use_s)) if use])
        want = wanted_grads([*args[:5], zero], d_o * use_o, d_s * use_s)
        for name, x, y in zip(NAMES, got, want):
            near(x, y, GRAD, name)


@pytest.mark.gpu
def test_gradients_behind_closed_gates_and_beta_zero():
    args = inputs(1, 150, 1, 1, 32, 32, torch.float32, seed=4)
    args[3][0, 70] = -math.inf
    args[3][0, 20] = -400.0
    args[4][0, 30:40] = 0.0
    leaves = [x.detach().requires_grad_() for x in args]
    o, s = mlt.gated_delta_rule(*leaves[:5], initial_state=leaves[5])
    d_o, d_s = torch.randn_like(o), torch.randn_like(s)
    got = torch.autograd.grad((o, s), leaves, (d_o, d_s))
    finite = [x.clone() for x in args]
    finite[3][0, 70] = -1e4                       # the same decay, 0, without 0 * inf in the recurrence's own gradient
    want = wanted_grads(finite, d_o, d_s)
    for name, x, y in zip(NAMES, got, want):
        near(x, y, GRAD, name)


@pytest.mark.gpu
def test_gradients_by_differences():
    """Against central differences of the operator's own outputs along one direction for every input. Step h = 2^-6 on
    outputs of order 1: the differences' own error is h^2 of the third derivative (2^-12, relative) plus the outputs'
    error over h (16 * 2^-22 * 2^6 = 2^-12): 2^-9 covers their sum eight times over two."""
    args = inputs(1, 80, 1, 2, 32, 32, torch.float32, seed=8)
    leaves = [x.detach().requires_grad_() for x in args]
    o, s = mlt.gated_delta_rule(*leaves[:5], initial_state=leaves[5])
    d_o, d_s = torch.randn_like(o), torch.randn_like(s)
    got = torch.autograd.grad((o, s), leaves, (d_o, d_s))
    value = lambda x: sum((a.double() * b.double()).sum() for a, b in zip(mlt.gated_delta_rule(*x[:5], initial_state=x[5]), (d_o, d_s)))  # noqa: E731
    h = 2.0 ** -6
    for i, name in enumerate(NAMES):
        along = got[i] / got[i].norm()              # where the function changes most: the derivative is the gradient's length
        up, down = ([x + sign * h * along if j == i else x for j, x in enumerate(args)] for sign in (1, -1))
        want = (value(up) - value(down)).item() / (2 * h)
        assert abs(want - got[i].norm().item()) <= 2.0 ** -9 * got[i].norm().item(), name


@pytest.mark.gpu
def test_second_derivatives_are_refused():
    args = inputs(1, 10, 1, 1, 16, 16, torch.float32)
    q = args[0].requires_grad_()
    o, _ = mlt.gated_delta_rule(q, *args[1:5])
    (dq,) = torch.autograd.grad(o.square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        dq.sum().backward()


# ---------------------------------------------------------------------------
# Tokens one at a time
# ---------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1, 1), (3, 1, 2, 4, 128, 128), (2, 3, 1, 2, 17, 30), (5, 2, 1, 1, 96, 256), (2, 1, 3, 3, 64, 33)])
def test_step(shape, dtype):
    q, k, v, g, beta, s0 = inputs(*shape, dtype, seed=2)
    state = s0.clone()
    o = mlt.gated_delta_step(q, k, v, g, beta, state)
    want_o, want_s = recurrence(q, k, v, g, beta, s0)
    near(o, want_o, tolerance(dtype), "o")
    near(state, want_s, F32, "state")


@pytest.mark.gpu
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_step_slots(index):
    """Slots in any order, padding, slots past the pool, a slot named three times, a pool inside a larger cache."""
    b, t, h, hv, dk, dv = 7, 2, 1, 2, 48, 64
    q, k, v, g, beta, _ = inputs(b, t, h, hv, dk, dv, torch.bfloat16, seed=6)
    cache = torch.randn(9, 2, hv, dk, dv, device="cuda") * 0.3
    before = cache.clone()
    slots = [4, -1, 0, 4, 9, 8, 4]
    o = mlt.gated_delta_step(q, k, v, g, beta, cache[:, 1], slots=torch.tensor(slots, dtype=index).cuda())
    pool = before[:, 1].double().cpu()
    for r, slot in enumerate(slots):
        if not 0 <= slot < 9:
            assert not o[r].any()
            continue
        row = [x[r:r + 1] for x in (q, k, v, g, beta)]
        want_o, pool[slot:slot + 1] = recurrence(*row, pool[slot:slot + 1])
        near(o[r:r + 1], want_o, tolerance(torch.bfloat16), f"row {r}")
    near(cache[:, 1], pool, F32)
    assert torch.equal(cache[:, 0], before[:, 0])
    untouched = [i for i in range(9) if i not in slots]
    assert torch.equal(cache[untouched], before[untouched])


@pytest.mark.gpu
def test_step_large_pool_offsets():
    """A slot whose state lies behind 2^31 elements."""
    hv, dk, dv = 64, 128, 128
    slots = (1 << 31) // (hv * dk * dv) + 3
    pool = torch.zeros(slots, hv, dk, dv, device="cuda")
    q, k, v, g, beta, s0 = inputs(1, 1, 1, hv, dk, dv, torch.bfloat16)
    pool[-1] = s0[0]
    o = mlt.gated_delta_step(q, k, v, g, beta, pool, slots=torch.tensor([slots - 1]).cuda())
    want_o, want_s = recurrence(q, k, v, g, beta, s0)
    near(o, want_o, tolerance(torch.bfloat16))
    near(pool[-1:], want_s, F32)
    assert not pool[:-1].any()


# ---------------------------------------------------------------------------
# Streams, graphs, compilation
# ---------------------------------------------------------------------------

@pytest.mark.gpu
def test_streams_of_their_own():
    calls = [inputs(1, 300, 2, 4, 64, 64, torch.bfloat16, seed=i) for i in range(4)]
    want = [mlt.gated_delta_rule(*c[:5], initial_state=c[5]) for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = []
    for c, stream in zip(calls, streams):
        with torch.cuda.stream(stream):
            got.append(mlt.gated_delta_rule(*c[:5], initial_state=c[5]))
    torch.cuda.synchronize()
    for (a, b), (c, d) in zip(got, want):
        assert torch.equal(a, c) and torch.equal(b, d)


@pytest.mark.gpu
def test_captured_and_replayed():
    """Forward, backward and a decoding step in graphs; two graphs captured on one stream and replayed on two do not share
    a workspace."""
    a, b = (inputs(1, 200, 2, 2, 64, 64, torch.bfloat16, seed=i) for i in (1, 2))
    side = torch.cuda.Stream()

    def train(args):
        leaves = [x.detach().requires_grad_() for x in args]
        o, s = mlt.gated_delta_rule(*leaves[:5], initial_state=leaves[5])
        return (o, s, *torch.autograd.grad((o, s), leaves, (torch.ones_like(o), torch.ones_like(s))))

    want = [[x.detach().clone() for x in train(args)] for args in (a, b)]
    graphs, outs = [], []
    with torch.cuda.stream(side):
        for args in (a, b):
            train(args)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                outs.append(train(args))
            graphs.append(graph)
    torch.cuda.synchronize()
    others = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for graph, stream in zip(graphs, others):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for got, w in zip(outs, want):
            assert all(torch.equal(x, y) for x, y in zip(got, w))

    q, k, v, g, beta, s0 = inputs(3, 1, 2, 2, 64, 64, torch.bfloat16)
    state, slots = s0.clone(), torch.tensor([2, 0, 1]).cuda()
    with torch.cuda.stream(side):
        mlt.gated_delta_step(q, k, v, g, beta, state, slots=slots)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            o = mlt.gated_delta_step(q, k, v, g, beta, state, slots=slots)
    torch.cuda.synchronize()
    state.copy_(s0)
    other = s0.clone()
    for _ in range(3):
        graph.replay()
        want_o = mlt.gated_delta_step(q, k, v, g, beta, other, slots=slots)
        torch.cuda.synchronize()
        assert torch.equal(o, want_o) and torch.equal(state, other)


@pytest.mark.gpu
def test_compiled():
    """torch.compile sees the custom operators (backend "eager": the graph is traced, not rewritten)."""
    q, k, v, g, beta, s0 = inputs(1, 70, 1, 2, 32, 32, torch.float32)

    def f(q, k, v, g, beta, s0):
        o, s = mlt.gated_delta_rule(q, k, v, g, beta, initial_state=s0)
        return o * 2, s

    want = f(q, k, v, g, beta, s0)
    leaves = [x.detach().requires_grad_() for x in (q, k, v, g, beta, s0)]
    got = torch.compile(f, backend="aot_eager", fullgraph=True)(*leaves)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    grads = torch.autograd.grad(got, leaves, [torch.ones_like(x) for x in got])
    plain = torch.autograd.grad(f(*leaves), leaves, [torch.ones_like(x) for x in want])
    assert all(torch.equal(x, y) for x, y in zip(grads, plain))


@pytest.mark.gpu
def test_compiled_step():
    q, k, v, g, beta, s0 = inputs(3, 1, 1, 2, 32, 32, torch.bfloat16)
    slots = torch.tensor([2, -1, 0], device="cuda")

    def f(q, k, v, g, beta, state):
        return mlt.gated_delta_step(q, k, v, g, beta, state, slots=slots) * 2

    a, b = s0.clone(), s0.clone()
    want = f(q, k, v, g, beta, a)
    got = torch.compile(f, backend="aot_eager", fullgraph=True)(q, k, v, g, beta, b)
    assert torch.equal(got, want) and torch.equal(a, b)


@pytest.mark.gpu
def test_two_threads_at_once():
    """The library's stream is the calling thread's: calls of several threads, each on its own stream, do not meet."""
    import threading
    calls = [inputs(1, 200 + 64 * i, 2, 2, 64, 64, torch.bfloat16, seed=i) for i in range(4)]
    want = [mlt.gated_delta_rule(*c[:5], initial_state=c[5]) for c in calls]
    torch.cuda.synchronize()
    got = [None] * len(calls)

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i] = mlt.gated_delta_rule(*calls[i][:5], initial_state=calls[i][5])
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for (a, b), (c, d) in zip(got, want):
        assert torch.equal(a, c) and torch.equal(b, d)


@pytest.mark.gpu
def test_ragged_without_tokens():
    q, k, v, g, beta, s0 = inputs(1, 0, 1, 2, 16, 24, torch.bfloat16, n=3)
    cu = torch.zeros(4, dtype=torch.int32, device="cuda")
    leaves = [x.requires_grad_() for x in (q, k, v, g, beta, s0)]
    o, s = mlt.gated_delta_rule(*leaves[:5], initial_state=leaves[5], cu_seqlens=cu)
    assert o.shape == (1, 0, 2, 24) and torch.equal(s, s0)
    ds = torch.randn_like(s)
    grads = torch.autograd.grad((o, s), leaves, (torch.zeros_like(o), ds))
    assert torch.equal(grads[5], ds) and grads[0].shape == q.shape
    o = mlt.gated_delta_step(*(x.detach()[:, :0] for x in leaves[:5]), s0.detach())
    assert o.shape == (1, 0, 2, 24)


@pytest.mark.gpu
def test_expanded_gradients():
    """sum().backward() hands in a gradient of stride 0."""
    args = inputs(1, 70, 1, 1, 16, 16, torch.float32)
    leaves = [x.detach().requires_grad_() for x in args]
    o, s = mlt.gated_delta_rule(*leaves[:5], initial_state=leaves[5])
    (o.sum() + s.sum()).backward()
    for name, x, y in zip(NAMES, leaves, wanted_grads(args, torch.ones_like(o), torch.ones_like(s))):
        near(x.grad, y, GRAD, name)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Tokens 2^26 elements apart: the last ones lie behind 2^31."""
    q, k, v, g, beta, s0 = inputs(1, 40, 1, 1, 32, 32, torch.bfloat16)
    far = torch.empty_strided((1, 40, 1, 32), (0, 1 << 26, 32, 1), dtype=torch.bfloat16, device="cuda")
    want = mlt.gated_delta_rule(q, k, v, g, beta, initial_state=s0)
    far.copy_(k)
    got = mlt.gated_delta_rule(q, far, v, g, beta, initial_state=s0)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    far.copy_(v)
    got = mlt.gated_delta_rule(q, k, far, g, beta, initial_state=s0)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
def test_prompt_then_tokens():
    """A prompt in two pieces, then single tokens by the step, is the whole sequence at once."""
    q, k, v, g, beta, s0 = inputs(2, 140, 2, 4, 64, 64, torch.float32, seed=9)
    want_o, want_s = recurrence(q, k, v, g, beta, s0)
    cut = lambda a, b: [x[:, a:b] for x in (q, k, v, g, beta)]  # noqa: E731
    o1, s = mlt.gated_delta_rule(*cut(0, 70), initial_state=s0)
    o2, s = mlt.gated_delta_rule(*cut(70, 135), initial_state=s)
    pool = torch.zeros(5, *s.shape[1:], device="cuda")
    slots = torch.tensor([3, 1], device="cuda")
    pool[slots] = s
    rest = [mlt.gated_delta_step(*cut(t, t + 1), pool, slots=slots) for t in range(135, 140)]
    near(torch.cat([o1, o2, *rest], 1), want_o, F32)
    near(pool[slots], want_s, F32)


@pytest.mark.gpu
@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_tensors_of_another_gpu_than_the_current_one():
    args = [x.to("cuda:1") for x in inputs(1, 70, 1, 1, 32, 32, torch.bfloat16)]
    with torch.cuda.device(0):
        o, s = mlt.gated_delta_rule(*args[:5], initial_state=args[5])
    want_o, want_s = recurrence(*args)
    near(o, want_o, tolerance(torch.bfloat16))
    near(s, want_s, F32)


# ---------------------------------------------------------------------------
# Long sequences, eager and captured; tokens of no sequence; pools that graphs have saved
# ---------------------------------------------------------------------------

LONG = [
    # B, T, H, HV, Dk, Dv, bounds
    (1, 64 * 200 + 17, 1, 2, 64, 32, None), (2, 64 * 128, 1, 1, 128, 16, None), (1, 64 * 127 + 63, 2, 2, 16, 48, None),
    (1, 64 * 200, 1, 2, 64, 32, (0, 64 * 200)), (1, 64 * 200, 1, 1, 32, 24, (5, 64 * 130 + 5)), (1, 64 * 300, 1, 1, 32, 16, (0, 100)),
    (1, 64 * 192, 1, 1, 64, 64, (64, 64 * 129)),
]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", LONG, ids=str)
def test_long_sequences(shape):
    """Again and captured: the same products in the same order, bit for bit. And the float64 recurrence's, from a few tokens
    before the end on (a sequence in two calls)."""
    b, t, h, hv, dk, dv, bounds = shape
    q, k, v, g, beta, s0 = inputs(b, t, h, hv, dk, dv, torch.bfloat16, seed=t)
    cu = None if bounds is None else torch.tensor(bounds, dtype=torch.int32, device="cuda")
    call = lambda: mlt.gated_delta_rule(q, k, v, g, beta, initial_state=s0, cu_seqlens=cu)  # noqa: E731
    o, s = call()
    again = call()
    assert torch.equal(o, again[0]) and torch.equal(s, again[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        whole = call()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(o, whole[0]) and torch.equal(s, whole[1])
    first, last = (0, t) if bounds is None else bounds
    cut = max(first, last - 50)
    part = lambda a, z: [x[:, a:z] for x in (q, k, v, g, beta)]  # noqa: E731
    _, middle = mlt.gated_delta_rule(*part(first, cut), initial_state=s0)
    want_o, want_s = recurrence(*part(cut, last), middle)
    near(o[:, cut:last], want_o, tolerance(torch.bfloat16))
    near(s, want_s, F32)


@pytest.mark.gpu
def test_long_sequences_on_many_streams_and_threads():
    import threading
    args = inputs(1, 64 * 150, 1, 2, 64, 32, torch.bfloat16)
    want = mlt.gated_delta_rule(*args[:5], initial_state=args[5])
    torch.cuda.synchronize()
    got, failed = {}, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(4):
                    got[i] = mlt.gated_delta_rule(*args[:5], initial_state=args[5])
        except Exception as e:      # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [x.start() for x in threads]
    [x.join() for x in threads]
    torch.cuda.synchronize()
    assert not failed and all(torch.equal(a, b) for r in got.values() for a, b in zip(r, want))


@pytest.mark.gpu
def test_tokens_before_the_first_sequence():
    q, k, v, g, beta, s0 = inputs(1, 300, 1, 2, 32, 48, torch.float32, n=2)
    cu = torch.tensor([70, 130, 210], device="cuda")
    torch.full((1, 300, 2, 48), float("nan"), device="cuda")       # what the allocator hands out next
    leaves = [x.requires_grad_() for x in (q, k, v, g, beta)]
    o, s = mlt.gated_delta_rule(*leaves, initial_state=s0, cu_seqlens=cu)
    grads = torch.autograd.grad((o, s), leaves, (torch.ones_like(o), torch.ones_like(s)))
    inside = [x.detach()[:, 70:210] for x in leaves]
    other, _ = mlt.gated_delta_rule(*inside, initial_state=s0, cu_seqlens=cu - 70)
    assert torch.equal(o[:, 70:210], other)
    for x in (o, *grads):
        assert not x[:, :70].any() and not x[:, 210:].any() and x.isfinite().all()


@pytest.mark.gpu
def test_a_step_tells_the_graph_that_saved_its_pool():
    q, k, v, g, beta, pool = inputs(2, 1, 1, 1, 16, 16, torch.float32)
    o, _ = mlt.gated_delta_rule(q.requires_grad_(), k, v, g, beta, initial_state=pool)
    with torch.no_grad():
        mlt.gated_delta_step(q, k, v, g, beta, pool)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("n, length", [(300, 70), (7, 130), (1, 200)])
def test_ragged_rows_of_one_length_are_a_batch(n, length):
    """Whatever order the sequences start in: the batch's results, bit for bit, and its gradients (the backward pass may share
    its chains between other numbers of warps)."""
    q, k, v, g, beta, s0 = inputs(n, length, 1, 2, 32, 16, torch.bfloat16, seed=n)
    grads_of = lambda o, s, leaves: torch.autograd.grad((o, s), leaves, (torch.ones_like(o), torch.ones_like(s)))  # noqa: E731
    batch = [x.clone().requires_grad_() for x in (q, k, v, g, beta, s0)]
    rows = [x.reshape(1, n * length, *x.shape[2:]).clone().requires_grad_() for x in (q, k, v, g, beta)] + [s0.clone().requires_grad_()]
    cu = torch.arange(n + 1, device="cuda", dtype=torch.int32) * length
    o, s = mlt.gated_delta_rule(*batch[:5], initial_state=batch[5])
    ro, rs = mlt.gated_delta_rule(*rows[:5], initial_state=rows[5], cu_seqlens=cu)
    assert torch.equal(o.reshape(ro.shape), ro) and torch.equal(s, rs)
    for x, y in zip(grads_of(o, s, batch), grads_of(ro, rs, rows)):
        near(y.reshape(x.shape), x, tolerance(torch.bfloat16, grad=True))


# ---------------------------------------------------------------------------
# Bounds that are the caller's mistake: everything that is written lies inside the call's own buffers
# ---------------------------------------------------------------------------

GUARD, MARK = 8192, 0xA5


class Guarded:
    """Buffers of one allocation, each between two stretches that hold a pattern."""

    def __init__(self, **sizes):
        self.at, end = {}, GUARD
        for name, size in sizes.items():
            self.at[name] = (end, size)
            end += -(-size // 256) * 256 + GUARD
        self.memory = torch.full((end,), MARK, dtype=torch.uint8, device="cuda")

    def __getitem__(self, name):
        return self.memory.data_ptr() + self.at[name][0]

    def untouched(self):
        outside = torch.ones(self.memory.numel(), dtype=torch.bool, device="cuda")
        for start, size in self.at.values():
            outside[start:start + size] = False
        return bool((self.memory[outside] == MARK).all())


def guarded_calls(args, cu, d_o, d_s):
    """Both directions through the C entries, every output and the workspace between guards."""
    import struct

    from metal_linalg_torch import _delta
    q, k, v, g, beta, s0 = args
    p = _delta._problem(q, k, v, g, beta, 0.5, s0, cu, cu.element_size())
    size = lambda *xs: [x.numel() * x.element_size() for x in xs]  # noqa: E731
    need = [_lib.lib.metal_linalg_gated_delta_rule_workspace_bytes(p, back) for back in (0, 1)]
    _lib.use_stream_of(q)
    sizes = dict(zip(("o", "s"), size(v, s0)))
    b = Guarded(**sizes, ws=need[0])
    _lib.check(_lib.lib.metal_linalg_gated_delta_rule(p, b["o"], b["s"], b["ws"], need[0]))
    torch.cuda.synchronize()
    assert b.untouched()
    b = Guarded(**dict(zip(("dq", "dk", "dv", "dg", "db", "ds"), size(*args))), ws=need[1])
    _lib.check(_lib.lib.metal_linalg_gated_delta_rule_backward(p, d_o.data_ptr(), struct.pack("=3q", *d_o.stride()[:3]), d_s.data_ptr(),
                                                               *(b[n] for n in ("dq", "dk", "dv", "dg", "db", "ds")), b["ws"], need[1]))
    torch.cuda.synchronize()
    assert b.untouched()


BAD = [[0, 300, 0, 300], [50, 40, 30, 20], [-7, 100, 5000, 300], [0, 2 ** 31 - 1, 0, 2 ** 31 - 1], [300, 0, 300, 0], [-5, -4, -3, -2],
       [2 ** 31 - 1] * 4, [-2 ** 31, 2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1], [300, 300, 300, 0], [0, 65, 64, 300]]


@pytest.mark.gpu
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("bounds", BAD, ids=str)
def test_bad_bounds_write_nothing_outside(bounds, index):
    args, _ = ragged([100, 100, 100], 1, 2, 32, 40, torch.float32)
    cu = torch.tensor(bounds, dtype=index).cuda()
    guarded_calls(args, cu, torch.randn_like(args[2]), torch.randn_like(args[5]))


@pytest.mark.gpu
def test_overlapping_sequences_of_more_chunks_than_an_int_counts():
    """32768 times all of 2^22 tokens: 2^31 chunks by their bounds, of which there is room for 131071."""
    t, n = 1 << 22, 65535
    one = torch.zeros(1, 1, 1, 16, device="cuda", dtype=torch.bfloat16)
    q = one.expand(1, t, 1, 16)
    gate = torch.zeros(1, 1, 1, device="cuda").expand(1, t, 1)
    s0 = torch.ones(n, 1, 16, 16, device="cuda")
    cu = (torch.arange(n + 1) % 2 * t).to("cuda", torch.int32)
    guarded_calls((q, q, q, gate, gate, s0), cu, q, s0)


# ---------------------------------------------------------------------------
# Every way in which warps share a chain. Which one a call takes goes by its number of chains (16 value columns of a value head
# and sequence): with one chain a multiprocessor (148) at most, four warps, forward in 16 bits up to two; then two; backward
# one beyond two chains a multiprocessor, but for float16 and ragged batches.
# ---------------------------------------------------------------------------

def recurrence_and_gradients(args, d_o, d_s, cu=None):
    """In float64, token by token, on the GPU (torch's own operations): a ragged batch's sequences by themselves."""
    leaves = [x.detach().double().requires_grad_() for x in args]
    q, k, v, g, beta, s0 = leaves
    up = v.shape[2] // q.shape[2]
    spans = [(slice(None), 0, q.shape[1])] if cu is None else [(slice(i, i + 1), a, b) for i, (a, b) in enumerate(zip(cu, cu[1:]))]
    outs, states = [], []
    for rows, a, b in spans:
        s = s0[rows]
        for t in range(a, b):
            kt, qt = (x[:, t].repeat_interleave(up, 1)[..., None] for x in (k, q))
            s = s * g[:, t].exp()[..., None, None]
            s = s + kt * (beta[:, t, :, None] * (v[:, t] - (kt * s).sum(-2)))[..., None, :]
            outs.append(q.shape[-1] ** -0.5 * (qt * s).sum(-2))
        states.append(s)
    o, s = torch.stack(outs, 1), torch.cat(states)
    return o.detach(), s.detach(), torch.autograd.grad((o, s), leaves, (d_o.double(), d_s.double()))


def check_all(args, dtype, cu=None):
    leaves = [x.detach().requires_grad_() for x in args]
    bounds = None if cu is None else torch.tensor(cu, device="cuda", dtype=torch.int32)
    o, s = mlt.gated_delta_rule(*leaves[:5], initial_state=leaves[5], cu_seqlens=bounds)
    gen = torch.Generator(device="cuda").manual_seed(7)
    d_o = torch.randn(o.shape, device="cuda", generator=gen).to(dtype)
    d_s = 0.3 * torch.randn(s.shape, device="cuda", generator=gen)
    got = torch.autograd.grad((o, s), leaves, (d_o, d_s), retain_graph=True)
    want_o, want_s, want = recurrence_and_gradients(args, d_o, d_s, cu)
    near(o, want_o.cpu(), tolerance(dtype), "o")
    near(s, want_s.cpu(), F32, "state")
    for name, x, y in zip(NAMES, got, want):
        near(x, y.cpu(), tolerance(x.dtype, grad=True), name)
    assert all(torch.equal(x, y) for x, y in zip(got, torch.autograd.grad((o, s), leaves, (d_o, d_s))))


@pytest.mark.gpu
@pytest.mark.parametrize("dk", [64, 128])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("chains", [144, 160, 320])
def test_chains_of_several_chunks(chains, dtype, dk):
    """Forward by four warps (144; 16 bits: 160), by two (float32: 160; 320); backward by four, two, one (float16: two)."""
    hv = chains // 16
    check_all(inputs(2, 215, hv // 2 if hv % 2 == 0 else hv, hv, dk, 128, dtype, seed=chains), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dk", [60, 128])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens", [[130, 0, 215, 64], [3, 130, 64, 0, 70, 215, 129, 1, 66, 100]], ids=len)
def test_ragged_chains_of_several_chunks(lens, dtype, dk):
    """96 and 240 chains: four warps a chain, and two."""
    args, cu = ragged(lens, 2, 4, dk, 96, dtype, seed=len(lens))
    check_all(args, dtype, cu.tolist())


@pytest.mark.gpu
def test_what_no_sequence_holds_is_not_read():
    """Tokens of no sequence, and the inputs of a step's padding rows, may hold anything."""
    q, k, v, g, beta, s0 = inputs(1, 300, 1, 2, 32, 48, torch.float32, n=2)
    cu = torch.tensor([70, 130, 210], device="cuda")
    d_o, d_s = torch.randn_like(v), torch.randn_like(s0)

    def run(*args, d_o):
        leaves = [x.detach().clone().requires_grad_() for x in args]
        o, s = mlt.gated_delta_rule(*leaves[:5], initial_state=leaves[5], cu_seqlens=cu)
        return (o, s, *torch.autograd.grad((o, s), leaves, (d_o, d_s)))

    want = run(q, k, v, g, beta, s0, d_o=d_o)
    bad = [x.clone() for x in (q, k, v, g, beta, d_o)]
    for i, x in enumerate(bad):
        x[:, :70] = (math.nan, math.inf, -math.inf)[i % 3]
        x[:, 210:] = (math.inf, math.nan)[i % 2]
    assert all(torch.equal(x, y) for x, y in zip(run(*bad[:5], s0, d_o=bad[5]), want))
    q, k, v, g, beta, s0 = inputs(3, 1, 1, 2, 32, 48, torch.float32)
    slots = torch.tensor([1, -1, 0], device="cuda")
    for x in (q, k, v, g, beta):
        x[1] = math.nan
    state = s0.clone()
    o = mlt.gated_delta_step(q, k, v, g, beta, state, slots=slots)
    assert not o[1].any() and state.isfinite().all() and o.isfinite().all() and torch.equal(state[2], s0[2])


@pytest.mark.gpu
def test_decoding_in_inference_mode():
    args = inputs(2, 70, 1, 2, 32, 32, torch.bfloat16)
    want_o, want_s = mlt.gated_delta_rule(*args[:5], initial_state=args[5])
    last = [x[:, -1:] for x in args[:5]]
    with torch.no_grad():
        pool = want_s.clone()
        want = mlt.gated_delta_step(*last, pool)
    with torch.inference_mode():
        o, state = mlt.gated_delta_rule(*args[:5], initial_state=args[5])
        got = mlt.gated_delta_step(*last, state)
    assert torch.equal(o, want_o) and torch.equal(got, want) and torch.equal(state, pool)
