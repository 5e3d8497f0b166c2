"""The gated delta rule for PyTorch: `gated_delta_rule` (whole sequences, differentiable) and
`gated_delta_step` (a few tokens a sequence on a pool of states, in place).

A state S [Dk, Dv] for each value head is carried through the tokens of a sequence,

    S <- exp(g_t) S;   d_t = beta_t (v_t - S^T k_t);   S <- S + k_t d_t^T;   o_t = scale S^T q_t,

a product of decayed (generalised) Householder reflections: the library computes it in chunks of 64 tokens by their
compact-WY form, as its QR keeps its row blocks. States, sums and gates are float32 (sums of gates 64 bits) whatever
the inputs' type; results are rounded once.

Calls take CUDA tensors and enqueue on torch's current stream of the tensors' device. The workspace is a tensor of
torch's allocator, so calls on several streams and in several captured graphs never share one.
"""
import struct

import torch
from torch import Tensor

from . import _lib
from ._eager import direct

__all__ = ["gated_delta_rule", "gated_delta_step"]

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_FLOATING = frozenset((torch.float32, torch.bfloat16, torch.float16, torch.float64))
_PLACES = frozenset(("cuda", "meta"))
_INDICES = frozenset((torch.int32, torch.int64))
_changed = torch.autograd.graph.increment_version
_PROBLEM = struct.Struct("=9IfiI7Q15q")


def _fail(name, message, kind=ValueError):
    raise kind(f"metal_linalg_torch.{name}: {message}")


def _check(name, q, k, v, g, beta):
    """Refuses inputs the library cannot take; returns their sizes."""
    try:
        shape, v_shape, dtype, device = q.shape, v.shape, q.dtype, q.device
        fine = (len(shape) == 4 and len(v_shape) == 4 and k.shape == shape and v_shape[:2] == shape[:2] and dtype in _DTYPES
                and k.dtype == dtype and v.dtype == dtype and g.shape == v_shape[:3] and beta.shape == v_shape[:3]
                and g.dtype in _FLOATING and beta.dtype in _FLOATING and v_shape[2] % max(shape[2], 1) == 0 and shape[2] and v_shape[2]
                and 1 <= shape[3] <= 128 and 1 <= v_shape[3] <= 256 and device.type in _PLACES
                and k.device == device and v.device == device and g.device == device and beta.device == device)
    except AttributeError:
        fine = False
    if not fine:
        _explain(name, q, k, v, g, beta)
    return (*shape, *v_shape[2:])


def _explain(name, q, k, v, g, beta):
    """Says what is wrong with inputs that _check found wanting."""
    for what, x in (("q", q), ("k", k), ("v", v), ("g", g), ("beta", beta)):
        if not isinstance(x, Tensor):
            _fail(name, f"{what} must be a tensor, got {type(x).__name__}", TypeError)
    if q.dtype not in _DTYPES:
        _fail(name, f"q, k and v must be float32, bfloat16 or float16, got {q.dtype}", TypeError)
    if k.dtype != q.dtype or v.dtype != q.dtype:
        _fail(name, f"q, k and v must have one dtype, got {q.dtype}, {k.dtype} and {v.dtype}", TypeError)
    if g.dtype not in _FLOATING or beta.dtype not in _FLOATING:
        _fail(name, f"g and beta must be floating point, got {g.dtype} and {beta.dtype}", TypeError)
    if q.dim() != 4 or v.dim() != 4 or k.shape != q.shape or v.shape[:2] != q.shape[:2]:
        _fail(name, "expected q and k [B, T, H, Dk] and v [B, T, HV, Dv], got "
                    f"{tuple(q.shape)}, {tuple(k.shape)} and {tuple(v.shape)}")
    h, dk = q.shape[2:]
    hv, dv = v.shape[2:]
    if g.shape != v.shape[:3] or beta.shape != v.shape[:3]:
        _fail(name, f"expected g and beta [B, T, HV] = {tuple(v.shape[:3])}, got {tuple(g.shape)} and {tuple(beta.shape)}")
    if h == 0 or hv == 0 or hv % h:
        _fail(name, f"the {hv} heads of v must be a multiple of the {h} of q and k")
    if not 1 <= dk <= 128 or not 1 <= dv <= 256:
        _fail(name, f"Dk must be 1 to 128 and Dv 1 to 256, got {dk} and {dv}")
    if q.device.type not in _PLACES:
        _fail(name, f"tensors on {q.device} are not supported; use CUDA (this library has no CPU path)")
    for what, x in (("k", k), ("v", v), ("g", g), ("beta", beta)):
        if x.device != q.device:
            _fail(name, f"{what} is on {x.device}, q on {q.device}")
    _fail(name, "unsupported inputs")


def _rows(x):
    return x if x.stride(-1) == 1 or x.shape[-1] <= 1 else x.contiguous()


def _float(x):
    return x if x.dtype == torch.float32 else x.float()


def _scale(scale, dk):
    return float(dk) ** -0.5 if scale is None else float(scale)


def _problem(q, k, v, g, beta, scale, initial=None, cu=None, index_bytes=4):
    """A metal_linalg_delta as bytes."""
    b, t, h, dk = q.shape
    _, _, hv, dv = v.shape
    q0, q1, q2, _ = q.stride()
    k0, k1, k2, _ = k.stride()
    v0, v1, v2, _ = v.stride()
    return _PROBLEM.pack(b, t, h, hv, dk, dv, 0 if cu is None else cu.numel() - 1, _DTYPES[q.dtype], index_bytes, scale,
                         q.get_device(), 0, q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(),
                         0 if initial is None else initial.data_ptr(), 0 if cu is None else cu.data_ptr(),
                         q0, q1, q2, k0, k1, k2, v0, v1, v2, *g.stride(), *beta.stride())


def _workspace(problem, backward, device):
    size = _lib.lib.metal_linalg_gated_delta_rule_workspace_bytes(problem, int(backward))
    return torch.empty(size, dtype=torch.uint8, device=device)


def _sequences(name, q, cu_seqlens):
    if cu_seqlens is None:
        return q.shape[0]
    if not isinstance(cu_seqlens, Tensor) or cu_seqlens.dtype not in _INDICES:
        _fail(name, "cu_seqlens must be an int32 or int64 tensor", TypeError)
    if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 2:
        _fail(name, f"cu_seqlens must hold the N + 1 bounds of N >= 1 sequences, got shape {tuple(cu_seqlens.shape)}")
    if q.shape[0] != 1:
        _fail(name, f"with cu_seqlens the sequences lie in one row: B must be 1, got {q.shape[0]}")
    if cu_seqlens.device != q.device:
        _fail(name, f"cu_seqlens is on {cu_seqlens.device}, q on {q.device}")
    return cu_seqlens.numel() - 1


def _forward(q, k, v, g, beta, scale, initial, cu):
    q, k, v = _rows(q), _rows(k), _rows(v)
    cu = None if cu is None else cu.contiguous()
    n = q.shape[0] if cu is None else cu.numel() - 1
    hv, dv = v.shape[2:]
    o = v.new_empty(v.shape)
    last = g.new_empty((n, hv, q.shape[3], dv))
    p = _problem(q, k, v, g, beta, scale, initial, cu, 4 if cu is None else cu.element_size())
    ws = _workspace(p, False, v.device)
    _lib.use_stream_of(v)
    _lib.check(_lib.lib.metal_linalg_gated_delta_rule(p, o.data_ptr(), last.data_ptr(), ws.data_ptr(), ws.numel()))
    return o, last


def _backward(d_o, d_last, q, k, v, g, beta, scale, initial, cu):
    q, k, v, d_o = _rows(q), _rows(k), _rows(v), _rows(d_o)
    d_last = None if d_last is None else d_last.contiguous()
    cu = None if cu is None else cu.contiguous()
    new = lambda x: x.new_empty(x.shape)  # noqa: E731
    dq, dk, dv, dg, dbeta = new(q), new(k), new(v), new(g), new(beta)
    d_initial = None if initial is None else new(initial)
    p = _problem(q, k, v, g, beta, scale, initial, cu, 4 if cu is None else cu.element_size())
    ws = _workspace(p, True, v.device)
    strides = struct.pack("=3q", *d_o.stride()[:3])
    _lib.use_stream_of(v)
    _lib.check(_lib.lib.metal_linalg_gated_delta_rule_backward(
        p, d_o.data_ptr(), strides, None if d_last is None else d_last.data_ptr(), dq.data_ptr(), dk.data_ptr(),
        dv.data_ptr(), dg.data_ptr(), dbeta.data_ptr(), None if d_initial is None else d_initial.data_ptr(),
        ws.data_ptr(), ws.numel()))
    return dq, dk, dv, dg, dbeta, d_initial


@torch.library.custom_op("metal_linalg::gated_delta_rule", mutates_args=())
def _rule_op(q: Tensor, k: Tensor, v: Tensor, g: Tensor, beta: Tensor, scale: float, initial_state: Tensor | None,
             cu_seqlens: Tensor | None) -> tuple[Tensor, Tensor]:
    return _forward(q, k, v, g, beta, scale, None if initial_state is None else initial_state.contiguous(), cu_seqlens)


@_rule_op.register_fake
def _(q, k, v, g, beta, scale, initial_state, cu_seqlens):
    n = q.shape[0] if cu_seqlens is None else cu_seqlens.shape[0] - 1
    return torch.empty_like(v, memory_format=torch.contiguous_format), v.new_empty((n, v.shape[2], q.shape[3], v.shape[3]), dtype=torch.float32)


@torch.library.custom_op("metal_linalg::gated_delta_rule_backward", mutates_args=())
def _rule_backward_op(d_o: Tensor, d_final: Tensor | None, q: Tensor, k: Tensor, v: Tensor, g: Tensor, beta: Tensor,
                      scale: float, initial_state: Tensor | None,
                      cu_seqlens: Tensor | None) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    got = _backward(d_o, d_final, q, k, v, g, beta, scale,
                    None if initial_state is None else initial_state.contiguous(), cu_seqlens)
    return (*got[:5], v.new_empty(0, dtype=torch.float32) if got[5] is None else got[5])


@_rule_backward_op.register_fake
def _(d_o, d_final, q, k, v, g, beta, scale, initial_state, cu_seqlens):
    new = lambda x: x.new_empty(x.shape)  # noqa: E731
    return (new(q), new(k), new(v), new(g), new(beta),
            v.new_empty(0, dtype=torch.float32) if initial_state is None else new(initial_state))


def _rule_setup(ctx, inputs, output):
    ctx.set_materialize_grads(False)
    q, k, v, g, beta, scale, initial, cu = inputs
    ctx.scale = scale
    ctx.save_for_backward(q, k, v, g, beta, initial, cu)


def _grads(ctx, d_o, d_last, run=None):
    q, k, v, g, beta, initial, cu = ctx.saved_tensors
    if d_o is None and d_last is None:
        return (None,) * 8
    if d_o is None:
        d_o = torch.zeros(v.shape, dtype=v.dtype, device=v.device)
    if run is None or not direct("gated_delta_rule", d_o, d_last, q, k, v, g, beta, initial, cu):
        run = torch.ops.metal_linalg.gated_delta_rule_backward
    dq, dk, dv, dg, dbeta, d_initial = run(d_o, d_last, q, k, v, g, beta, ctx.scale, initial, cu)
    return dq, dk, dv, dg, dbeta, None, None if initial is None else d_initial, None


_rule_op.register_autograd(_grads, setup_context=_rule_setup)


class _Rule(torch.autograd.Function):
    """The operator without the dispatcher's detour, for eager calls that need a gradient."""

    @staticmethod
    def forward(ctx, q, k, v, g, beta, scale, initial, cu):
        _rule_setup(ctx, (q, k, v, g, beta, scale, initial, cu), None)
        return _forward(q, k, v, g, beta, scale, initial, cu)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_o, d_last):
        return _grads(ctx, d_o, d_last, _backward)


def gated_delta_rule(q, k, v, g, beta, *, scale=None, initial_state=None, cu_seqlens=None):
    """The gated delta rule over whole sequences. Returns ``(o, final_state)``.

    ``q``, ``k`` [B, T, H, Dk] and ``v`` [B, T, HV, Dv] are float32, bfloat16 or float16; HV is a multiple of H and value
    head ``i`` reads head ``i // (HV / H)`` of q and k. ``g`` [B, T, HV] are the logarithms of the decays (at most 0 as
    a rule; ``-inf`` clears the state) and ``beta`` [B, T, HV] the steps, in any floating type, used in float32. Dk is at
    most 128, Dv at most 256. ``scale`` multiplies the outputs (default Dk ** -0.5). Any strides are taken as they are as
    long as the last dimensions of q, k and v are contiguous; others are copied.

    Each batch row is a sequence. With ``cu_seqlens`` (int32 or int64, on the GPU, N + 1 values from 0 on, none falling) B is
    1 and sequence ``i`` is the tokens ``cu_seqlens[i] .. cu_seqlens[i + 1] - 1``; a sequence may be empty, and tokens of no
    sequence give zeros. ``initial_state`` [B or N, HV, Dk, Dv] (float32; default zero) is where each starts;
    ``final_state`` has its shape. ``o`` has v's shape and type. At most 65535 sequences, fewer than 2 ** 30 tokens each.

    Differentiable once in q, k, v, g, beta and initial_state, through both results (not in forward mode).
    """
    name = "gated_delta_rule"
    b, t, h, dk, hv, dv = _check(name, q, k, v, g, beta)
    n = _sequences(name, q, cu_seqlens)
    if initial_state is not None:
        if not isinstance(initial_state, Tensor) or initial_state.dtype != torch.float32:
            _fail(name, "initial_state must be a float32 tensor", TypeError)
        if initial_state.shape != (n, hv, dk, dv):
            _fail(name, f"expected initial_state {(n, hv, dk, dv)}, got {tuple(initial_state.shape)}")
        if initial_state.device != q.device:
            _fail(name, f"initial_state is on {initial_state.device}, q on {q.device}")
    scale = _scale(scale, dk)
    g, beta = _float(g), _float(beta)
    if not direct(name, q, k, v, g, beta, initial_state, cu_seqlens):
        return torch.ops.metal_linalg.gated_delta_rule(q, k, v, g, beta, scale, initial_state, cu_seqlens)
    initial = None if initial_state is None else initial_state.contiguous()
    tensors = (q, k, v, g, beta) if initial is None else (q, k, v, g, beta, initial)
    if torch.is_grad_enabled() and any(x.requires_grad for x in tensors):
        return _Rule.apply(q, k, v, g, beta, scale, initial, cu_seqlens)
    return _forward(q, k, v, g, beta, scale, initial, cu_seqlens)


def _step(q, k, v, g, beta, state, slots, scale):
    q, k, v = _rows(q), _rows(k), _rows(v)
    slots = None if slots is None else slots.contiguous()
    o = v.new_empty(v.shape)
    p = _problem(q, k, v, g, beta, scale, None, None, 4 if slots is None else slots.element_size())
    _lib.use_stream_of(v)
    _lib.check(_lib.lib.metal_linalg_gated_delta_step(p, o.data_ptr(), state.data_ptr(), state.stride(0), state.shape[0],
                                                      None if slots is None else slots.data_ptr()))
    return o


@torch.library.custom_op("metal_linalg::gated_delta_step", mutates_args=("state",))
def _step_op(q: Tensor, k: Tensor, v: Tensor, g: Tensor, beta: Tensor, state: Tensor, slots: Tensor | None,
             scale: float) -> Tensor:
    return _step(q, k, v, g, beta, state, slots, scale)


@_step_op.register_fake
def _(q, k, v, g, beta, state, slots, scale):
    return torch.empty_like(v, memory_format=torch.contiguous_format)


def _explain_step(name, q, b, hv, dk, dv, state, slots):
    """Refuses a pool or slots that cannot be used; returns where the pool's strides only look unusual (dimensions of one)."""
    if not isinstance(state, Tensor) or state.dtype != torch.float32:
        _fail(name, "state must be a float32 tensor", TypeError)
    if state.dim() != 4 or state.shape[1:] != (hv, dk, dv):
        _fail(name, f"expected state [S, {hv}, {dk}, {dv}], got {tuple(state.shape)}")
    if state.device != q.device:
        _fail(name, f"state is on {state.device}, q on {q.device}")
    s0, s1, s2, s3 = state.stride()
    if state.numel() and (s3 != 1 and dv > 1 or s2 != dv and dk > 1 or s1 != dk * dv and hv > 1):
        _fail(name, f"each slot of state must be contiguous, got strides {tuple(state.stride())}")
    if state.shape[0] > 1 and s0 < hv * dk * dv:
        _fail(name, "the slots of state overlap")
    if slots is not None:
        if not isinstance(slots, Tensor) or slots.dtype not in _INDICES:
            _fail(name, "slots must be an int32 or int64 tensor", TypeError)
        if slots.shape != (b,) or slots.device != q.device:
            _fail(name, f"expected slots [{b}] on {q.device}, got {tuple(slots.shape)} on {slots.device}")
    elif b > state.shape[0]:
        _fail(name, f"{b} rows and {state.shape[0]} slots: name them with slots")


def gated_delta_step(q, k, v, g, beta, state, *, slots=None, scale=None):
    """A few tokens of every sequence through the gated delta rule, for decoding; updates ``state`` in place and returns
    ``o`` [B, T, HV, Dv].

    The inputs are `gated_delta_rule`'s (T is 1, or the tokens of a draft). ``state`` is a pool [S, HV, Dk, Dv] of float32
    states, each contiguous (a layer's part of a larger cache is fine). Row ``b`` uses slot ``slots[b]`` (int32 or int64, on
    the GPU; default: slot ``b``). A row whose slot is not one of the pool's, -1 say, is padding: its outputs are zero and no
    state changes. Rows that name the same slot run one after another, in their order. At most 65535 rows. Not differentiable.
    """
    name = "gated_delta_step"
    b, t, h, dk, hv, dv = _check(name, q, k, v, g, beta)
    try:
        shape, (s0, s1, s2, s3) = state.shape, state.stride()
        fine = (state.dtype == torch.float32 and shape[1:] == (hv, dk, dv) and state.device == q.device
                and s3 == 1 and s2 == dv and s1 == dk * dv and s0 >= hv * s1
                and (b <= shape[0] if slots is None else slots.dtype in _INDICES and slots.shape == (b,) and slots.device == q.device))
    except (AttributeError, ValueError):
        fine = False
    if not fine:
        _explain_step(name, q, b, hv, dk, dv, state, slots)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or g.requires_grad or
                                    beta.requires_grad or state.requires_grad):
        _fail(name, "not differentiable; use gated_delta_rule for training, or torch.no_grad()", RuntimeError)
    scale = _scale(scale, dk)
    g, beta = _float(g), _float(beta)
    if not direct(name, q, k, v, g, beta, state, slots):
        return torch.ops.metal_linalg.gated_delta_step(q, k, v, g, beta, state, slots, scale)
    _changed(state)                 # a graph that saved the pool for its backward pass finds it changed
    return _step(q, k, v, g, beta, state, slots, scale)
