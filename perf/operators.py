"""What is measured of the sequence and 8-bit operators, and their plain forms.

`run` with `own` false computes each operator with elementary torch operations in 32 bits (decays' exponents in 64,
where sums of many gates are subtracted from one another); with `own` true it makes the calls a user makes:

    gated_delta_rule    a prompt through the gated delta rule, forward alone or with every gradient
    gated_delta_step    single tokens on a pool of states, in place
    quantize_fp8        blocks of 128 (or 128 x 128) to 8-bit floating point with a float32 scale each
    matmul_fp8          the product of two such operands
    linear_fp8          a linear map on quantised operands, forward and backward (six quantisations, three products)
"""
import math
import os
import random
import sys

import torch

own = False

CHUNK = 64
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
FP8_MAX = 448.0                       # of e4m3


def _package():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "metal-linalg_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import metal_linalg_torch
    return metal_linalg_torch


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------

def _delta(name, batch, tokens, heads, value_heads, dk, dv, dtype, seqs=0, grad=False):
    return {"name": name, "op": "delta", "batch": batch, "tokens": tokens, "heads": heads, "value_heads": value_heads,
            "dk": dk, "dv": dv, "dtype": dtype, "seqs": seqs, "grad": grad}


def _step(name, batch, tokens, heads, value_heads, dk, dv, dtype, pool):
    return {"name": name, "op": "step", "batch": batch, "tokens": tokens, "heads": heads, "value_heads": value_heads,
            "dk": dk, "dv": dv, "dtype": dtype, "pool": pool}


def listed():
    return [
        # one request's next token: nothing but latency
        _step("step 1", 1, 1, 4, 8, 128, 128, "bf16", 1),
        # a full decoding batch on a pool of states with free slots between, two rows of padding
        _step("step 128 of a pool", 128, 1, 16, 32, 128, 128, "bf16", 160),
        # a short prompt of odd length, heads narrower than the tensor core's tiles
        _delta("prompt 1000", 1, 1000, 4, 8, 64, 96, "fp16"),
        # a ragged batch of prompts packed behind one another, each with a state to go on from
        _delta("ragged 8192", 1, 8192, 8, 16, 128, 128, "bf16", seqs=11),
        # one long document
        _delta("long 32768", 1, 32768, 8, 16, 128, 128, "bf16"),
        # a training step's layer in float32, small
        _delta("train 2 x 777 fp32", 2, 777, 4, 4, 64, 64, "fp32", grad=True),
        # a training step's layer
        _delta("train 2 x 4096", 2, 4096, 8, 16, 128, 128, "bf16", grad=True),
        # a weight matrix in 128 x 128 blocks
        {"name": "quantise weight", "op": "quantize", "rows": 4096, "cols": 8192, "block": 128, "transpose": False, "dtype": "bf16"},
        # activations transposed for a weight's gradient, odd sizes, float32
        {"name": "quantise transposed", "op": "quantize", "rows": 1999, "cols": 2050, "block": 1, "transpose": True, "dtype": "fp32"},
        # a decoding batch against a weight
        {"name": "product 16 rows", "op": "matmul", "m": 16, "n": 4096, "k": 8192, "b_block": 128, "out": "bf16"},
        # a prompt's projection
        {"name": "product 8192 rows", "op": "matmul", "m": 8192, "n": 8192, "k": 4096, "b_block": 128, "out": "bf16"},
        # a training step's projection, forward and backward
        {"name": "linear train", "op": "linear", "m": 4096, "n": 4096, "k": 2048, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("step", "delta", "delta", "train", "quantize", "matmul", "linear"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    heads = rng.choice((1, 2, 3, 4, 8))
    value_heads = heads * rng.choice((1, 1, 2, 4))
    dk = rng.choice((128, 128, 64, rng.randint(8, 128)))
    dv = rng.choice((128, 128, 64, rng.randint(8, 128)))
    if op == "step":
        batch = _log_int(rng, 1, 128)
        c = _step("", batch, rng.choice((1, 1, 1, 2, 4)), heads, value_heads, dk, dv, dtype, batch + rng.randint(0, 40))
    elif op == "delta":
        tokens = _log_int(rng, 1, 16384)
        seqs = rng.choice((0, 0, rng.randint(1, 24)))
        batch = 1 if seqs else rng.choice((1, 2, 3)) if tokens <= 4096 else 1
        c = _delta("", batch, tokens, heads, value_heads, dk, dv, dtype, seqs=seqs)
    elif op == "train":
        tokens = _log_int(rng, 1, 4096)
        seqs = rng.choice((0, 0, rng.randint(1, 12)))
        c = _delta("", 1 if seqs else rng.choice((1, 2)), tokens, min(heads, 4), min(heads, 4) * rng.choice((1, 2)), dk, dv,
                   dtype, seqs=seqs, grad=True)
    elif op == "quantize":
        c = {"op": "quantize", "rows": _log_int(rng, 1, 8192), "cols": _log_int(rng, 16, 8192), "block": rng.choice((1, 128)),
             "transpose": rng.choice((False, True)), "dtype": dtype}
    elif op == "matmul":
        c = {"op": "matmul", "m": _log_int(rng, 1, 8192), "n": _log_int(rng, 16, 8192), "k": _log_int(rng, 16, 4096),
             "b_block": rng.choice((1, 128, 128)), "out": dtype}
    else:
        c = {"op": "linear", "m": _log_int(rng, 1, 4096), "n": _log_int(rng, 16, 4096), "k": _log_int(rng, 16, 2048), "dtype": dtype}
    c.pop("name", None)
    return c


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _delta_inputs(c, gen, batch, tokens):
    """Queries and keys as a gated layer makes them (silu, unit length), gates -A softplus(x) with a rate A for each head."""
    dt, dev = DTYPES[c["dtype"]], "cuda"
    silu = torch.nn.functional.silu

    def unit(*shape):
        x = silu(torch.randn(*shape, device=dev, generator=gen))
        return (x / x.norm(dim=-1, keepdim=True).clamp_min(1e-6)).to(dt)

    h, hv, dk, dv = c["heads"], c["value_heads"], c["dk"], c["dv"]
    q, k = unit(batch, tokens, h, dk), unit(batch, tokens, h, dk)
    v = silu(torch.randn(batch, tokens, hv, dv, device=dev, generator=gen)).to(dt)
    beta = torch.sigmoid(torch.randn(batch, tokens, hv, device=dev, generator=gen))
    rate = 16.0 * torch.rand(hv, device=dev, generator=gen)
    bias = torch.empty(hv, device=dev).uniform_(math.log(1e-3), math.log(1e-1), generator=gen)
    g = -rate * torch.nn.functional.softplus(0.5 * torch.randn(batch, tokens, hv, device=dev, generator=gen) + bias)
    return q, k, v, g, beta


def _lengths(total, seqs, seed):
    """`seqs` lengths that add up to `total`, uneven; one may be empty."""
    r = random.Random(seed)
    cuts = sorted(int(total * r.random() ** 1.3) for _ in range(seqs - 1))
    ends = [0] + cuts + [total]
    return [b - a for a, b in zip(ends, ends[1:])]


def _fp8_operand(rows, cols, block, gen):
    """An 8-bit operand [rows, cols] and its scales, in rows a multiple of 16 bytes apart."""
    wide = -(-cols // 16) * 16
    values = torch.randn(rows, wide, device="cuda", generator=gen) * 90.0
    values = values.clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)[:, :cols]
    scale = torch.exp(torch.randn(-(-rows // block), -(-cols // 128), device="cuda", generator=gen)) * 1e-2
    return values, scale


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": c}
    if c["op"] == "delta":
        q, k, v, g, beta = _delta_inputs(c, gen, c["batch"], c["tokens"])
        lens = _lengths(c["tokens"], c["seqs"], seed) if c["seqs"] else None
        n = c["seqs"] or c["batch"]
        s0 = torch.randn(n, c["value_heads"], c["dk"], c["dv"], device="cuda", generator=gen) * 0.1
        s.update(q=q, k=k, v=v, g=g, beta=beta, s0=s0, cu=None, longest=c["tokens"])
        if lens is not None:
            s["longest"] = max(lens)
            s["cu"] = torch.tensor([0] + lens, device="cuda").cumsum(0).to(torch.int32)
        if c["grad"]:
            s["do"] = torch.randn(v.shape, device="cuda", generator=gen).to(v.dtype)
            s["ds"] = torch.randn(s0.shape, device="cuda", generator=gen) * 0.1
            for name in ("q", "k", "v", "g", "beta", "s0"):
                s[name].requires_grad_(True)
    elif c["op"] == "step":
        q, k, v, g, beta = _delta_inputs(c, gen, c["batch"], c["tokens"])
        pool = torch.randn(c["pool"], c["value_heads"], c["dk"], c["dv"], device="cuda", generator=gen) * 0.1
        slots = torch.randperm(c["pool"], device="cuda", generator=gen)[:c["batch"]].to(torch.int32)
        if c["batch"] > 2:
            slots[-2:] = -1                                   # rows of padding
        s.update(q=q, k=k, v=v, g=g, beta=beta, pool=pool, slots=slots)
    elif c["op"] == "quantize":
        x = torch.randn(c["rows"], c["cols"], device="cuda", generator=gen)
        s["x"] = (x * torch.exp(torch.randn(c["rows"], 1, device="cuda", generator=gen))).to(DTYPES[c["dtype"]])
    elif c["op"] == "matmul":
        s["a"], s["sa"] = _fp8_operand(c["m"], c["k"], 1, gen)
        s["b"], s["sb"] = _fp8_operand(c["n"], c["k"], c["b_block"], gen)
    else:
        dt = DTYPES[c["dtype"]]
        s["x"] = torch.randn(c["m"], c["k"], device="cuda", generator=gen).to(dt).requires_grad_(True)
        s["w"] = (torch.randn(c["n"], c["k"], device="cuda", generator=gen) / math.sqrt(c["k"])).to(dt).requires_grad_(True)
        s["dy"] = torch.randn(c["m"], c["n"], device="cuda", generator=gen).to(dt)
    return s


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------

def _lower_inverse(a):
    """(I + a)^-1 for strictly lower triangular blocks of 64: blocks of 1, 2, 4 ... joined,
    [[X, 0], [C, Y]]^-1 = [[X^-1, 0], [-Y^-1 C X^-1, Y^-1]]."""
    n = a.shape[-1]
    inv = torch.ones(*a.shape[:-2], n, 1, 1, dtype=a.dtype, device=a.device)        # [..., blocks, size, size]
    size = 1
    while size < n:
        pairs = n // (2 * size)
        blocks = a.reshape(*a.shape[:-2], pairs, 2 * size, pairs, 2 * size)
        at = torch.arange(pairs, device=a.device)
        blocks = blocks.transpose(-3, -2)[..., at, at, :, :]
        x, y = inv[..., 0::2, :, :], inv[..., 1::2, :, :]
        below = -(y @ blocks[..., size:, :size] @ x)
        inv = torch.cat([torch.cat([x, torch.zeros_like(below)], -1), torch.cat([below, y], -1)], -2)
        size *= 2
    return inv[..., 0, :, :]


def _plain_delta(q, k, v, g, beta, s0, scale):
    """[N, T, HV, D] in float32, T a multiple of the chunk: (o, final state)."""
    n, t, h, _ = q.shape
    cut = lambda x: x.transpose(1, 2).reshape(n, h, t // CHUNK, CHUNK, *x.shape[3:])  # noqa: E731
    q, k, v, g, beta = cut(q), cut(k), cut(v), cut(g.double()), cut(beta)
    total = g.cumsum(-1)
    lower = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=q.device).tril()
    decay = (total[..., :, None] - total[..., None, :]).masked_fill(~lower, -math.inf).exp().float()
    e, left = total.exp().float()[..., None], (total[..., -1:] - total).exp().float()[..., None]
    last = total[..., -1].exp().float()[..., None, None]
    strict = lower.tril(-1)
    inv = _lower_inverse((k @ k.mT) * decay * beta[..., None] * strict)
    p = (q @ k.mT) * decay
    s, out = s0, []
    for i in range(t // CHUNK):
        r = beta[:, :, i, :, None] * (v[:, :, i] - e[:, :, i] * (k[:, :, i] @ s))
        d = inv[:, :, i] @ r
        out.append(scale * (e[:, :, i] * (q[:, :, i] @ s) + p[:, :, i] @ d))
        s = last[:, :, i] * s + (left[:, :, i] * k[:, :, i]).mT @ d
    o = torch.stack(out, 2).reshape(n, h, t, -1).transpose(1, 2) if out else v.new_zeros(n, t, h, v.shape[-1])
    return o, s


def _spread(x, cu, longest, length):
    """[1, total, ...] -> [N, length, ...] with zeros behind each sequence."""
    at = cu[:-1, None].long() + torch.arange(length, device=x.device)
    fits = at < cu[1:, None]
    y = x[0][at.clamp(max=x.shape[1] - 1)]
    return y * fits.reshape(*fits.shape, *[1] * (x.dim() - 2)).to(y.dtype)


def _gather(o, cu, total):
    """The inverse of _spread: [N, length, ...] -> [1, total, ...]."""
    at = torch.arange(total, device=o.device)
    row = torch.searchsorted(cu[1:].long(), at, right=True)
    return o[row, at - cu.long()[row]][None]


def _plain_delta_call(s):
    c = s["case"]
    q, k, v, g, beta, s0 = (s[n].float() for n in ("q", "k", "v", "g", "beta", "s0"))
    up = c["value_heads"] // c["heads"]
    q, k = q.repeat_interleave(up, 2), k.repeat_interleave(up, 2)
    length = -(-s["longest"] // CHUNK) * CHUNK
    if s["cu"] is not None:
        q, k, v, g, beta = (_spread(x, s["cu"], s["longest"], length) for x in (q, k, v, g, beta))
    else:
        pad = length - c["tokens"]
        q, k, v = (torch.nn.functional.pad(x, (0, 0, 0, 0, 0, pad)) for x in (q, k, v))
        g, beta = (torch.nn.functional.pad(x, (0, 0, 0, pad)) for x in (g, beta))
    o, last = _plain_delta(q, k, v, g, beta, s0, c["dk"] ** -0.5)
    o = _gather(o, s["cu"], c["tokens"]) if s["cu"] is not None else o[:, :c["tokens"]]
    return o.to(s["v"].dtype), last


def _plain_step(s):
    c = s["case"]
    up = c["value_heads"] // c["heads"]
    q, k = (s[n].float().repeat_interleave(up, 2) for n in ("q", "k"))
    v, g, beta = (s[n].float() for n in ("v", "g", "beta"))
    live = s["slots"] >= 0
    at = s["slots"].long()
    state = s["pool"][at.clamp_min(0)]
    out = []
    for t in range(c["tokens"]):
        state = state * g[:, t].exp()[..., None, None]
        d = beta[:, t, :, None] * (v[:, t] - (k[:, t, :, None, :] @ state)[..., 0, :])
        state = state + k[:, t, :, :, None] * d[..., None, :]
        out.append((q[:, t, :, None, :] @ state)[..., 0, :] * c["dk"] ** -0.5)
    o = (torch.stack(out, 1) * live[:, None, None, None]).to(s["v"].dtype)
    s["pool"].index_copy_(0, at[live], state[live])
    return o, s["pool"]


def _plain_quantize(x, block):
    """[M, N] -> values (e4m3) and scales [ceil(M / block), ceil(N / 128)]."""
    m, n = x.shape
    mb, nb = -(-m // block), -(-n // 128)
    y = torch.nn.functional.pad(x.float(), (0, nb * 128 - n, 0, mb * block - m)).reshape(mb, block, nb, 128)
    top = y.abs().amax((1, 3))
    scale = (top / torch.full_like(top, FP8_MAX)).clamp_min(2.0 ** -126)      # by a tensor: by a number it is a product with 1 / 448
    values = (y / scale[:, None, :, None]).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
    return values.reshape(mb * block, nb * 128)[:m, :n], scale


def _plain_dequantize(values, scale):
    m, n = values.shape
    block = 1 if scale.shape[0] == m else 128
    full = scale.repeat_interleave(block, 0)[:m].repeat_interleave(128, 1)[:, :n]
    return values.float() * full


def _plain_linear(x, w, dy):
    deq = lambda t, block: _plain_dequantize(*_plain_quantize(t, block))  # noqa: E731
    y = deq(x, 1) @ deq(w, 128).mT
    dx = deq(dy, 1) @ deq(w.mT, 128).mT
    dw = deq(dy.mT, 1) @ deq(x.mT, 1).mT
    return y.to(x.dtype), dx.to(x.dtype), dw.to(w.dtype)


def run(state):
    s = state
    c = s["case"]
    if c["op"] == "delta":
        if own:
            o, last = _package().gated_delta_rule(s["q"], s["k"], s["v"], s["g"], s["beta"], initial_state=s["s0"],
                                                  cu_seqlens=s["cu"])
        else:
            o, last = _plain_delta_call(s)
        if not c["grad"]:
            return o, last
        leaves = [s[n] for n in ("q", "k", "v", "g", "beta", "s0")]
        return (o.detach(), last.detach(), *torch.autograd.grad((o, last), leaves, (s["do"], s["ds"])))
    if c["op"] == "step":
        if own:
            o = _package().gated_delta_step(s["q"], s["k"], s["v"], s["g"], s["beta"], s["pool"], slots=s["slots"])
            return o, s["pool"]
        return _plain_step(s)
    if c["op"] == "quantize":
        if own:
            return _package().quantize_fp8(s["x"], block=(c["block"], 128), transpose=c["transpose"])
        return _plain_quantize(s["x"].mT if c["transpose"] else s["x"], c["block"])
    if c["op"] == "matmul":
        if own:
            return _package().matmul_fp8(s["a"], s["sa"], s["b"], s["sb"], out_dtype=DTYPES[c["out"]])
        return (_plain_dequantize(s["a"], s["sa"]) @ _plain_dequantize(s["b"], s["sb"]).mT).to(DTYPES[c["out"]])
    if own:
        y = _package().linear_fp8(s["x"], s["w"])
        return (y.detach(), *torch.autograd.grad(y, (s["x"], s["w"]), s["dy"]))
    return _plain_linear(s["x"].detach(), s["w"].detach(), s["dy"])


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    c = case
    if c["op"] in ("delta", "step"):
        size = 4 if c["dtype"] == "fp32" else 2
        tokens, h, hv, dk, dv = c["batch"] * c["tokens"], c["heads"], c["value_heads"], c["dk"], c["dv"]
        rows = tokens * (2 * h * dk + hv * dv) * size + tokens * hv * 8        # q, k, v, g, beta
        out = tokens * hv * dv * size
        if c["op"] == "step":
            live = c["batch"] - (2 if c["batch"] > 2 else 0)
            return {"bytes": rows + out + 2 * 4 * live * hv * dk * dv, "flops": 6 * live * c["tokens"] * hv * dk * dv}
        states = 4 * (c["seqs"] or c["batch"]) * hv * dk * dv
        # a chunk's useful products: K K^T and Q K^T (triangles), K S, Q S, K^T D, and T R, P D (triangles)
        forward = tokens * hv * (2 * CHUNK * dk + 6 * dk * dv + 2 * CHUNK * dv)
        if not c["grad"]:
            return {"bytes": rows + out + 2 * states, "flops": forward}
        # backward: P^T dO, T^T dD, dO D^T, dR D^T (triangles), four products with Q and K (triangles), K dS, Q^T dO, K^T dR,
        # dO S^T, dR S^T, D dS^T
        backward = tokens * hv * (4 * CHUNK * dv + 4 * CHUNK * dk + 12 * dk * dv)
        return {"bytes": 2 * (rows + out) + 4 * states, "flops": forward + backward}
    if c["op"] == "quantize":
        size = 4 if c["dtype"] == "fp32" else 2
        m, n = (c["cols"], c["rows"]) if c["transpose"] else (c["rows"], c["cols"])
        return {"bytes": m * n * (size + 1) + 4 * -(-m // c["block"]) * -(-n // 128), "flops": 2 * m * n}
    m, n, k = c["m"], c["n"], c["k"]
    if c["op"] == "matmul":
        size = 4 if c["out"] == "fp32" else 2
        scales = 4 * -(-k // 128) * (m + -(-n // c["b_block"]))
        return {"bytes": (m + n) * k + scales + m * n * size, "flops": 2 * m * n * k}
    size = 4 if c["dtype"] == "fp32" else 2
    return {"bytes": size * 2 * (m * k + n * k + m * n), "flops": 6 * m * n * k}


# ---------------------------------------------------------------------------
# From the definitions, in 64 bits
# ---------------------------------------------------------------------------

def _exact_tokens(q, k, v, g, beta, s0, scale, do=None, ds=None):
    """Token by token, [N, T, HV, D] in float64; with `do` and `ds`, the gradients by the recurrence run backward from
    states kept every 64 tokens."""
    t_all = q.shape[1]
    decay = g.exp()
    o = torch.empty_like(v)
    s, kept = s0, []

    def one(s, t):
        held = s * decay[:, t, :, None, None]
        miss = v[:, t] - torch.einsum("nhk,nhkv->nhv", k[:, t], held)
        return held, miss, held + torch.einsum("nhk,nhv->nhkv", k[:, t], beta[:, t, :, None] * miss)

    for t in range(t_all):
        if do is not None and t % 64 == 0:
            kept.append(s)
        s = one(s, t)[2]
        o[:, t] = scale * torch.einsum("nhk,nhkv->nhv", q[:, t], s)
    if do is None:
        return o, s
    dq, dk, dv, dg, dbeta = (torch.zeros_like(x) for x in (q, k, v, g, beta))
    last = s
    for part in range(len(kept) - 1, -1, -1):
        states = [kept[part]]
        for t in range(64 * part, min(64 * part + 64, t_all)):
            states.append(one(states[-1], t)[2])
        for t in range(min(64 * part + 64, t_all) - 1, 64 * part - 1, -1):
            before, after = states[t - 64 * part], states[t - 64 * part + 1]
            held, miss, _ = one(before, t)
            ds = ds + scale * q[:, t, :, :, None] * do[:, t, :, None, :]
            dq[:, t] = scale * torch.einsum("nhkv,nhv->nhk", after, do[:, t])
            b = beta[:, t, :, None]
            dd = torch.einsum("nhkv,nhk->nhv", ds, k[:, t])
            dbeta[:, t] = (dd * miss).sum(-1)
            dv[:, t] = b * dd
            dk[:, t] = torch.einsum("nhkv,nhv->nhk", ds, b * miss) - b * torch.einsum("nhkv,nhv->nhk", held, dd)
            ds = ds - k[:, t, :, :, None] * (b * dd)[:, :, None, :]
            dg[:, t] = (ds * held).sum((-1, -2))
            ds = ds * decay[:, t, :, None, None]
    return o, last, dq, dk, dv, dg, dbeta, ds


def _exact_delta(s):
    c = s["case"]
    h, hv, total = c["heads"], c["value_heads"], c["tokens"]
    q, k, v, g, beta, s0 = (s[n].detach().double() for n in ("q", "k", "v", "g", "beta", "s0"))
    head = torch.arange(hv, device=q.device) // (hv // h)
    q, k = q[:, :, head], k[:, :, head]
    do, ds = (s["do"].double(), s["ds"].double()) if c["grad"] else (None, None)
    if s["cu"] is None:
        got = _exact_tokens(q, k, v, g, beta, s0, c["dk"] ** -0.5, do, ds)
    else:
        ends = s["cu"].tolist()

        def apart(x):
            y = x.new_zeros(len(ends) - 1, s["longest"], *x.shape[2:])
            for i, (a, b) in enumerate(zip(ends, ends[1:])):
                y[i, :b - a] = x[0, a:b]
            return y

        def joined(y):
            return torch.cat([y[i, :b - a] for i, (a, b) in enumerate(zip(ends, ends[1:]))])[None]

        got = _exact_tokens(*(apart(x) for x in (q, k, v, g, beta)), s0, c["dk"] ** -0.5, None if do is None else apart(do), ds)
        states = (1, 7)
        got = tuple(x if i in states else joined(x) for i, x in enumerate(got))
    if not c["grad"]:
        return tuple(got)
    o, last, dq, dk, dv, dg, dbeta, ds0 = got
    dq, dk = (x.reshape(*x.shape[:2], h, hv // h, x.shape[-1]).sum(3) for x in (dq, dk))
    return o, last, dq, dk, dv, dg, dbeta, ds0


def _exact_step(s):
    c = s["case"]
    head = torch.arange(c["value_heads"], device="cuda") // (c["value_heads"] // c["heads"])
    pool = s["pool"].double()
    o = torch.zeros(s["v"].shape, dtype=torch.float64, device="cuda")
    rows = [i for i, slot in enumerate(s["slots"].tolist()) if slot >= 0]
    slots = s["slots"][rows].long()
    q, k, v, g, beta = (s[n][rows].double() for n in ("q", "k", "v", "g", "beta"))
    o[rows], pool[slots] = _exact_tokens(q[:, :, head], k[:, :, head], v, g, beta, pool[slots], c["dk"] ** -0.5)
    return o, pool


def _exact_round(y):
    """To the nearest value of e4m3 (three bits behind the leading one, smallest step 2^-9), ties to even."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -30))).clamp_min(-6.0) - 3.0)
    return (torch.round(y / step) * step).clamp(-FP8_MAX, FP8_MAX)


def _exact_quantize(x, block):
    x = x.double()
    m, n = x.shape
    row, col = torch.arange(m, device=x.device) // block, torch.arange(n, device=x.device) // 128
    size = (m - 1) // block + 1, (n - 1) // 128 + 1
    at = row[:, None] * size[1] + col
    top = torch.zeros(size[0] * size[1], dtype=torch.float64, device=x.device)
    top.scatter_reduce_(0, at.reshape(-1), x.abs().reshape(-1), "amax")
    scale = (top / FP8_MAX).clamp_min(2.0 ** -126).float().double()            # a float32 by definition, and so is the quotient:
    return _exact_round((x / scale[at]).float().double()), scale.reshape(size), scale[at]      # it decides the ties


def exact(case, seed):
    c = case
    s = prepare(c, seed)
    if c["op"] == "delta":
        return _exact_delta(s)
    if c["op"] == "step":
        return _exact_step(s)
    if c["op"] == "quantize":
        return _exact_quantize(s["x"].mT if c["transpose"] else s["x"], c["block"])[:2]
    if c["op"] == "matmul":
        cols = torch.arange(c["k"], device="cuda") // 128
        rows = torch.arange(c["n"], device="cuda") // c["b_block"]
        a = s["a"].double() * s["sa"].double()[:, cols]
        b = s["b"].double() * s["sb"].double()[rows][:, cols]
        return a @ b.mT
    x, w, dy = s["x"].detach(), s["w"].detach(), s["dy"]

    def held(t, block):
        values, _, scale = _exact_quantize(t, block)
        return values * scale

    return (held(x, 1) @ held(w, 128).mT, held(dy, 1) @ held(w.mT, 128).mT, held(dy.mT, 1) @ held(x.mT, 1).mT)
