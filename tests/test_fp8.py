"""Products in 8-bit floating point with block scales, against 64 bits.

The quantiser's results are its definition's bit for bit. The product's tolerance, for every element and relative to
sum |a| |b| (scales included): the tensor core adds 32 exact products to a float32 at a time, each addition off by at most
2^-23 of the sums' magnitude (cut, not rounded), K / 32 of them; a block's sum times the scales is added in float32,
another K / 128 roundings of 2^-24 and two of the scales' products: (K / 32 + K / 128 + 2) * 2^-23. The result's type adds half a
step, finfo(t).eps / 2 of the value.
"""
import math

import pytest
import torch

import metal_linalg_torch as mlt
from metal_linalg_torch import _lib

E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2
TYPES = [torch.bfloat16, torch.float16, torch.float32]
TOP = {E4M3: 448.0, E5M2: 57344.0}


def round_fp8(y, dtype):
    """float64 to the nearest value of an 8-bit type (3 or 2 bits behind the leading one, smallest normal 2^-6 or 2^-14),
    ties to even, by arithmetic."""
    bits, low = (3, -6) if dtype == E4M3 else (2, -14)
    e = torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -60))).clamp_min(low)
    step = torch.exp2(e - bits)
    return (torch.round(y / step) * step).clamp(-TOP[dtype], TOP[dtype])


def wanted(x, block_rows, dtype):
    """(values, scales, the scales spread over the values) in float64 on the CPU; the scale and the quotient are
    float32 numbers by definition."""
    x = x.detach().cpu().double()
    m, n = x.shape[-2:]
    rows, cols = torch.arange(m) // block_rows, torch.arange(n) // 128
    top = torch.zeros(*x.shape[:-2], -(-m // block_rows), -(-n // 128), dtype=torch.float64)
    for i in range(top.shape[-2]):
        for j in range(top.shape[-1]):
            top[..., i, j] = x[..., i * block_rows:(i + 1) * block_rows, 128 * j:128 * j + 128].abs().amax((-1, -2))
    scale = (top / TOP[dtype]).float().double().clamp_min(2.0 ** -126)
    full = scale[..., rows[:, None], cols]
    return round_fp8((x / full).float().double(), dtype), scale, full


def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="meta")


# ---------------------------------------------------------------------------
# Refusals and shapes (no GPU needed)
# ---------------------------------------------------------------------------

def test_meta_gives_shapes():
    v, s = mlt.quantize_fp8(meta(3, 200, 300))
    assert v.shape == (3, 200, 300) and v.dtype == E4M3 and s.shape == (3, 200, 3) and v.stride(-2) == 304
    v, s = mlt.quantize_fp8(meta(200, 300), block=(128, 128), transpose=True, dtype=E5M2)
    assert v.shape == (300, 200) and v.dtype == E5M2 and s.shape == (3, 2)
    a, sa = mlt.quantize_fp8(meta(2, 5, 256))
    b, sb = mlt.quantize_fp8(meta(7, 256), block=(128, 128))
    assert mlt.matmul_fp8(a, sa, b, sb).shape == (2, 5, 7)
    assert mlt.matmul_fp8(a, sa, b, sb, out_dtype=torch.float32).dtype == torch.float32
    assert mlt.linear_fp8(meta(2, 5, 64), meta(9, 64)).shape == (2, 5, 9)


@pytest.mark.parametrize("args, error", [
    (dict(x=meta(4)), ValueError), (dict(x=meta(4, 4, dtype=torch.float64)), TypeError), (dict(x=meta(4, 4), block=(1, 64)), ValueError),
    (dict(x=meta(4, 4), dtype=torch.float16), TypeError), (dict(x=torch.zeros(4, 4)), ValueError), (dict(x=[1.0]), TypeError),
    (dict(x=meta(4, 4).requires_grad_()), RuntimeError),
])
def test_quantize_refuses(args, error):
    with pytest.raises(error, match="quantize_fp8"):
        mlt.quantize_fp8(**args)


@pytest.mark.parametrize("change, error", [
    (dict(a=meta(5, 256)), TypeError), (dict(b=meta(7, 255, dtype=E4M3)), ValueError), (dict(a_scale=meta(5, 3, dtype=torch.float32)), ValueError),
    (dict(a_scale=meta(4, 2, dtype=torch.float32)), ValueError), (dict(a_scale=meta(5, 2)), TypeError), (dict(out_dtype=torch.float64), TypeError),
    (dict(b=meta(3, 7, 256, dtype=E4M3), b_scale=meta(3, 1, 2, dtype=torch.float32)), ValueError),
    (dict(a=torch.zeros(5, 256).to(E4M3)), ValueError), (dict(b_scale=meta(1, 2, dtype=torch.float32).requires_grad_()), RuntimeError),
])
def test_matmul_refuses(change, error):
    good = dict(a=meta(5, 256, dtype=E4M3), a_scale=meta(5, 2, dtype=torch.float32), b=meta(7, 256, dtype=E5M2),
                b_scale=meta(1, 2, dtype=torch.float32))
    mlt.matmul_fp8(**good)
    with pytest.raises(error, match="matmul_fp8"):
        mlt.matmul_fp8(**{**good, **change})


@pytest.mark.parametrize("x, w, error", [
    (meta(4, 8), meta(3, 9), ValueError), (meta(4, 8), meta(8), ValueError), (meta(4, 8, dtype=torch.float64), meta(3, 8), TypeError),
    (torch.zeros(4, 8), torch.zeros(3, 8), ValueError),
])
def test_linear_refuses(x, w, error):
    with pytest.raises(error, match="linear_fp8"):
        mlt.linear_fp8(x, w)


def test_c_entries_refuse_without_a_gpu():
    import numpy as np
    from metal_linalg_torch._fp8 import _OPERAND
    lib = _lib.lib
    host = np.zeros(4096, np.float32)
    at = (host.ctypes.data + 15) // 16 * 16
    quantize = lambda dtype=0, rows=4, cols=8, strides=(32, 8, 1), block=1, kind=3, values=at, stride=16, device=-1: lib.metal_linalg_quantize_fp8(  # noqa: E731
        at, dtype, 1, rows, cols, *strides, block, kind, values, stride, at, device)
    for bad in (dict(dtype=3), dict(kind=0), dict(block=2), dict(strides=(32, 8, 2)), dict(values=at + 4), dict(stride=24), dict(stride=0),
                dict(rows=1 << 30), dict(device=-2), {}):   # the last: host pointers
        assert quantize(**bad) == _lib.INVALID_ARGUMENT and "[quantize_fp8]" in _lib.last_error()
    assert quantize(rows=0) == _lib.OK
    operand = lambda values=at, scales=at, stride=128, across=0, kind=3, block=1: _OPERAND.pack(values, scales, stride, across, kind, block)  # noqa: E731
    matmul = lambda a=operand(), b=operand(), m=4, k=128, dtype=0: lib.metal_linalg_matmul_fp8(a, b, 1, m, 4, k, at, dtype, -1)  # noqa: E731
    for bad in (dict(dtype=3), dict(m=1 << 30), {}):
        assert matmul(**bad) == _lib.INVALID_ARGUMENT and "[matmul_fp8]" in _lib.last_error()
    assert lib.metal_linalg_matmul_fp8(None, operand(), 1, 4, 4, 128, at, 0, -1) == _lib.INVALID_ARGUMENT
    assert matmul(m=0) == _lib.OK
    with mlt.CpuOnly():
        assert matmul() == _lib.RUNTIME_ERROR and quantize() == _lib.RUNTIME_ERROR


def layouts(device):
    """Matrices with a row or a column of one whose strides are both other than 1, in two to five dimensions."""
    f = lambda *s: torch.arange(math.prod(s), dtype=torch.float32, device=device).reshape(s)  # noqa: E731
    return [f(5, 6)[:, ::2][:, :1], f(5, 6)[::2, ::3][:1], f(4, 5, 6)[..., ::2][..., :1], f(4, 5, 6)[:, :1, ::2], f(2, 3, 5, 4, 2)[..., :1, 0],
            f(2, 3, 5, 7)[..., ::8], f(2, 3, 1, 8)[..., ::2], f(2, 3, 5, 8)[:, :, :1, ::2], f(2, 3, 2, 5, 6)[..., ::2][..., :1],
            f(3, 2, 4, 6).transpose(0, 1)[..., ::2][..., :1], f(3, 2, 4, 6).transpose(0, 1)[..., :1, ::3], f(2, 3, 4, 6)[..., ::2],
            f(2, 3, 4, 6)[..., ::2, ::3], f(1, 1).expand(4, 7), f(2, 1, 1, 1).expand(2, 3, 4, 7), f(2, 1, 4, 1).expand(2, 3, 4, 7),
            f(2, 3, 4, 1)[:, :, ::2], f(1, 2, 1, 1)]


@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("which", range(18))
def test_quantize_hands_on_strides_that_read_the_matrix(which, transpose, monkeypatch):
    """What the C entry is given, read back with numpy: one stride is 1, and the values are x's."""
    import types

    import numpy as np
    from metal_linalg_torch import _fp8
    x = layouts("cpu")[which]
    seen = []

    def entry(at, dtype, batch, rows, cols, *rest):
        import ctypes
        across, down, along = rest[:3]
        assert down == 1 or along == 1
        reach = (batch - 1) * across + (rows - 1) * down + (cols - 1) * along + 1
        flat = np.ctypeslib.as_array(ctypes.cast(at, ctypes.POINTER(ctypes.c_float)), (reach,))
        seen.append(np.lib.stride_tricks.as_strided(flat, (batch, rows, cols), tuple(4 * s for s in (across, down, along))).copy())
        return _lib.OK

    monkeypatch.setattr(_lib, "lib", types.SimpleNamespace(metal_linalg_quantize_fp8=entry))
    monkeypatch.setattr(_lib, "use_stream_of", lambda x: 0)
    values, scales = _fp8._quantize(x, 1, transpose, E4M3)
    want = x.mT if transpose else x
    assert values.shape == want.shape and scales.shape == (*want.shape[:-1], -(-want.shape[-1] // 128))
    assert np.array_equal(seen[0], want.reshape(-1, *want.shape[-2:]).numpy())


# ---------------------------------------------------------------------------
# The quantiser
# ---------------------------------------------------------------------------

def same(got, want, what):
    got = got.cpu().double()
    assert torch.equal(got.isnan(), want.isnan()), what
    there = ~want.isnan()
    assert torch.equal(got[there], want[there]), f"{what}: {(got[there] != want[there]).sum().item()} differ"


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [E4M3, E5M2])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("block", [1, 128])
@pytest.mark.parametrize("shape", [(1, 1), (1, 128), (128, 128), (3, 129), (130, 7), (257, 200), (2, 136, 264), (2, 3, 33, 40)])
def test_quantize(shape, block, transpose, dtype, kind):
    torch.manual_seed(sum(shape))
    x = (torch.randn(shape, device="cuda") * torch.exp(3 * torch.randn(*shape[:-1], 1, device="cuda"))).to(dtype)
    values, scales = mlt.quantize_fp8(x, block=(block, 128), transpose=transpose, dtype=kind)
    v, s, _ = wanted(x.mT if transpose else x, block, kind)
    assert values.dtype == kind and values.stride(-2) % 16 == 0
    same(scales, s, "scales")
    same(values.float(), v, "values")


@pytest.mark.gpu
@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("block", [1, 128])
def test_quantize_what_is_not_ordinary(block, transpose):
    x = torch.randn(300, 300, device="cuda")
    x[0, :128] = 0                          # zeros
    x[5, 3] = math.nan
    x[6, 200] = math.inf
    x[140] *= 1e-42                         # below the smallest normal float32
    x[141] = 3e38
    x[142] = -0.0
    if transpose:
        x = x.mT.contiguous()
    values, scales = mlt.quantize_fp8(x, block=(block, 128), transpose=transpose)
    v, s, full = wanted(x.mT if transpose else x, block, E4M3)
    same(scales, s, "scales")
    # a block with an infinity: the scale is infinite and a value 0 or NaN, NaN either way once multiplied
    assert (values.cpu().double() * full)[6, 128:256].isnan().all() and (values.cpu().double() * full)[5, :128].isnan().all()
    there = full.isfinite()
    same(values.float().cpu()[there], v[there], "values")


@pytest.mark.gpu
def test_quantize_strides():
    base = torch.randn(4, 70, 3, 200, device="cuda", dtype=torch.bfloat16)
    for x in (base[:, :, 1], base[:, 1:, 0, 3:], base.transpose(1, 3)[1], base[..., ::2], base[:1].expand(5, -1, -1, -1)[:, :, 0],
              base[0, :, 0, :1], base[0, :1, 0].mT, base[:, :0, 0], base[1, 0].mT):
        for block in (1, 128):
            got, want = (mlt.quantize_fp8(y, block=(block, 128)) for y in (x, x.contiguous()))
            assert torch.equal(got[0].float(), want[0].float()) and torch.equal(got[1], want[1])
            got, want = mlt.quantize_fp8(x, block=(block, 128), transpose=True), mlt.quantize_fp8(x.mT.contiguous(), block=(block, 128))
            assert torch.equal(got[0].float(), want[0].float()) and torch.equal(got[1], want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("block", [1, 128])
def test_quantize_rows_and_columns_of_one(block, transpose):
    for x in layouts("cuda"):
        values, scales = mlt.quantize_fp8(x, block=(block, 128), transpose=transpose)
        v, s, _ = wanted(x.mT if transpose else x, block, E4M3)
        same(scales, s, "scales")
        same(values.float(), v, "values")


@pytest.mark.gpu
@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("block", [1, 128])
def test_quantize_more_matrices_than_a_grid_has_rows(block, transpose):
    """Each as if it were alone; the last ones, behind the 65535th, and those on either side of it."""
    torch.manual_seed(block)
    x = torch.randn(70000, 3, 20, device="cuda").bfloat16()
    values, scales = mlt.quantize_fp8(x, block=(block, 128), transpose=transpose)
    for part in (slice(0, 3), slice(65533, 65538), slice(69990, 70000)):
        v, s = mlt.quantize_fp8(x[part], block=(block, 128), transpose=transpose)
        assert torch.equal(values[part].float(), v.float()) and torch.equal(scales[part], s)
    if not transpose:
        v, s = mlt.quantize_fp8(x.reshape(-1, 20))          # a scale a row: the matrices' rows behind one another
        assert block != 1 or (torch.equal(values.reshape(-1, 20).float(), v.float()) and torch.equal(scales.reshape(-1, 1), s))
    a = mlt.matmul_fp8(values, scales, values[0], scales[0], out_dtype=torch.float32)
    one = mlt.matmul_fp8(values[-1:], scales[-1:], values[0], scales[0], out_dtype=torch.float32)
    assert torch.equal(a[-1:], one)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [E4M3, E5M2])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("block", [1, 128])
def test_quantize_bytes(block, transpose, dtype, kind):
    """Byte for byte: zeros of both signs, and values of both signs that round to zero, among ordinary ones."""
    torch.manual_seed(8)
    x = torch.randn(260, 300, device="cuda")
    x[::3, ::5] = 0.0
    x[1::3, ::4] = -0.0
    x[2::3, 1::7] = -1e-9
    x[::7, 2::9] = 1e-9
    x = x.to(dtype)
    values, _ = mlt.quantize_fp8(x, block=(block, 128), transpose=transpose, dtype=kind)
    want = wanted(x.mT if transpose else x, block, kind)[0].float().to(kind)
    assert (want.view(torch.uint8) == 0x80).sum() > 3000
    assert torch.equal(values.contiguous().view(torch.uint8).cpu(), want.view(torch.uint8))


# ---------------------------------------------------------------------------
# The product
# ---------------------------------------------------------------------------

def operand(rows, k, block, kind, seed, lead=()):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    wide = -(-k // 16) * 16
    values = (torch.randn(*lead, rows, wide, device="cuda", generator=gen) * TOP[kind] / 5).clamp(-TOP[kind], TOP[kind]).to(kind)[..., :k]
    scales = torch.exp(torch.randn(*lead, -(-rows // block), -(-k // 128), device="cuda", generator=gen)) / TOP[kind]
    return values, scales


def spread(values, scales):
    """The operand's values in float64."""
    m, k = values.shape[-2:]
    block = 1 if scales.shape[-2] == m else 128
    rows, cols = torch.arange(m, device="cuda") // block, torch.arange(k, device="cuda") // 128
    return values.double() * scales.double()[..., rows[:, None], cols]


def check_product(c, a, b, k):
    """a, b: spread operands."""
    want, size = a @ b.mT, a.abs() @ b.abs().mT
    short = torch.finfo(c.dtype).eps / 2
    allowed = short * want.abs() + (k / 32 + k / 128 + 2) * 2.0 ** -23 * size * (1 + short)
    over = ((c.double() - want).abs() - allowed).max().item()
    assert over <= 0, f"{over:.3g} over the bound"


SIZES = [
    # m, n, k: every tile width, shares of k, ragged edges, single rows and columns
    (1, 1, 1), (1, 128, 128), (16, 256, 1024), (3, 1000, 300), (17, 129, 128), (33, 640, 4096), (64, 4096, 512), (65, 65, 65),
    (128, 128, 128), (100, 200, 2000), (300, 77, 515), (1000, 16, 256), (257, 1, 129), (512, 512, 1024), (1000, 3001, 777), (2111, 2500, 384),
]


@pytest.mark.gpu
@pytest.mark.parametrize("blocks", [(1, 128), (1, 1), (128, 128), (128, 1)])
@pytest.mark.parametrize("size", SIZES)
def test_matmul(size, blocks):
    m, n, k = size
    a, sa = operand(m, k, blocks[0], E4M3, 1)
    b, sb = operand(n, k, blocks[1], E4M3, 2)
    for dtype in TYPES:
        check_product(mlt.matmul_fp8(a, sa, b, sb, out_dtype=dtype), spread(a, sa), spread(b, sb), k)


@pytest.mark.gpu
@pytest.mark.parametrize("kinds", [(E4M3, E5M2), (E5M2, E4M3), (E5M2, E5M2)])
@pytest.mark.parametrize("size", [(5, 300, 600), (300, 400, 256)])
def test_matmul_types(size, kinds):
    m, n, k = size
    a, sa = operand(m, k, 1, kinds[0], 3)
    b, sb = operand(n, k, 128, kinds[1], 4)
    check_product(mlt.matmul_fp8(a, sa, b, sb, out_dtype=torch.float32), spread(a, sa), spread(b, sb), k)


@pytest.mark.gpu
@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("size", [(4, 200, 256), (150, 130, 300), (1, 64, 64)])
def test_matmul_batches(size, shared):
    m, n, k = size
    a, sa = operand(m, k, 1, E4M3, 5, (2, 3))
    b, sb = operand(n, k, 128, E4M3, 6, () if shared else (2, 3))
    c = mlt.matmul_fp8(a, sa, b, sb, out_dtype=torch.float32)
    assert c.shape == (2, 3, m, n)
    check_product(c, spread(a, sa), spread(b, sb), k)
    one = mlt.matmul_fp8(a[1, 2], sa[1, 2], b if shared else b[1, 2], sb if shared else sb[1, 2], out_dtype=torch.float32)
    check_product(one, spread(a, sa)[1, 2], spread(b, sb) if shared else spread(b, sb)[1, 2], k)


@pytest.mark.gpu
def test_matmul_strides_and_nothing():
    a, sa = operand(50, 200, 1, E4M3, 7)
    b, sb = operand(60, 200, 1, E4M3, 8)
    want = mlt.matmul_fp8(a, sa, b, sb)
    for x in (a.contiguous(), a.mT.contiguous().mT, torch.cat([a.float(), a.float()], 1).to(E4M3)[:, 200:]):
        assert torch.equal(mlt.matmul_fp8(x, sa.mT.contiguous().mT, b, sb), want)
    assert mlt.matmul_fp8(a[:0], sa[:0], b, sb).shape == (0, 60)
    assert not mlt.matmul_fp8(a[:, :0], sa[:, :0], b[:, :0], sb[:, :0]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(7, 300, 1000), (300, 300, 300)])
def test_matmul_what_is_not_finite_stays_in_its_row(size):
    m, n, k = size
    a, sa = operand(m, k, 1, E4M3, 9)
    b, sb = operand(n, k, 1, E4M3, 10)
    clean = mlt.matmul_fp8(a, sa, b, sb)
    a = a.float()
    a[2, 1] = math.nan
    sa[4, 0] = math.inf
    c = mlt.matmul_fp8(a.to(E4M3), sa, b, sb)
    rest = [i for i in range(m) if i not in (2, 4)]
    assert c[2].isnan().all() and not c[4].isfinite().any() and torch.equal(c[rest], clean[rest])


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(16, 4096, 8192), (700, 700, 700), (2900, 4000, 512)])
def test_matmul_gives_the_same_bits_twice(size):
    m, n, k = size
    a, sa = operand(m, k, 1, E4M3, 11)
    b, sb = operand(n, k, 128, E4M3, 12)
    want = mlt.matmul_fp8(a, sa, b, sb)
    for _ in range(3):
        assert torch.equal(mlt.matmul_fp8(a, sa, b, sb), want)
    check_product(want, spread(a, sa), spread(b, sb), k)
    _lib.synchronize()                      # no wait ran out


# ---------------------------------------------------------------------------
# The linear map
# ---------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("types", [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32), (torch.float16, torch.float32)])
@pytest.mark.parametrize("shape", [((1, 16), 16), ((130, 100), 60), ((2, 70, 256), 300)])
def test_linear(shape, types):
    lead, n = shape
    torch.manual_seed(n)
    x = torch.randn(lead, device="cuda").to(types[0]).requires_grad_()
    w = torch.randn(n, lead[-1], device="cuda").to(types[1]).requires_grad_()
    y = mlt.linear_fp8(x, w)
    dy = torch.randn(*lead[:-1], n, device="cuda").to(types[0])
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert y.shape == dy.shape and dx.dtype == types[0] and dw.dtype == types[1]
    flat, d = x.detach().reshape(-1, lead[-1]), dy.reshape(-1, n)

    def held(t, block):
        values, _, full = wanted(t, block, E4M3)
        return (values * full).cuda()

    check_product(y.detach().reshape(-1, n), held(flat, 1), held(w, 128), lead[-1])
    check_product(dx.reshape(-1, lead[-1]), held(d, 1), held(w.mT, 128), n)
    check_product(dw, held(d.mT, 1), held(flat.mT, 1), flat.shape[0])
    with torch.no_grad():
        assert torch.equal(mlt.linear_fp8(x, w), y)


@pytest.mark.gpu
def test_linear_gradient_by_differences():
    """The map is piecewise linear in what it multiplies: with operands that 8 bits hold exactly (small whole numbers, each
    block's largest a power of two times 448) its differences along such steps are the gradient itself."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    whole = lambda *s: torch.randint(-4, 5, s, device="cuda", generator=gen).float() * 4  # noqa: E731
    x, w, dy = whole(40, 128), whole(24, 128), whole(40, 24)
    for t in (x, w, dy):
        t[:, 0] = 448.0                     # the scale is 1 in every block of every direction
        t[0, :] = 448.0
    x.requires_grad_()
    w.requires_grad_()
    y = mlt.linear_fp8(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    step = 4.0
    for leaf, grad, where in ((x, dx, (5, 7)), (x, dx, (39, 100)), (w, dw, (3, 9)), (w, dw, (23, 127))):
        up, down = leaf.detach().clone(), leaf.detach().clone()
        up[where], down[where] = 4.0, -4.0
        f = lambda t: (mlt.linear_fp8(*((t, w.detach()) if leaf is x else (x.detach(), t))).double() * dy.double()).sum()  # noqa: E731
        assert (f(up) - f(down)).item() / (2 * step) == grad[where].item()


@pytest.mark.gpu
def test_linear_of_nothing():
    for rows, n, k in ((0, 5, 16), (3, 0, 16), (3, 5, 0)):
        x = torch.randn(rows, k, device="cuda").requires_grad_()
        w = torch.randn(n, k, device="cuda").requires_grad_()
        y = mlt.linear_fp8(x, w)
        dx, dw = torch.autograd.grad(y, (x, w), torch.ones_like(y))
        assert y.shape == (rows, n) and not y.any() and dx.shape == x.shape and dw.shape == w.shape
        assert not dx.any() and not dw.any()


@pytest.mark.gpu
def test_a_mixing_layer_as_it_is_used():
    """Projections in 8 bits, the gated delta rule over a ragged batch of prompts, the projection back, with gradients; then
    the next token of every sequence from the final states. Against the same layer with the operators' own definitions."""
    from test_delta import recurrence
    torch.manual_seed(5)
    d, h, hv, dk, dv = 128, 2, 4, 32, 32
    lens = [70, 1, 130]
    cu = torch.tensor([0] + lens).cumsum(0)
    total = int(cu[-1])
    x = (torch.randn(total + 3, d, device="cuda") * 0.5).requires_grad_()
    w_in = (torch.randn(2 * h * dk + hv * dv + 2 * hv, d, device="cuda") / math.sqrt(d)).requires_grad_()
    w_out = (torch.randn(d, hv * dv, device="cuda") / math.sqrt(hv * dv)).requires_grad_()

    def layer(x, linear, mix):
        y = linear(x, w_in)
        q, k, v, g, beta = y.split([h * dk, h * dk, hv * dv, hv, hv], -1)
        unit = lambda t: torch.nn.functional.normalize(t.reshape(-1, h, dk), dim=-1)  # noqa: E731
        o, s = mix(unit(q), unit(k), v.reshape(-1, hv, dv), -torch.nn.functional.softplus(g), torch.sigmoid(beta))
        return linear(o.reshape(-1, hv * dv), w_out), s

    def operators(q, k, v, g, beta):
        o, s = mlt.gated_delta_rule(*(t[None] for t in (q, k, v, g, beta)), cu_seqlens=cu.cuda())
        return o[0], s

    def definitions(q, k, v, g, beta):
        outs, states = [], []
        for a, b in zip(cu.tolist(), cu.tolist()[1:]):
            o, s = recurrence(*(t[None, a:b] for t in (q, k, v, g, beta)), torch.zeros(1, hv, dk, dv))
            outs.append(o[0])
            states.append(s)
        return torch.cat(outs).float().cuda(), torch.cat(states).float().cuda()

    y, s = layer(x[:total], mlt.linear_fp8, operators)
    grads = torch.autograd.grad((y, s), (x, w_in, w_out), (torch.ones_like(y), torch.ones_like(s)), retain_graph=True)
    want_y, want_s = layer(x[:total], mlt.linear_fp8, definitions)
    want = torch.autograd.grad((want_y, want_s), (x, w_in, w_out), (torch.ones_like(want_y), torch.ones_like(want_s)))
    # both sides quantise the same numbers but for their last bits; a value next to a rounding border of e4m3 then moves by a
    # whole step, 2^-3 of it at most: among the up to 2^14 values of a quantised operand a few do, (few * 2^-6 / 2^14)^1/2 < 2^-8
    for a, b in zip((y, s, *grads), (want_y, want_s, *want)):
        assert (a - b).norm() <= 2.0 ** -8 * b.norm()

    with torch.no_grad():
        pool = s.detach().clone()
        nxt, _ = layer(x[total:], mlt.linear_fp8, lambda q, k, v, g, beta: (
            mlt.gated_delta_step(*(t[:, None] for t in (q, k, v, g, beta)), pool)[:, 0], pool))
        after = [None]

        def one(q, k, v, g, beta):
            o, after[0] = recurrence(*(t[:, None] for t in (q, k, v, g, beta)), s)
            return o[:, 0].float().cuda(), after[0]

        want_next, _ = layer(x[total:], mlt.linear_fp8, one)
    assert (nxt - want_next).norm() <= 2.0 ** -8 * want_next.norm()
    assert (pool.double().cpu() - after[0]).norm() <= 2.0 ** -18 * after[0].norm()


@pytest.mark.gpu
def test_streams_and_graphs():
    x, w = torch.randn(200, 256, device="cuda").bfloat16(), torch.randn(130, 256, device="cuda").bfloat16()
    want = mlt.linear_fp8(x, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = mlt.linear_fp8(x, w)
        leaf = x.detach().requires_grad_()
        graph = torch.cuda.CUDAGraph()
        torch.autograd.grad(mlt.linear_fp8(leaf, w), leaf, torch.ones_like(want))
        with torch.cuda.graph(graph, stream=side):
            y = mlt.linear_fp8(leaf, w)
            (dx,) = torch.autograd.grad(y, leaf, torch.ones_like(y))
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    with torch.no_grad():
        leaf.mul_(2.0)                      # a power of two: scales double, values stay
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, 2 * want)
    assert torch.equal(dx, torch.autograd.grad(mlt.linear_fp8(leaf, w), leaf, torch.ones_like(want))[0])


@pytest.mark.gpu
def test_compiled():
    x, w = torch.randn(70, 64, device="cuda"), torch.randn(30, 64, device="cuda")
    leaves = [t.detach().requires_grad_() for t in (x, w)]
    y = torch.compile(lambda a, b: mlt.linear_fp8(a, b) * 2, backend="aot_eager", fullgraph=True)(*leaves)
    assert torch.equal(y, mlt.linear_fp8(x, w) * 2)
    grads = torch.autograd.grad(y, leaves, torch.ones_like(y))
    plain = torch.autograd.grad(mlt.linear_fp8(*leaves) * 2, leaves, torch.ones_like(y))
    assert all(torch.equal(a, b) for a, b in zip(grads, plain))

    def product(a, b):
        return mlt.matmul_fp8(*mlt.quantize_fp8(a), *mlt.quantize_fp8(b, block=(128, 128)))

    assert torch.equal(torch.compile(product, backend="aot_eager", fullgraph=True)(x, w), product(x, w))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [5, 200, 1100])
def test_a_call_sees_what_the_one_before_it_wrote(rows):
    """Kernels start ahead of the end of those before them: a chain of maps through the same few buffers, values, scales and
    inputs written by one call and read by the next, is what the same chain gives with a wait behind every call."""
    torch.manual_seed(rows)
    w = [torch.randn(256, 256, device="cuda").bfloat16() / 16 for _ in range(3)]
    first = torch.randn(rows, 256, device="cuda").bfloat16()

    def chain(wait):
        outs, x = [], first
        for i in range(60):
            a, sa = mlt.quantize_fp8(x)
            wait()
            b, sb = mlt.quantize_fp8(w[i % 3], block=(1 if i % 2 else 128, 128))
            wait()
            x = mlt.matmul_fp8(a, sa, b, sb)
            wait()
            outs.append(x.clone())
        return outs

    want = chain(torch.cuda.synchronize)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(chain(lambda: None), want))


@pytest.mark.gpu
@pytest.mark.parametrize("blocks", [(1, 128), (1, 1)])
@pytest.mark.parametrize("size", [(16, 300, 4096), (33, 200, 1024), (100, 128, 4096), (300, 200, 128), (2304, 2300, 300), (4000, 4000, 256)])
def test_a_product_that_gives_up_surfaces(size, blocks):
    """Products that share a tile's k (their clusters exchange NaN) and that do not, one tile a block and several. The failure is
    made on the host: the kernel starts as if its waits had run out, issues no copy and no product. No GPU waits or faults."""
    m, n, k = size
    a, sa = operand(m, k, blocks[0], E4M3, 13)
    b, sb = operand(n, k, blocks[1], E4M3, 14)
    want = mlt.matmul_fp8(a, sa, b, sb)
    _lib.synchronize()
    _lib.lib.metal_linalg_inject_wait_failures(1)
    assert mlt.matmul_fp8(a, sa, b, sb).isnan().all()
    with pytest.raises(RuntimeError, match=r"gave up on a bounded wait \(a copy or a tensor-core product in 8-bit floating point\); the tiles"):
        _lib.synchronize()
    _lib.synchronize()                      # reported once
    assert torch.equal(mlt.matmul_fp8(a, sa, b, sb), want)
    _lib.synchronize()


@pytest.mark.gpu
def test_failures_of_several_kinds_are_all_named():
    import os
    a, sa = operand(100, 256, 1, E4M3, 15)
    x = torch.randn(600, 600, device="cuda")
    mlt.matmul_fp8(a, sa, a, sa)
    os.environ["QR_KERNEL"] = "blocked"
    try:
        mlt.qr(x)
        _lib.synchronize()
        _lib.lib.metal_linalg_inject_wait_failures(2)
        assert mlt.qr(x)[1].isnan().all() and mlt.matmul_fp8(a, sa, a, sa).isnan().all()
    finally:
        os.environ.pop("QR_KERNEL")
        _lib.lib.metal_linalg_inject_wait_failures(0)
    with pytest.raises(RuntimeError) as failed:
        _lib.synchronize()
    for part in ("blocked QR", "8-bit floating point", "600 x 600", "tiles concerned"):
        assert part in str(failed.value)
    _lib.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("block", [1, 128])
def test_quantize_past_32_bits(block):
    """Matrices of more than 2^31 elements, straight and transposed: their last rows as if they were alone."""
    x = torch.empty(70000, 33000, device="cuda", dtype=torch.bfloat16)
    x[-300:] = torch.randn(300, 33000, device="cuda").bfloat16()
    rows = 70000 % 128 + 128                    # whole blocks from the first row on
    x[-rows:] = torch.randn(rows, 33000, device="cuda").bfloat16()
    values, scales = mlt.quantize_fp8(x, block=(block, 128))
    v, s = mlt.quantize_fp8(x[-rows:], block=(block, 128))
    assert torch.equal(values[-rows:].view(torch.uint8), v.view(torch.uint8)) and torch.equal(scales[-s.shape[0]:], s)
    del values, scales
    values, scales = mlt.quantize_fp8(x, block=(block, 128), transpose=True)
    v, s = mlt.quantize_fp8(x[-rows:], block=(block, 128), transpose=True)
    assert torch.equal(values[:, -rows:].contiguous().view(torch.uint8), v.contiguous().view(torch.uint8))
    assert torch.equal(scales[:, -s.shape[1]:], s)


@pytest.mark.gpu
def test_matmul_past_32_bits():
    """A product of more than 2^31 elements, and operands of more than 2^31 bytes: their last rows as if they were alone (the
    same tiles, so the same bits)."""
    a, sa = operand(47104, 100, 1, E4M3, 16)
    b, sb = operand(47104, 100, 128, E4M3, 17)
    c = mlt.matmul_fp8(a, sa, b, sb)
    check_product(c[-200:, -500:], spread(a, sa)[-200:], spread(b, sb)[-500:], 100)
    check_product(c[:100, -500:], spread(a, sa)[:100], spread(b, sb)[-500:], 100)
    del c
    a = torch.zeros(270000, 8192, device="cuda", dtype=torch.uint8).view(E4M3)
    one, s_one = operand(256, 8192, 1, E4M3, 18)
    a[-256:] = one
    sa = torch.ones(270000, 64, device="cuda")
    sa[-256:] = s_one
    b, sb = operand(64, 8192, 128, E4M3, 19)
    c = mlt.matmul_fp8(a, sa, b, sb, out_dtype=torch.float32)
    check_product(c[-256:], spread(one, s_one), spread(b, sb), 8192)
    assert not c[:-256].any()
