"""The block-scaled formats on the device against tests/mxref.py (64 bits, from the definition):
quantisation and the way back bit for bit, the norm, the tensor-core product and the few-row product
within tolerances that count their roundings."""
import numpy as np
import pytest
import torch

import lyth_b200 as lb
from tests import mxref as mx

pytestmark = pytest.mark.gpu

FMTS = [lb.MX_FP8, lb.MX_FP4, lb.MX_NVFP4]
TYPES = [torch.float32, torch.float16, torch.bfloat16]
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SENTINEL = 0xA5


def empty(fmt, rows, cols, cuda):
    codes, scales = lb.mx_empty(fmt, rows, cols, cuda)
    codes.fill_(SENTINEL)
    scales.fill_(SENTINEL)
    return codes, scales


def wide(t):
    return t.double().cpu().numpy()


def check_quantized(fmt, codes, scales, want_codes, want_scales):
    rows, blocks = want_scales.shape
    assert np.array_equal(codes.cpu().numpy(), mx.pack(fmt, want_codes))
    # rows behind the last keep what they held
    assert np.array_equal(scales.cpu().numpy(), mx.tile(want_scales, SENTINEL))


def sample(rows, cols, ty, seed, cuda):
    """Normal values over many magnitudes, with exact halfway values among them."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-9, 9, (rows, 1)))
    half = rng.integers(-60, 61, (rows, cols)) / 8.0
    x = np.where(rng.random((rows, cols)) < 0.3, half, x)
    return torch.from_numpy(x.astype(np.float32)).to(cuda).to(ty)


# one value; less than a block; a scale word; odd widths; more rows than a scale tile; long rows
SHAPES = [(1, 1), (1, 31), (3, 64), (5, 129), (33, 96), (129, 200), (130, 1024), (257, 4101), (2, 20000), (700, 33)]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantize_bit_exact(cuda, fmt, ty, rows, cols):
    x = sample(rows, cols, ty, 5 + rows + cols, cuda)
    if fmt == lb.MX_NVFP4 and ty == torch.float32:
        x = x.bfloat16().float()  # f32 of more bits can lie within f32 rounding of a code's border
    codes, scales = empty(fmt, rows, cols, cuda)
    lb.quantize_mx(fmt, x, codes, scales)
    check_quantized(fmt, codes, scales, *mx.quantize(fmt, wide(x)))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("off,pad", [(0, 3), (1, 0), (8, 8), (5, 11)])
def test_quantize_strided_rows(cuda, fmt, off, pad):
    rows, cols = 70, 333
    x = sample(rows, off + cols + pad, torch.bfloat16, 9, cuda)[:, off:off + cols]
    codes, scales = empty(fmt, rows, cols, cuda)
    lb.quantize_mx(fmt, x, codes, scales)
    check_quantized(fmt, codes, scales, *mx.quantize(fmt, wide(x)))
    out = torch.full((rows, off + cols + pad), 7.0, dtype=torch.float32, device=cuda)
    lb.dequantize_mx(fmt, codes, scales, out[:, off:off + cols])
    want = mx.values(fmt, *mx.quantize(fmt, wide(x)))[:, :cols]
    assert np.array_equal(wide(out)[:, off:off + cols], want)
    assert (out[:, :off] == 7).all() and (out[:, off + cols:] == 7).all()


@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_extreme_values(cuda, fmt):
    # zeros of both signs, the smallest and largest f32, subnormals, halfway codes, infinities, NaN:
    # one kind in each block, so a bad block's neighbours keep their values
    b = mx.BLOCK[fmt]
    rng = np.random.default_rng(3)
    x = rng.standard_normal((12, 8 * b)).astype(np.float32)
    big = np.finfo(np.float32).max
    specials = [0.0, -0.0, 1e-45, -1e-45, 1.1754944e-38, big, -big, np.inf, -np.inf, np.nan, 2.0 ** -120, 3e38, 448.0, 0.75]
    for i in range(x.shape[0]):
        for j in range(0, 8, 2):
            x[i, j * b:(j + 1) * b] = x[i, j * b:(j + 1) * b] * np.float32(0.0 if (i + j) % 3 else 1e-40)
            x[i, j * b + int(rng.integers(b))] = specials[(4 * i + j // 2) % len(specials)]
    if fmt == lb.MX_NVFP4:
        x = torch.from_numpy(x).bfloat16().float().numpy()
    xd = torch.from_numpy(x).to(cuda)
    codes, scales = empty(fmt, *x.shape, cuda)
    lb.quantize_mx(fmt, xd, codes, scales)
    check_quantized(fmt, codes, scales, *mx.quantize(fmt, x.astype(np.float64)))


@pytest.mark.parametrize("g", [0.25, 2.0 ** -14, 2.0 ** 20])
def test_nvfp4_tensor_scale(cuda, g):
    # powers of two: value / (6 g) and code * scale * g are exact where the definition's are
    x = sample(40, 500, torch.bfloat16, 21, cuda)
    codes, scales = empty(lb.MX_NVFP4, 40, 500, cuda)
    lb.quantize_mx(lb.MX_NVFP4, x, codes, scales, tensor_scale=g)
    wc, ws = mx.quantize(lb.MX_NVFP4, wide(x), g)
    check_quantized(lb.MX_NVFP4, codes, scales, wc, ws)
    out = torch.empty(40, 500, device=cuda)
    lb.dequantize_mx(lb.MX_NVFP4, codes, scales, out, tensor_scale=g)
    assert np.array_equal(wide(out), mx.values(lb.MX_NVFP4, wc, ws, g)[:, :500])


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("ty", TYPES)
def test_dequantize_every_code(cuda, fmt, ty):
    # every byte of codes under every scale byte's value that the type can tell apart
    rows, k = 256, 4 * mx.BLOCK[fmt] * 2
    rng = np.random.default_rng(8)
    codes = rng.integers(0, 256 if fmt == lb.MX_FP8 else 16, (rows, k))
    scales = np.broadcast_to(np.arange(rows)[:, None], (rows, k // mx.BLOCK[fmt])).copy()
    if fmt == lb.MX_NVFP4:
        scales &= 127
    cd = torch.from_numpy(mx.pack(fmt, codes)).to(cuda)
    sd = torch.from_numpy(mx.tile(scales)).to(cuda)
    out = torch.empty(rows, k, dtype=ty, device=cuda)
    lb.dequantize_mx(fmt, cd, sd, out)
    want = mx.values(fmt, codes, scales)
    with np.errstate(over="ignore"):
        want = torch.from_numpy(want.astype(np.float32)).to(ty)  # f32 holds every finite product or its rounding
    got = out.cpu()
    same = (got == want) | (got.isnan() & want.isnan())
    assert bool(same.all())


def norm_ref(x, r, w, eps):
    h = x if r is None else x + r
    return h, h / np.sqrt((h * h).mean(1, keepdims=True) + eps) * w


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("rows,cols,residual", [(1, 4096, True), (3, 1, True), (5, 100, False), (130, 777, True), (9, 8200, True),
                                                (4, 33000, True), (2, 70001, False), (1300, 2048, True), (2600, 512, False)])
def test_rmsnorm(cuda, fmt, ty, rows, cols, residual):
    gen = torch.Generator().manual_seed(rows * 31 + cols)
    x = torch.randn(rows, cols, generator=gen).to(ty).to(cuda)
    r = (3 * torch.randn(rows, cols, generator=gen)).to(ty).to(cuda) if residual else None
    w = (1 + 0.2 * torch.randn(cols, generator=gen)).to(ty).to(cuda)
    codes, scales = empty(fmt, rows, cols, cuda)
    h = torch.full_like(x, 9.0)
    lb.rmsnorm_mx(fmt, x, w, codes, scales, residual=r, residual_out=h, eps=1e-5)
    rh, ry = norm_ref(wide(x), wide(r) if residual else None, wide(w), 1e-5)
    # h: one f32 addition, one rounding to the type
    assert np.abs(wide(h) - rh).max() <= (np.abs(rh) * (HALF_STEP[ty] * 1.001 + 2.0 ** -24)).max()
    # y before its rounding to codes is off by a few f32 roundings (the sum's tree has < 64 levels, then
    # a division, an addition, rsqrtf to 2 ulp, two products): 2^-17 covers them. Quantised that is
    # the definition's result, or a value whose code lies on the other side of a border: half a step
    # of the code (e4m3 2^-4, e2m1 at most 1 of the scale) away from y, or one more step where the
    # block's scale itself moved by one.
    got = mx.values(fmt, mx.unpack(fmt, codes.cpu().numpy()), scales.cpu().numpy()[mx.scale_at(rows, mx.padded(fmt, cols) // mx.BLOCK[fmt])])[:, :cols]
    wc, ws = mx.quantize(fmt, ry)
    want = mx.values(fmt, wc, ws)[:, :cols]
    lo, hi = (mx.values(fmt, *mx.quantize(fmt, ry * (1 + s * 2.0 ** -17)))[:, :cols] for s in (-1, 1))
    bound = np.maximum(np.maximum(lo, hi), want), np.minimum(np.minimum(lo, hi), want)
    off = (got > bound[0]) | (got < bound[1])
    # f32 inputs have no grid: a block whose scale moved at both ends is still inside the bounds
    assert not off.any(), (np.argwhere(off)[:4], got[off][:4], want[off][:4])
    assert (got != want).mean() <= 1e-2


def test_rmsnorm_in_place_and_poisoned_row(cuda):
    rows, cols, fmt = 6, 500, lb.MX_FP8
    for out_is in ("x", "residual"):
        x = sample(rows, cols, torch.bfloat16, 1, cuda)
        r = sample(rows, cols, torch.bfloat16, 2, cuda)
        w = torch.ones(cols, dtype=torch.bfloat16, device=cuda)
        x[3, 7] = float("nan")
        a, b = empty(fmt, rows, cols, cuda), empty(fmt, rows, cols, cuda)
        h = torch.empty_like(x)
        lb.rmsnorm_mx(fmt, x, w, *a, residual=r, residual_out=h)
        lb.rmsnorm_mx(fmt, x, w, *b, residual=r, residual_out=x if out_is == "x" else r)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        assert torch.equal((x if out_is == "x" else r).view(torch.int16), h.view(torch.int16))
        v = torch.empty(rows, cols, device=cuda)
        lb.dequantize_mx(fmt, *a, v)
        assert bool(v[3].isnan().all()) and bool(v[[0, 1, 2, 4, 5]].isfinite().all())


def product_bound(a, b, alpha, k, ty):
    """f32 accumulation of k exact products in any order, alpha's and the output's rounding. The
    tensor cores align a step's products and may cut instead of round (up to 2^-23 of the largest
    partial sum each step): 2 k 2^-24 of the sum of magnitudes covers a chain of k of either. Results
    below a type's smallest normal number are off by half its smallest step at most: f16 2^-25, bf16
    2^-134 (its step there is 2^-133), f32 2^-150 for each of k sums."""
    s = np.abs(a) @ np.abs(b).T * abs(alpha)
    r = np.abs(a @ b.T) * abs(alpha)
    return s * (2 * k + 4) * 2.0 ** -24 + r * (HALF_STEP[ty] + 2.0 ** -23) + {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 0.0}[ty] + k * 2.0 ** -150


MM = [(1, 1, 1), (130, 20000, 320), (2500, 1111, 256), (128, 128, 128), (5, 130, 64), (128, 128, 1024), (200, 136, 192), (257, 300, 1000), (1, 1000, 2048), (300, 515, 4160),
      (33, 16, 12288), (1024, 2056, 96)]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("m,n,k", MM)
def test_matmul(cuda, fmt, ty, m, n, k):
    rng = np.random.default_rng(m + n + k)
    a, sa, va = mx.random_operand(fmt, m, k, rng, 2)
    b, sb, vb = mx.random_operand(fmt, n, k, rng, 2)
    dev = [torch.from_numpy(t).to(cuda) for t in (a, sa, b, sb)]
    alpha = 0.75
    full = torch.full((m, n + 5), 3.0, dtype=ty, device=cuda)
    c = full[:, :n]
    lb.matmul_mx(fmt, *dev, c, alpha=alpha)
    torch.cuda.synchronize()
    assert lb.lib.lyth_b200_device_error() == 0
    want = alpha * (va @ vb.T)
    off = np.abs(wide(c) - want)
    assert (off <= product_bound(va, vb, alpha, k, ty)).all(), (off.max(), np.argwhere(off > product_bound(va, vb, alpha, k, ty))[:4])
    assert bool((full[:, n:] == 3).all())


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("ty", TYPES[1:])
@pytest.mark.parametrize("m,n,cols", [(1, 1, 1), (1, 14336, 256), (2, 100, 64), (3, 257, 1000), (4, 128, 4101), (5, 33, 192), (8, 300, 8192),
                                      (7, 1000, 777), (1, 64, 20000), (8, 16, 16384)])
def test_gemv(cuda, fmt, ty, m, n, cols):
    rng = np.random.default_rng(m + n + cols)
    w, sw, vw = mx.random_operand(fmt, n, cols, rng, 3)
    x = torch.from_numpy(rng.standard_normal((m, cols)).astype(np.float32)).to(ty)
    vx = x.double().numpy()
    y = torch.full((m, n + 3), 5.0, dtype=ty, device=cuda)
    lb.gemv_mx(fmt, x.to(cuda), torch.from_numpy(w).to(cuda), torch.from_numpy(sw).to(cuda), y[:, :n], alpha=0.5)
    want = 0.5 * (vx @ vw[:, :cols].T)
    assert (np.abs(wide(y)[:, :n] - want) <= product_bound(vx, vw[:, :cols], 0.5, cols, ty)).all()
    assert bool((y[:, n:] == 5).all())


# ------------------------------------------------------------------ values that are not numbers, and extremes
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,n", [(40, 70), (300, 20000)])  # single SMs and CTA pairs
def test_matmul_bad_and_zero_blocks_stay_in_their_rows(cuda, fmt, m, n):
    rng = np.random.default_rng(4)
    k = 512
    a, sa, va = mx.random_operand(fmt, m, k, rng, 1)
    b, sb, vb = mx.random_operand(fmt, n, k, rng, 1)
    where = mx.scale_at(max(m, n), k // mx.BLOCK[fmt])
    bad, zero = (0x7F if fmt == lb.MX_NVFP4 else 0xFF), 0
    sa[where[5, 3]] = bad          # one NaN scale: row 5 of the product, and only it
    sb[where[11, 0]] = bad         # column 11
    sa[where[7, :]] = zero         # a row of the smallest scales (NVFP4: of zeros)
    size = {lb.MX_NVFP4: 0.0}.get(fmt, 2.0 ** -127)
    va[7] = va[7] * 0 + mx.values(fmt, mx.unpack(fmt, a[7:8]), np.zeros((1, k // mx.BLOCK[fmt]), np.int64))[0]
    assert np.abs(va[7]).max() <= 448 * size
    dev = [torch.from_numpy(t).to(cuda) for t in (a, sa, b, sb)]
    c = torch.empty(m, n, device=cuda)
    lb.matmul_mx(fmt, *dev, c)
    got = wide(c)
    nan = np.zeros((m, n), bool)
    nan[5, :] = nan[:, 11] = True
    assert np.array_equal(np.isnan(got), nan)
    want = va @ vb.T
    ok = ~nan
    assert (np.abs(got - want)[ok] <= (product_bound(va, vb, 1.0, k, torch.float32) + 2.0 ** -126)[ok]).all()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("ty", TYPES[1:])
def test_gemv_tokens_do_not_touch_one_another(cuda, fmt, ty):
    # an infinity, a NaN, a huge, a tiny, a zero and a subnormal token beside ordinary ones
    m, n, k = 8, 200, 700
    rng = np.random.default_rng(6)
    w, sw, vw = mx.random_operand(fmt, n, k, rng, 2)
    x = torch.from_numpy(rng.standard_normal((m, k)).astype(np.float32))
    big, tiny = (1e30, 1e-30) if ty == torch.bfloat16 else (60.0, 1e-4)
    x[1] *= big
    x[2] *= tiny
    x[3] = 0
    x[4, 333] = float("inf")
    x[5, 17] = float("nan")
    x[6] *= 1e-39 if ty == torch.bfloat16 else 1e-7
    x = x.to(ty)
    vx = x.double().numpy()
    args = torch.from_numpy(w).to(cuda), torch.from_numpy(sw).to(cuda)
    y = torch.empty(m, n, dtype=ty, device=cuda)
    lb.gemv_mx(fmt, x.to(cuda), *args, y)
    got = wide(y)
    with np.errstate(invalid="ignore", over="ignore"):
        want = vx @ vw[:, :k].T
    assert np.array_equal(np.isnan(got[4:6]), np.isnan(want[4:6]))
    fin = np.isfinite(want)
    fin[4:6] = False
    bound = product_bound(np.where(np.isfinite(vx), vx, 0), vw[:, :k], 1.0, k, ty)
    top = torch.finfo(ty).max
    inside = fin & (np.abs(want) < top * 0.99)
    assert inside[[0, 2, 3, 6, 7]].all()
    with np.errstate(invalid="ignore"):
        off = np.abs(got - want)
    assert (off[inside] <= bound[inside]).all(), np.argwhere(inside & ~(off <= bound))[:5]
    assert (got[3] == 0).all()
    inf = ~np.isnan(want[4]) & np.isinf(want[4])
    assert np.array_equal(got[4][inf], want[4][inf])
    # each alone gives the same bits
    for i in (0, 1, 2, 7):
        one = torch.empty(1, n, dtype=ty, device=cuda)
        lb.gemv_mx(fmt, x[i:i + 1].to(cuda), *args, one)
        assert torch.equal(one[0].view(torch.int16), y[i].view(torch.int16)), i


def test_gemv_wide_range_within_a_token(cuda):
    # bf16 columns 2^20 apart, in one block and across blocks: the small ones still count
    rng = np.random.default_rng(7)
    n, k = 64, 1024
    w, sw, vw = mx.random_operand(lb.MX_FP4, n, k, rng, 0)
    x = torch.from_numpy(rng.standard_normal((1, k)).astype(np.float32))
    x[0, ::7] *= 2.0 ** 20
    x[0, 512:] *= 2.0 ** -90
    x = x.bfloat16()
    vx = x.double().numpy()
    y = torch.empty(1, n, dtype=torch.bfloat16, device=cuda)
    lb.gemv_mx(lb.MX_FP4, x.to(cuda), torch.from_numpy(w).to(cuda), torch.from_numpy(sw).to(cuda), y)
    assert (np.abs(wide(y) - vx @ vw.T) <= product_bound(vx, vw, 1.0, k, torch.bfloat16)).all()
    # only the far half of x: its own range
    x2 = torch.zeros_like(x)
    x2[0, 512:] = x[0, 512:]
    v2 = x2.double().numpy()
    lb.gemv_mx(lb.MX_FP4, x2.to(cuda), torch.from_numpy(w).to(cuda), torch.from_numpy(sw).to(cuda), y)
    assert (np.abs(wide(y) - v2 @ vw.T) <= product_bound(v2, vw, 1.0, k, torch.bfloat16)).all()


@pytest.mark.parametrize("fmt", FMTS)
def test_gemv_strided_and_unaligned_x(cuda, fmt):
    rng = np.random.default_rng(12)
    m, n, k = 3, 130, 1001
    w, sw, vw = mx.random_operand(fmt, n, k, rng, 2)
    full = torch.from_numpy(rng.standard_normal((m, k + 9)).astype(np.float32)).bfloat16().to(cuda)
    for off in (0, 1, 8):
        x = full[:, off:off + k]
        y = torch.full((m, n + 1), 2.0, dtype=torch.bfloat16, device=cuda)
        lb.gemv_mx(fmt, x, torch.from_numpy(w).to(cuda), torch.from_numpy(sw).to(cuda), y[:, 1:])
        vx = wide(x)
        assert (np.abs(wide(y)[:, 1:] - vx @ vw[:, :k].T) <= product_bound(vx, vw[:, :k], 1.0, k, torch.bfloat16)).all()
        assert bool((y[:, 0] == 2).all())


# ------------------------------------------------------------------ together, and the ways they are called
def block_ref(fmt, x, r, w_norm, weights, eps):
    """Norm, quantised; the product with quantised weights; 64 bits throughout but for the formats."""
    h, y = norm_ref(x, r, w_norm, eps)
    return h, mx.values(fmt, *mx.quantize(fmt, y)) @ weights.T


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("rows", [1, 37, 200])
def test_norm_then_projection(cuda, fmt, rows):
    # the block as it is used: residual + norm + quantise, then the projection's product on the codes, or
    # for a few rows on the unquantised activations
    k, n = 1024, 640
    rng = np.random.default_rng(30 + rows)
    gen = torch.Generator().manual_seed(rows)
    x, r = (torch.randn(rows, k, generator=gen).bfloat16().to(cuda) for _ in range(2))
    wn = (1 + 0.1 * torch.randn(k, generator=gen)).bfloat16().to(cuda)
    wf = torch.from_numpy((rng.standard_normal((n, k)) / 32).astype(np.float32)).bfloat16().to(cuda)
    wq = lb.mx_empty(fmt, n, k, cuda)
    lb.quantize_mx(fmt, wf, *wq)
    vw = mx.values(fmt, *mx.quantize(fmt, wide(wf)))
    aq = lb.mx_empty(fmt, rows, k, cuda)
    h, c = torch.empty_like(x), torch.empty(rows, n, device=cuda)
    lb.rmsnorm_mx(fmt, x, wn, *aq, residual=r, residual_out=h, eps=1e-5)
    lb.matmul_mx(fmt, *aq, *wq, c)
    _, want = block_ref(fmt, wide(x), wide(r), wide(wn), vw, 1e-5)
    # the product itself, on the codes the norm really made
    got_a = torch.empty(rows, k, device=cuda)
    lb.dequantize_mx(fmt, *aq, got_a)
    exact = wide(got_a) @ vw.T
    assert (np.abs(wide(c) - exact) <= product_bound(wide(got_a), vw, 1.0, k, torch.float32)).all()
    # and end to end: codes at a border may differ by a step (at most 1e-2 of them, test_rmsnorm), each
    # by half its value at most, so the norm of the difference is at most 0.1 * 0.5 of the whole
    assert np.linalg.norm(wide(c) - want) <= 0.05 * np.linalg.norm(want)
    if rows <= lb.GEMV_MX_MAX_M:
        a16, y = got_a.bfloat16(), torch.empty(rows, n, dtype=torch.bfloat16, device=cuda)
        lb.gemv_mx(fmt, a16, *wq, y)
        v16 = wide(a16)
        assert (np.abs(wide(y) - v16 @ vw.T) <= product_bound(v16, vw, 1.0, k, torch.bfloat16)).all()


def all_calls(fmt, s):
    lb.rmsnorm_mx(fmt, s["x"], s["wn"], *s["a"], residual=s["r"], residual_out=s["h"])
    lb.matmul_mx(fmt, *s["a"], *s["w"], s["c"])
    lb.quantize_mx(fmt, s["x"], *s["q"])
    lb.dequantize_mx(fmt, *s["q"], s["d"])
    lb.gemv_mx(fmt, s["d"], *s["w"], s["y"])


OUTPUTS = ["h", "c", "d", "y"]


def state(fmt, cuda, seed, rows=5, k=768, n=400):
    gen = torch.Generator().manual_seed(seed)
    s = {"x": torch.randn(rows, k, generator=gen).bfloat16().to(cuda), "r": torch.randn(rows, k, generator=gen).bfloat16().to(cuda),
         "wn": torch.ones(k, dtype=torch.bfloat16, device=cuda), "a": lb.mx_empty(fmt, rows, k, cuda), "q": lb.mx_empty(fmt, rows, k, cuda),
         "w": lb.mx_empty(fmt, n, k, cuda), "h": torch.empty(rows, k, dtype=torch.bfloat16, device=cuda),
         "d": torch.empty(rows, k, dtype=torch.bfloat16, device=cuda), "c": torch.empty(rows, n, device=cuda),
         "y": torch.empty(rows, n, dtype=torch.bfloat16, device=cuda)}
    lb.quantize_mx(fmt, torch.randn(n, k, generator=gen).to(cuda), *s["w"])
    return s


@pytest.mark.parametrize("fmt", FMTS)
def test_captured_and_replayed_on_new_inputs(cuda, fmt):
    s, t = state(fmt, cuda, 1), state(fmt, cuda, 2)
    all_calls(fmt, t)
    want = {o: t[o].clone() for o in OUTPUTS}
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        all_calls(fmt, s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            all_calls(fmt, s)
    torch.cuda.synchronize()
    for name in ("x", "r"):
        s[name].copy_(t[name])
    for a, b in zip(s["w"], t["w"]):
        a.copy_(b)
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    for o in OUTPUTS:
        assert torch.equal(s[o], want[o]), o


@pytest.mark.parametrize("fmt", FMTS)
def test_two_streams_and_repeats_give_the_same_bits(cuda, fmt):
    states = [state(fmt, cuda, i) for i in (3, 4)]
    want = []
    for s in states:
        all_calls(fmt, s)
        want.append({o: s[o].clone() for o in OUTPUTS})
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(10):
        for s, st in zip(states, streams):
            with torch.cuda.stream(st):
                all_calls(fmt, s)
    for s, st, w in zip(states, streams, want):
        st.synchronize()
        for o in OUTPUTS:
            assert torch.equal(s[o], w[o]), o
    # an explicit stream, as an object and as its handle
    s = states[0]
    s["c"].zero_()
    torch.cuda.synchronize()
    lb.matmul_mx(fmt, *s["a"], *s["w"], s["c"], stream=streams[0])
    streams[0].synchronize()
    assert torch.equal(s["c"], want[0]["c"])
    s["c"].zero_()
    torch.cuda.synchronize()
    lb.matmul_mx(fmt, *s["a"], *s["w"], s["c"], stream=streams[1].cuda_stream)
    streams[1].synchronize()
    assert torch.equal(s["c"], want[0]["c"])


@pytest.mark.parametrize("fmt", FMTS)
def test_no_rows_no_columns_of_the_product(cuda, fmt):
    w = state(fmt, cuda, 9)["w"]
    for m in (0,):
        lb.quantize_mx(fmt, torch.empty(m, 768, device=cuda), *lb.mx_empty(fmt, m, 768, cuda))
        lb.matmul_mx(fmt, *lb.mx_empty(fmt, m, 768, cuda), *w, torch.empty(m, 400, device=cuda))
        lb.gemv_mx(fmt, torch.empty(m, 768, dtype=torch.float16, device=cuda), *w, torch.empty(m, 400, dtype=torch.float16, device=cuda))
    lb.matmul_mx(fmt, *w, *lb.mx_empty(fmt, 0, 768, cuda), torch.empty(400, 0, device=cuda))
    torch.cuda.synchronize()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("cols", [20001, 40001, 40000])  # two chunks a thread; rows read twice, shifted and aligned
def test_rmsnorm_in_place_of_wide_rows(cuda, fmt, cols):
    w = torch.ones(cols, dtype=torch.bfloat16, device=cuda)
    for target in (0, 1):
        two = [sample(3, cols, torch.bfloat16, 5, cuda), sample(3, cols, torch.bfloat16, 6, cuda)]
        a, b = empty(fmt, 3, cols, cuda), empty(fmt, 3, cols, cuda)
        h = torch.empty_like(two[0])
        lb.rmsnorm_mx(fmt, two[0], w, *a, residual=two[1], residual_out=h)
        lb.rmsnorm_mx(fmt, two[0], w, *b, residual=two[1], residual_out=two[target])
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        assert torch.equal(two[target].view(torch.int16), h.view(torch.int16))


@pytest.mark.parametrize("fmt", FMTS)
def test_one_tensor_in_two_places(cuda, fmt):
    # x as its own residual; a matrix times itself
    x = sample(200, 320, torch.bfloat16, 12, cuda)
    w = torch.ones(320, dtype=torch.bfloat16, device=cuda)
    a, b = empty(fmt, 200, 320, cuda), empty(fmt, 200, 320, cuda)
    lb.rmsnorm_mx(fmt, x, w, *a, residual=x)
    lb.rmsnorm_mx(fmt, x * 2, w, *b)
    va, vb = torch.empty(200, 320, device=cuda), torch.empty(200, 320, device=cuda)
    lb.dequantize_mx(fmt, *a, va)
    lb.dequantize_mx(fmt, *b, vb)
    assert torch.equal(va, vb)
    c, d = torch.empty(200, 200, device=cuda), torch.empty(200, 200, device=cuda)
    lb.matmul_mx(fmt, *a, *a, c)
    lb.matmul_mx(fmt, *a, *[t.clone() for t in a], d)
    assert torch.equal(c, d)


FIRST = """
import threading
import torch
import lyth_b200 as lb

cuda = torch.device("cuda")
torch.manual_seed(0)
x = torch.randn(8, 512, device=cuda).bfloat16()
xw = torch.randn(20000, 512, device=cuda)
torch.cuda.synchronize()


def buffers():
    return {"w": lb.mx_empty(1, 20000, 512, cuda), "q": lb.mx_empty(1, 8, 512, cuda), "n": lb.mx_empty(1, 8, 512, cuda),
            "one": torch.ones(512, dtype=torch.bfloat16, device=cuda), "c": torch.empty(8, 20000, device=cuda),
            "l": torch.empty(20000, 20000, dtype=torch.bfloat16, device=cuda), "y": torch.empty(8, 20000, dtype=torch.bfloat16, device=cuda),
            "d": torch.empty(8, 512, device=cuda)}


def calls(b):
    lb.quantize_mx(1, xw, *b["w"])
    lb.quantize_mx(1, x, *b["q"])
    lb.dequantize_mx(1, *b["q"], b["d"])
    lb.rmsnorm_mx(1, x, b["one"], *b["n"])
    lb.matmul_mx(1, *b["n"], *b["w"], b["c"])
    lb.matmul_mx(1, *b["w"], *b["w"], b["l"])
    lb.gemv_mx(1, x, *b["w"], b["y"])


def same(a, b):
    return all(torch.equal(a[k], b[k]) for k in ("c", "l", "y", "d"))


MODE
print("OK")
"""
CAPTURED_FIRST = """
b, want = buffers(), buffers()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    calls(b)
g.replay()
calls(want)
torch.cuda.synchronize()
assert same(b, want)
"""
THREADS_FIRST = """
sets, failed = [buffers() for _ in range(4)], []
torch.cuda.synchronize()


def work(b):
    try:
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                calls(b)
            torch.cuda.current_stream().synchronize()
    except BaseException as e:
        failed.append(e)


threads = [threading.Thread(target=work, args=(b,)) for b in sets]
for t in threads:
    t.start()
for t in threads:
    t.join()
assert not failed, failed
want = buffers()
calls(want)
torch.cuda.synchronize()
assert all(same(b, want) for b in sets)
"""


@pytest.mark.parametrize("mode", [CAPTURED_FIRST, THREADS_FIRST], ids=["captured", "threads"])
def test_first_calls_of_a_process(cuda, mode):
    # a process whose first calls are captured, or come from four threads at once
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST.replace("MODE", mode)], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("OK"), r.stdout + r.stderr


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("m", [40, 19000])  # single SMs and CTA pairs
def test_matmul_rows_of_any_alignment(cuda, ty, m):
    # the same bits as into rows that start on 32 bytes, and nothing beside them
    fmt, k = lb.MX_FP8, 128
    gen = torch.Generator().manual_seed(m)
    a, b = empty(fmt, m, k, cuda), empty(fmt, 400, k, cuda)
    lb.quantize_mx(fmt, torch.randn(m, k, generator=gen).to(cuda), *a)
    lb.quantize_mx(fmt, torch.randn(400, k, generator=gen).to(cuda), *b)
    want = torch.empty(m, 400, dtype=ty, device=cuda)
    lb.matmul_mx(fmt, *a, *b, want)
    for i, n in enumerate([1, 2, 7, 15, 16, 17, 31, 33, 63, 64, 100, 129, 190, 193, 200, 383, 385, 399]):
        part = b[0][:n].contiguous(), b[1][:(n + 127) // 128 * 512 * (k // 128)].contiguous()
        for off, pad in ((i % 17, 1), ((5 * i + 3) % 16, (7 * i) % 16), (8, 16 - n % 16)):
            full = torch.full((m, off + n + pad), 3.0, dtype=ty, device=cuda)
            lb.matmul_mx(fmt, *a, *part, full[:, off:off + n])
            assert torch.equal(full[:, off:off + n], want[:, :n]), (n, off, pad)
            assert bool((full[:, :off] == 3).all()) and bool((full[:, off + n:] == 3).all()), (n, off, pad)


def chain(x, s, between):
    # every call reads what the one before it has just written, others' kernels and copies between them
    fmt = lb.MX_FP8
    for _ in range(3):
        lb.rmsnorm_mx(fmt, x, s["one"], *s["n"], residual=s["r"], residual_out=s["r"])
        between()
        lb.matmul_mx(fmt, *s["n"], *s["w"], s["c"], alpha=0.05)
        between()
        lb.quantize_mx(fmt, s["c"], *s["q"])
        between()
        lb.matmul_mx(fmt, *s["q"], *s["w"], s["d"], alpha=0.05)
        between()
        s["e"].copy_(s["d"])
        between()
        lb.gemv_mx(fmt, s["e"][:8], *s["w"], x[:8], alpha=0.05)
        between()
        lb.quantize_mx(fmt, x, *s["n"])
        between()
        lb.dequantize_mx(fmt, *s["n"], x)
        between()
        x.add_(s["e"])
        between()


@pytest.mark.parametrize("rows", [8, 300, 5000])
def test_a_chain_of_dependent_calls(cuda, rows):
    k = 512
    gen = torch.Generator().manual_seed(rows)
    start, r = torch.randn(rows, k, generator=gen).bfloat16().to(cuda), torch.randn(rows, k, generator=gen).bfloat16().to(cuda)
    s = {"one": torch.ones(k, dtype=torch.bfloat16, device=cuda), "n": empty(lb.MX_FP8, rows, k, cuda), "q": empty(lb.MX_FP8, rows, k, cuda),
         "w": empty(lb.MX_FP8, k, k, cuda), "c": torch.empty(rows, k, device=cuda), "d": torch.empty(rows, k, device=cuda),
         "e": torch.empty(rows, k, dtype=torch.bfloat16, device=cuda), "r": r.clone()}
    lb.quantize_mx(lb.MX_FP8, torch.randn(k, k, generator=gen).to(cuda), *s["w"])
    want = start.clone()
    chain(want, s, torch.cuda.synchronize)
    want_r = s["r"].clone()
    for _ in range(20):
        x = start.clone()
        s["r"].copy_(r)
        chain(x, s, lambda: None)
        assert torch.equal(x, want) and torch.equal(s["r"], want_r)
    # captured, with a second stream's work joined in the middle
    x, side = start.clone(), torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    y = torch.empty_like(x)
    with torch.cuda.graph(g):
        x.copy_(start)
        s["r"].copy_(r)
        chain(x, s, lambda: None)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            lb.quantize_mx(lb.MX_FP8, s["c"], *s["q"])
            y.copy_(x)
        lb.quantize_mx(lb.MX_FP8, x, *s["n"])
        torch.cuda.current_stream().wait_stream(side)
        lb.dequantize_mx(lb.MX_FP8, *s["q"], s["d"])
        lb.dequantize_mx(lb.MX_FP8, *s["n"], s["e"])
    for _ in range(5):
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(x, want) and torch.equal(y, want) and torch.equal(s["r"], want_r)
    for src, (codes, scales), got in ((s["c"], s["q"], s["d"]), (x, s["n"], s["e"])):
        again, out = empty(lb.MX_FP8, rows, k, cuda), torch.empty_like(got)
        lb.quantize_mx(lb.MX_FP8, src, *again)
        torch.cuda.synchronize()
        lb.dequantize_mx(lb.MX_FP8, *again, out)
        assert torch.equal(codes, again[0]) and torch.equal(got, out)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,n,k", [(1, 19500, 192), (100, 19001, 64), (128, 19500, 1024), (129, 19456, 320), (600, 14336, 128),
                                   (250, 14336, 320), (1000, 4100, 1000), (512, 14330, 640), (2048, 4096, 192)])
def test_matmul_tile_widths(cuda, fmt, m, n, k):
    # more 128 x 128 tiles than SMs: each width of a pair's tile, in one round and in several, rows and
    # columns of it that do not exist
    test_matmul(cuda, fmt, torch.bfloat16, m, n, k)


def test_inputs_written_on_another_stream(cuda):
    # an event of another stream between two calls of this one, eager and captured
    fmt, n, k = lb.MX_FP4, 8192, 4096
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(40, k, generator=gen).bfloat16().to(cuda)
    ws = [torch.randn(n, k, generator=gen).bfloat16().to(cuda) for _ in range(3)]
    one = torch.ones(k, dtype=torch.bfloat16, device=cuda)
    a, w = empty(fmt, 40, k, cuda), empty(fmt, n, k, cuda)
    c, y = torch.empty(40, n, dtype=torch.bfloat16, device=cuda), torch.empty(4, n, dtype=torch.bfloat16, device=cuda)
    side, src = torch.cuda.Stream(), torch.empty_like(ws[0])

    def step():
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            lb.quantize_mx(fmt, src, *w)
        lb.rmsnorm_mx(fmt, x, one, *a)
        torch.cuda.current_stream().wait_stream(side)
        lb.gemv_mx(fmt, x[:4], *w, y)
        lb.matmul_mx(fmt, *a, *w, c)

    want = []
    for t in ws:
        src.copy_(t)
        torch.cuda.synchronize()
        lb.quantize_mx(fmt, src, *w)
        lb.rmsnorm_mx(fmt, x, one, *a)
        torch.cuda.synchronize()
        lb.gemv_mx(fmt, x[:4], *w, y)
        torch.cuda.synchronize()
        lb.matmul_mx(fmt, *a, *w, c)
        torch.cuda.synchronize()
        want.append((c.clone(), y.clone()))
    main = torch.cuda.Stream()
    main.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(main):
        for i in range(30):
            src.copy_(ws[i % 3])
            step()
            got = c.clone(), y.clone()
            main.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(got, want[i % 3])), i
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=main):
            step()
        for i in range(30):
            src.copy_(ws[i % 3])
            g.replay()
            main.synchronize()
            assert torch.equal(c, want[i % 3][0]) and torch.equal(y, want[i % 3][1]), i
    torch.cuda.synchronize()
