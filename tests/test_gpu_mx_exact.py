"""The block-scaled operators where a rounding could be one too many or fall the wrong way: tensor scales that
are not powers of two, values next to the border between two results. References in 64 bits, where every
product of a code, a block scale and a tensor scale is exact (4 + 4 + 24 bits)."""
import numpy as np
import pytest
import torch

import lyth_b200 as lb
from tests import mxref as mx

pytestmark = pytest.mark.gpu

NV = lb.MX_NVFP4
BITS = {torch.float32: (24, -126), torch.float16: (11, -14), torch.bfloat16: (8, -126)}


def rounded(v, ty):
    """float64 values to the nearest of the type, ties to even, in one step."""
    bits, low = BITS[ty]
    e = np.maximum(np.frexp(v)[1] - 1, low)
    ulp = np.ldexp(1.0, e - (bits - 1))
    return np.rint(v / ulp) * ulp


def scales_beside_halfway(ty, count):
    """f32 tensor scales g for which some code * scale * g is next to halfway between two values of the type, so
    near that rounding it to f32 first would end on halfway."""
    rng = np.random.default_rng(11)
    g = rng.integers(1 << 23, 1 << 24, 200000) * 2.0 ** -30
    hit = np.zeros(g.shape, bool)
    for m in (9, 15, 21, 27, 33, 39, 45):  # odd parts of code * scale
        f32, once = rounded(m * g, torch.float32), rounded(m * g, ty)
        hit |= rounded(f32, ty) != once
    return g[hit][:count]


@pytest.mark.parametrize("ty", [torch.float32, torch.float16, torch.bfloat16])
def test_nvfp4_back_rounds_once(cuda, ty):
    # every code under every scale, times tensor scales at which two roundings would differ from one
    codes = np.tile(np.arange(16), (127, 4))
    scales = np.repeat(np.arange(127)[:, None], 4, 1)
    cd, sd = torch.from_numpy(mx.pack(NV, codes)).to(cuda), torch.from_numpy(mx.tile(scales)).to(cuda)
    picked = scales_beside_halfway(ty, 24) if ty != torch.float32 else np.array([])
    assert ty == torch.float32 or len(picked) >= 8
    for g in [float(v) for v in picked] + [float(np.float32(x)) for x in (0.12 / 2688, 1 / 3, 1e-4, 8.1e-31, 1.1e30)]:
        if ty == torch.float16 and g > 1:
            continue
        out = torch.empty(127, 64, dtype=ty, device=cuda)
        lb.dequantize_mx(NV, cd, sd, out, tensor_scale=g)
        want = rounded(mx.values(NV, codes, scales, g), ty)
        got = out.double().cpu().numpy()
        assert np.array_equal(got, want), (g, np.argwhere(got != want)[:4])


# ------------------------------------------------------------------ quantisation under a calibrated tensor scale
# of weights and activations (largest value / 2688), and three of no particular size
SCALES = [float(np.float32(g)) for g in (0.12 / 2688, 64 / 2688, 1 / 3, 3.7e-5, 1234.5)]


def held(fmt, codes, scales, rows, cols):
    """Integer codes (rows x k) and scale bytes (rows x blocks) of device tensors."""
    k = mx.padded(fmt, cols)
    return mx.unpack(fmt, codes.cpu().numpy()), scales.cpu().numpy()[mx.scale_at(rows, k // mx.BLOCK[fmt])].astype(np.int64)


def check_near(fmt, codes, scales, y, g, delta):
    """codes and scales are the definition's for values within a factor 1 +- delta of y: each block's scale for its
    largest value, then, under that scale, each code."""
    rows, cols = y.shape
    c, s = held(fmt, codes, scales, rows, cols)
    k, b = c.shape[1], mx.BLOCK[fmt]
    low, high = (mx.quantize(fmt, y * f, g)[1] for f in (1 - delta, 1 + delta))
    assert ((s >= low) & (s <= high)).all()
    size = np.repeat((mx.E4M3[s] if fmt == NV else np.ldexp(1.0, s - 127)) * g, b, axis=1)
    wide = np.zeros((rows, k))
    wide[:, :cols] = y
    ratio = np.where(size > 0, np.abs(wide) / np.where(size > 0, size, 1.0), 0.0)
    levels = mx.E4M3 if fmt == lb.MX_FP8 else mx.E2M1
    mag, sign = (c & 127, c >> 7) if fmt == lb.MX_FP8 else (c & 7, c >> 3)
    least, most = (mx.nearest(levels, ratio * f) for f in (1 - delta, 1 + delta))
    assert ((mag >= least) & (mag <= most)).all(), np.argwhere((mag < least) | (mag > most))[:4]
    assert (sign == np.signbit(wide)).all()


@pytest.mark.parametrize("ty", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("g", SCALES)
@pytest.mark.parametrize("rows,cols", [(3, 16), (130, 1000), (40, 4101)])
def test_nvfp4_quantize_under_a_calibrated_scale(cuda, ty, g, rows, cols):
    # top / (6 g): 1 / (6 g) rounded to f32, a product rounded to f32, 2^-23 in all. value / (scale g): scale * g and
    # the quotient rounded to f32, 2^-23 in all. Twice that covers both and their products. (No share of blocks is
    # asked to be the definition's bit for bit: at g = f32(1 / 3), 6 g = 2 (1 + 2^-25), so every 16-bit value whose
    # half lies on a border is 2^-25 off it by the definition and on it in f32.)
    rng = np.random.default_rng(rows + cols)
    top = min(g * 2688, 6e4) / 8
    x = torch.from_numpy((rng.standard_normal((rows, cols)) * top).astype(np.float32)).to(ty).to(cuda)
    codes, scales = lb.mx_empty(NV, rows, cols, cuda)
    lb.quantize_mx(NV, x, codes, scales, tensor_scale=g)
    y = x.double().cpu().numpy()
    check_near(NV, codes, scales, y, g, 2.0 ** -22)
    c, s = held(NV, codes, scales, rows, cols)
    out = torch.empty(rows, cols, device=cuda)
    lb.dequantize_mx(NV, codes, scales, out, tensor_scale=g)
    assert np.array_equal(out.double().cpu().numpy(), rounded(mx.values(NV, c, s, g)[:, :cols], torch.float32))


# ------------------------------------------------------------------ the norm: strides, gaps, a tensor scale
@pytest.mark.parametrize("fmt,g", [(lb.MX_FP8, 1.0), (lb.MX_FP4, 1.0), (NV, 1.0), (NV, SCALES[1]), (NV, SCALES[2])])
@pytest.mark.parametrize("ty", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", [(1, 64), (5, 777), (200, 1024), (3, 20001)])
@pytest.mark.parametrize("out_is", ["new", "x", "residual"])
def test_norm_of_rows_with_three_strides(cuda, fmt, g, ty, rows, cols, out_is):
    gen = torch.Generator().manual_seed(rows + cols)

    def strided(before, after, sigma):
        full = (sigma * torch.randn(rows, before + cols + after, generator=gen)).to(ty).to(cuda)
        return full, full[:, before:before + cols]

    (fx, x), (fr, r), (fo, o) = strided(0, 16, 1.0), strided(3, 6, 2.0), strided(5, 24, 1.0)
    w = (1 + 0.2 * torch.randn(cols + 3, generator=gen)).to(ty).to(cuda)[3:]
    dst_full, dst, before = {"new": (fo, o, 5), "x": (fx, x, 0), "residual": (fr, r, 3)}[out_is]
    keep = dst_full.clone()
    xd, rd, wd = (t.double().cpu().numpy() for t in (x, r, w))
    codes, scales = lb.mx_empty(fmt, rows, cols, cuda)
    lb.rmsnorm_mx(fmt, x, w, codes, scales, residual=r, residual_out=dst, eps=1e-5, tensor_scale=g)
    h = xd + rd
    got = dst.double().cpu().numpy()
    # one f32 addition and one rounding to the type, of every value by itself
    half = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[ty]
    assert (np.abs(got - h) <= np.abs(h) * (2.0 ** -24 + half * (1 + 2.0 ** -23)) + (2.0 ** -25 if ty == torch.float16 else 0.0)).all()
    assert torch.equal(dst_full[:, :before], keep[:, :before]) and torch.equal(dst_full[:, before + cols:], keep[:, before + cols:])
    # a sum of squares in a tree of fewer than 64 levels, a division, an addition, rsqrtf to 2 ulp, two products:
    # 2^-17 covers their roundings, and the quantisation's under a tensor scale
    y = h / np.sqrt((h * h).mean(1, keepdims=True) + 1e-5) * wd
    check_near(fmt, codes, scales, y, g, 2.0 ** -17)


# ------------------------------------------------------------------ what the products' sums hold
def integers(fmt, shape, rng):
    """Codes of whole numbers of either sign, and the numbers."""
    whole = np.array([v for v in (mx.E4M3 if fmt == lb.MX_FP8 else mx.E2M1) if v == np.rint(v)])
    v = rng.choice(whole, shape) * rng.choice([-1.0, 1.0], shape)
    levels = mx.E4M3 if fmt == lb.MX_FP8 else mx.E2M1
    return np.searchsorted(levels, np.abs(v)) | np.where(np.signbit(v), 0x80 if fmt == lb.MX_FP8 else 8, 0), v


@pytest.mark.parametrize("fmt", [lb.MX_FP8, lb.MX_FP4, NV])
@pytest.mark.parametrize("m,n,k", [(128, 128, 512), (100, 300, 1024), (300, 20000, 256)])
def test_whole_numbers_add_up_exactly(cuda, fmt, m, n, k):
    # sums of magnitudes below 2^24 need 24 bits and no more: any accumulation of that many bits is exact
    rng = np.random.default_rng(k)
    one = 0x38 if fmt == NV else 127
    (ca, va), (cb, vb) = integers(fmt, (m, k), rng), integers(fmt, (n, k), rng)
    dev = [torch.from_numpy(t).to(cuda) for c in (ca, cb)
           for t in (mx.pack(fmt, c), mx.tile(np.full((c.shape[0], k // mx.BLOCK[fmt]), one)))]
    assert (np.abs(va) @ np.abs(vb).T).max() < 2.0 ** 24
    out = torch.empty(m, n, device=cuda)
    lb.matmul_mx(fmt, *dev, out)
    assert np.array_equal(out.double().cpu().numpy(), va @ vb.T)


@pytest.mark.parametrize("fmt", [lb.MX_FP8, lb.MX_FP4])
@pytest.mark.parametrize("m,n", [(40, 70), (300, 20000)])
@pytest.mark.parametrize("ea,eb", [(254, 0), (0, 254), (240, 14), (254, 10), (2, 200), (190, 190), (127, 1)])
def test_product_of_scales_at_either_end(cuda, fmt, m, n, ea, eb):
    # ones under every scale: the sum is k times a power of two (190 and 190: 2^134, infinity in f32)
    k = 256
    code = np.full(k, 0x38 if fmt == lb.MX_FP8 else 2)
    dev = [torch.from_numpy(t).to(cuda) for rows, e in ((m, ea), (n, eb))
           for t in (mx.pack(fmt, np.tile(code, (rows, 1))), mx.tile(np.full((rows, k // 32), e)))]
    out = torch.empty(m, n, device=cuda)
    lb.matmul_mx(fmt, *dev, out)
    want = k * 2.0 ** (ea + eb - 254)
    assert bool((out.double() == (want if want < 2.0 ** 128 else np.inf)).all())
