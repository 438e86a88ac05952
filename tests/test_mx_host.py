"""The block-scaled entry points without a GPU: sizes, and refusals that come before any device work."""
import pytest

import lyth_b200 as lb
from tests import mxref as mx

FMTS = [lb.MX_FP8, lb.MX_FP4, lb.MX_NVFP4]
P = 4096  # a 16-byte aligned address that nothing reads: each call below is refused or has no rows
ODD = 4104
BF16, F32 = lb.NARROW_BF16, 0


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("rows,cols", [(1, 1), (128, 128), (129, 129), (5, 4101), (0, 64)])
def test_sizes(fmt, rows, cols):
    k = mx.padded(fmt, cols)
    assert lb.mx_row_bytes(fmt, cols) == (k if fmt == lb.MX_FP8 else k // 2)
    assert lb.mx_scale_bytes(fmt, rows, cols) == -(-rows // 128) * 128 * k // mx.BLOCK[fmt]


def test_unknown_format_has_no_size():
    assert lb.mx_row_bytes(3, 64) == 0 and lb.mx_scale_bytes(-1, 4, 64) == 0


def quantize(fmt=0, ty=BF16, rows=4, cols=64, x=P, ldx=64, g=1.0, codes=P, scales=P):
    return lb.lib.lyth_b200_quantize_mx(fmt, ty, rows, cols, x, ldx, g, codes, scales, None)


def dequantize(fmt=0, ty=BF16, rows=4, cols=64, codes=P, scales=P, g=1.0, out=P, ldo=64):
    return lb.lib.lyth_b200_dequantize_mx(fmt, ty, rows, cols, codes, scales, g, out, ldo, None)


def rmsnorm(fmt=0, ty=BF16, rows=4, cols=64, x=P, ldx=64, r=P, ldr=64, o=P, ldo=64, w=P, eps=1e-6, g=1.0, codes=P, scales=P):
    return lb.lib.lyth_b200_rmsnorm_mx(fmt, ty, rows, cols, x, ldx, r, ldr, o, ldo, w, eps, g, codes, scales, None)


def matmul(fmt=0, ty=BF16, m=4, n=4, cols=64, a=P, sa=P, b=P, sb=P, c=P, ldc=4):
    return lb.lib.lyth_b200_matmul_mx(fmt, ty, m, n, cols, a, sa, b, sb, 1.0, c, ldc, None)


def gemv(fmt=0, ty=BF16, m=1, n=4, cols=64, x=P, ldx=64, w=P, sw=P, y=P, ldy=4):
    return lb.lib.lyth_b200_gemv_mx(fmt, ty, m, n, cols, x, ldx, w, sw, 1.0, y, ldy, None)


@pytest.mark.parametrize("call", [quantize, dequantize, rmsnorm, matmul, gemv])
def test_unknown_format_or_type(call):
    assert call(fmt=3) == call(fmt=-1) == call(ty=3) == call(ty=-1) == lb.E_UNSUPPORTED


@pytest.mark.parametrize("call", [quantize, dequantize, rmsnorm, matmul, gemv])
def test_zero_columns(call):
    assert call(cols=0) == lb.E_INVALID


@pytest.mark.parametrize("call", [quantize, dequantize, rmsnorm])
def test_no_rows_is_no_work(call):
    assert call(rows=0) == lb.OK
    assert call(rows=0, codes=None, scales=None) == lb.OK
    assert call(rows=0, cols=0) == lb.E_INVALID


@pytest.mark.parametrize("call", [matmul, gemv])
def test_no_products_is_no_work(call):
    assert call(m=0) == call(n=0) == lb.OK


@pytest.mark.parametrize("call,names", [(quantize, ["x", "codes", "scales"]), (dequantize, ["out", "codes", "scales"]),
                                        (rmsnorm, ["x", "w", "codes", "scales"]), (matmul, ["a", "sa", "b", "sb", "c"]),
                                        (gemv, ["x", "w", "sw", "y"])])
def test_null_pointers(call, names):
    for name in names:
        assert call(**{name: None}) == lb.E_INVALID, name


@pytest.mark.parametrize("call,names", [(quantize, ["codes", "scales"]), (dequantize, ["codes", "scales"]),
                                        (rmsnorm, ["codes", "scales"]), (matmul, ["a", "sa", "b", "sb"]), (gemv, ["w", "sw"])])
def test_unaligned_codes_or_scales(call, names):
    for name in names:
        assert call(**{name: ODD}) == lb.E_UNSUPPORTED, name


@pytest.mark.parametrize("call,names", [(quantize, ["x"]), (dequantize, ["out"]), (rmsnorm, ["x", "r", "o", "w"]),
                                        (matmul, ["c"]), (gemv, ["x", "y"])])
def test_pointers_inside_an_element(call, names):
    for name in names:
        assert call(**{name: P + 1}) == lb.E_UNSUPPORTED, name
        if call is not gemv:
            assert call(ty=F32, **{name: P + 2}) == lb.E_UNSUPPORTED, name


@pytest.mark.parametrize("call,names", [(quantize, ["ldx"]), (dequantize, ["ldo"]), (rmsnorm, ["ldx", "ldr", "ldo"]),
                                        (gemv, ["ldx"])])
def test_stride_below_the_width(call, names):
    for name in names:
        assert call(**{name: 63}) == lb.E_INVALID, name


def test_output_stride_below_the_width():
    assert matmul(ldc=3) == gemv(ldy=3) == lb.E_INVALID


@pytest.mark.parametrize("call", [quantize, dequantize, rmsnorm])
def test_tensor_scales(call):
    for g in (0.0, -1.0, float("nan"), float("inf"), 2.0 ** -101, 2.0 ** 101):
        assert call(fmt=lb.MX_NVFP4, g=g) == lb.E_INVALID, g
    for fmt in (lb.MX_FP8, lb.MX_FP4):
        assert call(fmt=fmt, g=2.0) == lb.E_INVALID
    assert call(fmt=lb.MX_NVFP4, g=2.0 ** -100, rows=0) == call(fmt=lb.MX_NVFP4, g=2.0 ** 100, rows=0) == lb.OK


def test_rmsnorm_eps():
    assert rmsnorm(eps=-1e-6) == rmsnorm(eps=float("nan")) == lb.E_INVALID


def test_gemv_rows_and_type():
    assert gemv(m=lb.GEMV_MX_MAX_M + 1) == lb.E_UNSUPPORTED
    assert gemv(ty=F32) == lb.E_UNSUPPORTED


def test_sizes_past_an_index():
    assert quantize(cols=(1 << 30) + 1, ldx=1 << 31) == lb.E_INVALID
    assert quantize(rows=(1 << 40) + 1) == lb.E_INVALID
    assert matmul(m=(1 << 31) + 1) == lb.E_INVALID
    assert gemv(n=(1 << 31) + 1, ldy=1 << 32) == lb.E_INVALID


# ------------------------------------------------------------------ the wrappers' own checks
class Fake:
    """What the wrappers ask of a tensor, without a device."""

    def __init__(self, shape, dtype, stride=None, dev=0):
        self.shape, self.dtype, self.dev = tuple(shape), dtype, dev
        if stride is None:
            stride, step = [], 1
            for n in reversed(self.shape):
                stride.insert(0, step)
                step *= n
        self._stride = tuple(stride)
        self.is_cuda, self.device = dev >= 0, f"cuda:{dev}"

    def get_device(self):
        return self.dev

    def dim(self):
        return len(self.shape)

    def stride(self):
        return self._stride

    def is_contiguous(self):
        step = 1
        for n, s in zip(reversed(self.shape), reversed(self._stride)):
            if n > 1 and s != step:
                return False
            step *= n
        return True

    def numel(self):
        n = 1
        for s in self.shape:
            n *= s
        return n

    def data_ptr(self):
        return P


@pytest.fixture
def on_device0(monkeypatch):
    monkeypatch.setattr(lb, "_mx_device", lambda: 0)
    monkeypatch.setattr(lb, "_mx_current_stream", lambda dev: None)
    import torch

    monkeypatch.setattr(lb, "_mx_u8", torch.uint8)
    monkeypatch.setattr(lb, "_MX_TY", {torch.float32: 0, torch.float16: lb.NARROW_F16, torch.bfloat16: lb.NARROW_BF16})


def held(fmt, rows, cols, dev=0):
    import torch

    return (Fake((rows, lb.mx_row_bytes(fmt, cols)), torch.uint8, dev=dev),
            Fake((lb.mx_scale_bytes(fmt, rows, cols),), torch.uint8, dev=dev))


def test_wrappers_refuse_other_devices_shapes_and_types(on_device0):
    import torch

    bf = torch.bfloat16
    f = lb.MX_FP4
    ok = held(f, 4, 64)
    with pytest.raises(ValueError, match="current device"):
        lb.quantize_mx(f, Fake((4, 64), bf, dev=1), *ok)
    with pytest.raises(ValueError, match="current device"):
        lb.quantize_mx(f, Fake((4, 64), bf), *held(f, 4, 64, dev=1))
    with pytest.raises(ValueError, match="no CPU path"):
        lb.quantize_mx(f, Fake((4, 64), bf, dev=-1), *ok)
    with pytest.raises(TypeError, match="float32, float16 or bfloat16"):
        lb.quantize_mx(f, Fake((4, 64), torch.float64), *ok)
    with pytest.raises(ValueError, match="codes of 4 x 128 bytes"):
        lb.quantize_mx(f, Fake((4, 130), bf), *ok)
    with pytest.raises(ValueError, match="rows must be contiguous"):
        lb.quantize_mx(f, Fake((4, 64), bf, stride=(128, 2)), *ok)
    with pytest.raises(ValueError, match="rows overlap"):
        lb.quantize_mx(f, Fake((4, 64), bf, stride=(0, 1)), *ok)
    with pytest.raises(TypeError, match="expected torch.bfloat16"):
        lb.rmsnorm_mx(f, Fake((4, 64), bf), Fake((64,), bf), *ok, residual=Fake((4, 64), torch.float16))
    with pytest.raises(ValueError, match="residual_out: expected 4 x 64"):
        lb.rmsnorm_mx(f, Fake((4, 64), bf), Fake((64,), bf), *ok, residual_out=Fake((4, 65), bf))
    with pytest.raises(ValueError, match="weight: expected 64 values"):
        lb.rmsnorm_mx(f, Fake((4, 64), bf), Fake((63,), bf), *ok)
    b = held(f, 8, 256)
    with pytest.raises(ValueError, match="b: 8 x 128 takes codes"):
        lb.matmul_mx(f, *ok, *b, Fake((4, 8), bf))
    with pytest.raises(ValueError, match="gemv shapes"):
        lb.gemv_mx(f, Fake((2, 256), bf), *b, Fake((3, 8), bf))
    with pytest.raises(lb.LythError) as e:
        lb.gemv_mx(f, Fake((9, 256), bf), *b, Fake((9, 8), bf))
    assert e.value.status == lb.E_UNSUPPORTED


def test_wrappers_pass_no_rows_through(on_device0):
    import torch

    for fmt in FMTS:
        lb.quantize_mx(fmt, Fake((0, 64), torch.bfloat16), *held(fmt, 0, 64))
        lb.matmul_mx(fmt, *held(fmt, 0, 64), *held(fmt, 8, 64), Fake((0, 8), torch.float32))
        lb.gemv_mx(fmt, Fake((0, 64), torch.float16), *held(fmt, 8, 64), Fake((0, 8), torch.float16))


# ------------------------------------------------------------------ sizes that a 32-bit argument would cut
WIDE = (1 << 32) + 64


def refused(call, *args, **kw):
    with pytest.raises(lb.LythError) as e:
        call(*args, **kw)
    assert e.value.status == lb.E_INVALID


def wide_held(fmt, rows, cols):
    import torch

    k = mx.padded(fmt, cols)
    return (Fake((rows, k if fmt == lb.MX_FP8 else k // 2), torch.uint8), Fake((-(-rows // 128) * 128 * k // mx.BLOCK[fmt],), torch.uint8))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("cols", [WIDE, (1 << 32), (1 << 30) + 1, (1 << 33) + 1])
def test_wrappers_refuse_columns_past_the_limit(on_device0, fmt, cols):
    # no rows: a size that arrived cut would be taken as nothing to do
    import torch

    bf = torch.bfloat16
    x, ops = Fake((0, cols), bf), wide_held(fmt, 0, cols)
    refused(lb.quantize_mx, fmt, x, *ops)
    refused(lb.dequantize_mx, fmt, *ops, x)
    refused(lb.rmsnorm_mx, fmt, x, Fake((cols,), bf), *ops)
    refused(lb.matmul_mx, fmt, *ops, *wide_held(fmt, 4, cols), Fake((0, 4), bf))
    refused(lb.gemv_mx, fmt, x, *wide_held(fmt, 4, cols), Fake((0, 4), bf))


@pytest.mark.parametrize("fmt", FMTS)
def test_wrappers_refuse_rows_past_the_limit(on_device0, fmt):
    import torch

    bf = torch.bfloat16
    k = 128
    # 2^32 rows cut to 32 bits are none, which would be nothing to do
    refused(lb.matmul_mx, fmt, *wide_held(fmt, 1 << 32, k), *wide_held(fmt, 4, k), Fake((1 << 32, 4), bf))
    refused(lb.matmul_mx, fmt, *wide_held(fmt, 4, k), *wide_held(fmt, 1 << 32, k), Fake((4, 1 << 32), bf))
    refused(lb.gemv_mx, fmt, Fake((1, k), bf), *wide_held(fmt, 1 << 32, k), Fake((1, 1 << 32), bf))
    with pytest.raises(lb.LythError) as e:
        lb.gemv_mx(fmt, Fake((1 << 32, k), bf), *wide_held(fmt, 4, k), Fake((1 << 32, 4), bf))
    assert e.value.status == lb.E_UNSUPPORTED  # more rows than GEMV_MX_MAX_M, however many


@pytest.mark.parametrize("fmt", FMTS)
def test_sizes_of_what_no_call_takes(fmt):
    refused(lb.mx_row_bytes, fmt, WIDE)
    refused(lb.mx_scale_bytes, fmt, 4, WIDE)
    refused(lb.mx_empty, fmt, 4, WIDE, "cpu")
    refused(lb.mx_row_bytes, fmt, -1)
    refused(lb.mx_scale_bytes, fmt, -1, 64)
    refused(lb.mx_scale_bytes, fmt, 1 << 64, 64)


def test_a_format_past_32_bits_is_unknown(on_device0):
    import torch

    assert lb.mx_row_bytes(1 << 32, 64) == 0 and lb.mx_scale_bytes(1 << 32, 4, 64) == 0
    with pytest.raises(lb.LythError) as e:
        lb.quantize_mx(1 << 32, Fake((0, 64), torch.bfloat16), *held(lb.MX_FP8, 0, 64))
    assert e.value.status == lb.E_UNSUPPORTED


@pytest.mark.parametrize("call", [quantize, dequantize])
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("rows,cols", [(1 << 40, 1 << 30), ((1 << 38) + 1, 1 << 30), ((1 << 39) + 3, (1 << 30) - 5), (1 << 40, 1 << 20)])
def test_more_chunks_than_a_launch(call, fmt, rows, cols):
    # rows x columns of 16 whose count passes 64 bits must not come back as a few
    ld = {"ldx" if call is quantize else "ldo": cols}
    assert call(fmt=fmt, rows=rows, cols=cols, **ld) == lb.E_INVALID


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("rows,cols", [(1 << 40, 1 << 30), ((1 << 38) + 1, 1 << 30), ((1 << 12) + 1, 1 << 30)])
def test_norm_of_more_values_than_an_offset_reaches(fmt, rows, cols):
    assert rmsnorm(fmt=fmt, rows=rows, cols=cols, ldx=cols, ldr=cols, ldo=cols) == lb.E_INVALID
