"""The block-scaled operators where 32-bit offsets end: more than 2^32 values, codes or results. The
far rows are compared with the same rows given alone, whose results test_gpu_mx.py holds to 64 bits."""
import pytest
import torch

import lyth_b200 as lb

pytestmark = pytest.mark.gpu


def codes_of(fmt, rows, cols, cuda, seed):
    """Random finite codes and scales of a matrix too large to quantise from values."""
    gen = torch.Generator(device=cuda).manual_seed(seed)
    codes, scales = lb.mx_empty(fmt, rows, cols, cuda)
    codes.random_(0, 256, generator=gen)
    if fmt == lb.MX_FP8:
        codes &= 0xF7  # no NaN code
    scales.random_(0x30, 0x48, generator=gen) if fmt == lb.MX_NVFP4 else scales.random_(120, 132, generator=gen)
    return codes, scales


def rows_alone(fmt, codes, scales, first, count):
    """The rows `first` .. of a matrix (a multiple of 128) as a matrix of their own."""
    per = scales.numel() // (-(-codes.shape[0] // 128))
    return codes[first:first + count].contiguous(), scales[first // 128 * per:][: -(-count // 128) * per].contiguous()


@pytest.mark.parametrize("fmt", [lb.MX_FP8, lb.MX_NVFP4])
def test_quantize_past_32_bits(cuda, fmt):
    rows, cols, tail = 68000, 65536, 32  # 4.46e9 values
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device=cuda)
    gen = torch.Generator(device=cuda).manual_seed(1)
    x[-tail:].normal_(generator=gen)
    x[:tail].normal_(generator=gen)
    x[tail:-tail].fill_(1.5)
    codes, scales = lb.mx_empty(fmt, rows, cols, cuda)
    lb.quantize_mx(fmt, x, codes, scales)
    back = torch.empty_like(x)
    lb.dequantize_mx(fmt, codes, scales, back)
    for part in (slice(0, tail), slice(rows - tail, rows)):
        one = x[part].contiguous()
        c, s = lb.mx_empty(fmt, tail, cols, cuda)
        lb.quantize_mx(fmt, one, c, s)
        assert torch.equal(codes[part], c)
        d = torch.empty_like(one)
        lb.dequantize_mx(fmt, c, s, d)
        assert torch.equal(back[part], d)
    assert bool((back[rows // 2] == 1.5).all())
    del x, back


def test_rmsnorm_past_32_bits(cuda):
    rows, cols, tail = 68000, 65536, 16
    x = torch.ones(rows, cols, dtype=torch.bfloat16, device=cuda)
    x[-tail:].normal_(generator=torch.Generator(device=cuda).manual_seed(2))
    w = torch.ones(cols, dtype=torch.bfloat16, device=cuda)
    codes, scales = lb.mx_empty(lb.MX_FP4, rows, cols, cuda)
    want = lb.mx_empty(lb.MX_FP4, tail, cols, cuda)
    lb.rmsnorm_mx(lb.MX_FP4, x[-tail:].contiguous(), w, *want)
    lb.rmsnorm_mx(lb.MX_FP4, x, w, codes, scales, residual=None, residual_out=x)
    assert torch.equal(codes[-tail:], want[0])
    del x


@pytest.mark.parametrize("fmt", [lb.MX_FP8, lb.MX_FP4])
def test_gemv_weights_past_32_bits(cuda, fmt):
    n, k = (270000, 16384) if fmt == lb.MX_FP8 else (540160, 16384)  # 4.42e9 bytes of codes
    w, s = codes_of(fmt, n, k, cuda, 3)
    x = torch.randn(2, k, generator=torch.Generator().manual_seed(4)).bfloat16().to(cuda)
    y = torch.empty(2, n, dtype=torch.bfloat16, device=cuda)
    lb.gemv_mx(fmt, x, w, s, y)
    first = (n - 200) // 128 * 128
    one = torch.empty(2, n - first, dtype=torch.bfloat16, device=cuda)
    lb.gemv_mx(fmt, x, *rows_alone(fmt, w, s, first, n - first), one)
    assert torch.equal(y[:, first:], one)
    v = torch.empty(n - first, k, device=cuda)
    lb.dequantize_mx(fmt, *rows_alone(fmt, w, s, first, n - first), v)
    ref = x.double() @ v.double().T
    assert float((one.double() - ref).norm() / ref.norm()) <= 2.0 ** -8


def test_matmul_result_and_operand_past_32_bits(cuda):
    # C has 4.4e9 elements; B's codes pass 2^32 bytes in the second product
    fmt, k = lb.MX_NVFP4, 64
    m = n = 66500
    a, b = codes_of(fmt, m, k, cuda, 5), codes_of(fmt, n, k, cuda, 6)
    c = torch.empty(m, n, dtype=torch.bfloat16, device=cuda)
    lb.matmul_mx(fmt, *a, *b, c)
    first = (m - 100) // 128 * 128
    one = torch.empty(m - first, n, dtype=torch.bfloat16, device=cuda)
    lb.matmul_mx(fmt, *rows_alone(fmt, *a, first, m - first), *b, one)
    assert torch.equal(c[first:], one)
    del c, one
    n, k = 270000, 32768
    b = codes_of(lb.MX_FP4, n, k, cuda, 7)
    a = codes_of(lb.MX_FP4, 16, k, cuda, 8)
    c = torch.empty(16, n, dtype=torch.float32, device=cuda)
    lb.matmul_mx(lb.MX_FP4, *a, *b, c)
    first = (n - 300) // 128 * 128
    va, vb = torch.empty(16, k, device=cuda), torch.empty(n - first, k, device=cuda)
    lb.dequantize_mx(lb.MX_FP4, *a, va)
    lb.dequantize_mx(lb.MX_FP4, *rows_alone(lb.MX_FP4, *b, first, n - first), vb)
    ref = va.double() @ vb.double().T
    assert float((c[:, first:].double() - ref).norm() / ref.norm()) <= 1e-5
