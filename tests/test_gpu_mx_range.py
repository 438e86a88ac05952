"""The few-row product over the whole range of block scales: weights at either end of E8M0 against bf16 x
whose products with them are ordinary numbers, in 64 bits."""
import numpy as np
import pytest
import torch

import lyth_b200 as lb
from tests import mxref as mx
from tests.test_gpu_mx import product_bound, wide

pytestmark = pytest.mark.gpu

E8M0 = [lb.MX_FP8, lb.MX_FP4]
BF16 = torch.bfloat16


def weights(fmt, n, k, bytes_of, rng, cuda):
    """Codes of a normal matrix under scale bytes n x blocks: device operands and float64 values."""
    codes, _ = mx.quantize(fmt, rng.standard_normal((n, k)))
    scales = np.broadcast_to(bytes_of, (n, codes.shape[1] // 32)).astype(np.int64)
    return (torch.from_numpy(mx.pack(fmt, codes)).to(cuda), torch.from_numpy(mx.tile(scales, 0xFF)).to(cuda),
            mx.values(fmt, codes, scales)[:, :k])


def check(cuda, fmt, x, w, scales, vw):
    x = x.to(BF16)
    y = torch.empty(x.shape[0], vw.shape[0], dtype=BF16, device=cuda)
    lb.gemv_mx(fmt, x.to(cuda), w, scales, y)
    vx = x.double().numpy()
    want = vx @ vw.T
    assert np.abs(want).max() < 2.0 ** 127  # the case is an ordinary number
    got = wide(y)
    assert np.isfinite(got).all()
    bound = product_bound(vx, vw, 1.0, x.shape[1], BF16)
    assert (np.abs(got - want) <= bound).all(), (np.argwhere(np.abs(got - want) > bound)[:4], got, want)
    return y


@pytest.mark.parametrize("fmt", E8M0)
@pytest.mark.parametrize("m", [1, 3, 8])
@pytest.mark.parametrize("byte,ex", [(235, 0), (250, -100), (250, -30), (230, -120), (1, 110), (3, 60), (20, -10), (40, 100), (62, 0),
                                     (65, 0), (190, 0), (193, 0), (66, -60), (127, 100), (127, -110)])
def test_gemv_scales_at_either_end(cuda, fmt, m, byte, ex):
    rng = np.random.default_rng(byte + ex + m)
    n, k = 70, 300
    w, s, vw = weights(fmt, n, k, np.clip(byte + rng.integers(-2, 3, (n, mx.padded(fmt, k) // 32)), 0, 254), rng, cuda)
    x = torch.from_numpy(rng.standard_normal((m, k)).astype(np.float32)) * 2.0 ** ex
    check(cuda, fmt, x, w, s, vw)


@pytest.mark.parametrize("fmt", E8M0)
def test_gemv_one_code_under_a_large_scale(cuda, fmt):
    # 6 * 2^112 is an ordinary bf16 number; so is it with a step of the other sign beside it
    codes = np.zeros((2, 256), np.int64)
    six = {lb.MX_FP8: 0x4C, lb.MX_FP4: 7}[fmt]
    minus = {lb.MX_FP8: 0x80, lb.MX_FP4: 8}[fmt]
    codes[:, 0] = six
    codes[1, 128], codes[1, 200] = six | minus, six
    scales = np.full((2, 8), 127 + 112)
    y = torch.empty(1, 2, dtype=BF16, device=cuda)
    lb.gemv_mx(fmt, torch.ones(1, 256, dtype=BF16, device=cuda), torch.from_numpy(mx.pack(fmt, codes)).to(cuda),
               torch.from_numpy(mx.tile(scales)).to(cuda), y)
    assert wide(y).tolist() == [[6 * 2.0 ** 112, 6 * 2.0 ** 112]]


@pytest.mark.parametrize("fmt", E8M0)
def test_gemv_every_scale_in_one_row(cuda, fmt):
    # a scale byte for every 128 columns, x as far the other way, so that all products weigh alike
    rng = np.random.default_rng(2)
    bytes_ = np.array([4, 250, 30, 220, 63, 64, 191, 192, 127, 5, 249, 100], np.int64)
    n, k = 40, 128 * len(bytes_)
    w, s, vw = weights(fmt, n, k, np.repeat(bytes_, 4)[None, :], rng, cuda)
    x = torch.from_numpy((rng.standard_normal((5, k)) * np.repeat(np.exp2(127.0 - bytes_ - 4), 128)).astype(np.float32))
    y = check(cuda, fmt, x, w, s, vw)
    for i in range(5):  # alone the same bits
        one = torch.empty(1, n, dtype=BF16, device=cuda)
        lb.gemv_mx(fmt, x[i:i + 1].to(BF16).to(cuda), w, s, one)
        assert torch.equal(one[0].view(torch.int16), y[i].view(torch.int16))


@pytest.mark.parametrize("fmt", E8M0)
def test_gemv_bad_scale_beside_large_ones(cuda, fmt):
    # a NaN scale poisons its row and no other; results past bf16 are infinite
    rng = np.random.default_rng(9)
    n, k = 20, 256
    bytes_ = np.full((n, 8), 240)
    bytes_[3, 2] = 255
    bytes_[7, :] = 254
    codes, _ = mx.quantize(fmt, np.abs(rng.standard_normal((n, k))))
    y = torch.empty(2, n, dtype=BF16, device=cuda)
    x = torch.stack([torch.full((k,), 2.0 ** -60), torch.full((k,), 1.0)]).to(BF16).to(cuda)
    lb.gemv_mx(fmt, x, torch.from_numpy(mx.pack(fmt, codes)).to(cuda), torch.from_numpy(mx.tile(bytes_)).to(cuda), y)
    got = wide(y)
    assert np.isnan(got[:, 3]).all() and not np.isnan(np.delete(got, 3, 1)).any()
    assert np.isfinite(np.delete(got[0], 3)).all() and got[1, 7] == np.inf
