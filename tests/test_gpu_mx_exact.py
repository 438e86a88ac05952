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
