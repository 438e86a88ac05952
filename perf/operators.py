"""The microscaled operators: their cases, their plain form, their calls and their definition in 64 bits.

Formats (a row is cut into blocks along its columns; each block has one scale):

    mxfp8   E4M3 codes, 8 bits, blocks of 32, scale 2^e held as E8M0
    mxfp4   E2M1 codes, 4 bits, blocks of 32, scale 2^e held as E8M0
    nvfp4   E2M1 codes, 4 bits, blocks of 16, scale held as E4M3, times one f32 scale per tensor

A row of `cols` values is held as k >= cols codes, k the next multiple of four blocks; what is behind
`cols` is zero. Codes are row-major, the even column in a byte's low half. Scales lie in tiles of 128 rows x
4 blocks, 512 bytes each, tiles row-tile by row-tile: row r, block b of a tile at (r % 32) * 16 + (r // 32) * 4 + b.

quantize   x -> codes, scales; returned as the values they stand for
rmsnorm    h = x + residual; codes and scales of h / sqrt(mean(h^2) + eps) * weight, and h
matmul     c = alpha * a @ b.T, a and b microscaled
gemv       y = alpha * x @ w.T for a few rows of 16-bit x, w microscaled
"""
import math

import torch

own = False

# NVFP4 tensor scales, as a calibration leaves them: of weights, and of activations (f32 values)
WEIGHT_SCALE = float(torch.tensor(0.12 / (6 * 448)))
ACTIVATION_SCALE = float(torch.tensor(64.0 / (6 * 448)))
BLOCK = {"mxfp8": 32, "mxfp4": 32, "nvfp4": 16}
DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # a projection's weights, quantised once when a model is loaded
        {"name": "quantize weights nvfp4", "op": "quantize", "fmt": "nvfp4", "ty": "bf16", "rows": 14336, "cols": 4096, "pad": 0},
        # activations of a ragged batch, a slice of a wider buffer, odd width
        {"name": "quantize ragged mxfp4", "op": "quantize", "fmt": "mxfp4", "ty": "f16", "rows": 333, "cols": 4101, "pad": 59},
        # a full-precision master copy to 8 bits
        {"name": "quantize f32 mxfp8", "op": "quantize", "fmt": "mxfp8", "ty": "f32", "rows": 2048, "cols": 4096, "pad": 0},
        # one new token: the smallest call, all latency
        {"name": "rmsnorm token", "op": "rmsnorm", "fmt": "mxfp8", "ty": "bf16", "rows": 1, "cols": 4096, "residual": True},
        # a long prompt
        {"name": "rmsnorm prompt", "op": "rmsnorm", "fmt": "mxfp8", "ty": "bf16", "rows": 8192, "cols": 4096, "residual": True},
        # a ragged batch of odd width, the first norm (nothing to add yet)
        {"name": "rmsnorm ragged", "op": "rmsnorm", "fmt": "mxfp8", "ty": "f16", "rows": 777, "cols": 5003, "residual": False},
        # gate projection of a long prompt
        {"name": "matmul prompt nvfp4", "op": "matmul", "fmt": "nvfp4", "ty": "bf16", "m": 4096, "n": 14336, "k": 4096},
        # the square contraction of the benchmark, in 8 bits
        {"name": "matmul square mxfp8", "op": "matmul", "fmt": "mxfp8", "ty": "f16", "m": 4096, "n": 4096, "k": 4096},
        # nothing a multiple of a tile, full-precision result
        {"name": "matmul ragged mxfp4", "op": "matmul", "fmt": "mxfp4", "ty": "f32", "m": 1001, "n": 1111, "k": 4032},
        # one step of 32 sequences: weights read once, few rows
        {"name": "matmul few rows nvfp4", "op": "matmul", "fmt": "nvfp4", "ty": "bf16", "m": 32, "n": 14336, "k": 4096},
        # one token through the gate projection
        {"name": "gemv token nvfp4", "op": "gemv", "fmt": "nvfp4", "ty": "bf16", "m": 1, "n": 14336, "k": 4096},
        # four tokens through the way back
        {"name": "gemv four mxfp4", "op": "gemv", "fmt": "mxfp4", "ty": "f16", "m": 4, "n": 4096, "k": 14336},
    ]


def _spread(rng, low, high):
    """A whole number in [low, high], even over its logarithm, odd ones among them."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    op = rng.choice(["quantize", "rmsnorm", "matmul", "gemv"])
    fmt = rng.choice(["mxfp8", "mxfp4", "nvfp4"])
    if op == "quantize":
        cols = _spread(rng, 16, 16384)
        rows = _spread(rng, 1, min(16384, 14336 * 4096 // cols))
        return {"op": op, "fmt": fmt, "ty": rng.choice(["f32", "f16", "bf16"]), "rows": rows, "cols": cols, "pad": rng.choice([0, 0, 8, 37])}
    if op == "rmsnorm":
        cols = _spread(rng, 64, 16384)
        rows = _spread(rng, 1, min(8192, 8192 * 4096 // cols))
        return {"op": op, "fmt": "mxfp8", "ty": rng.choice(["f32", "f16", "bf16"]), "rows": rows, "cols": cols, "residual": rng.choice([True, False])}
    if op == "matmul":
        k = _spread(rng, 32, 8192)
        n = _spread(rng, 16, 14336)
        m = _spread(rng, 1, min(4096, max(1, 4096 * 14336 * 4096 // (n * k))))
        return {"op": op, "fmt": fmt, "ty": rng.choice(["f32", "f16", "bf16"]), "m": m, "n": n, "k": k}
    k = _spread(rng, 64, 16384)
    n = _spread(rng, 16, min(16384, 14336 * 4096 // k))
    return {"op": op, "fmt": fmt, "ty": rng.choice(["f16", "bf16"]), "m": rng.randint(1, 8), "n": n, "k": k}


def _padded(fmt, cols):
    word = 4 * BLOCK[fmt]
    return -(-cols // word) * word


def _row_bytes(fmt, cols):
    return _padded(fmt, cols) // (1 if fmt == "mxfp8" else 2)


def _scale_bytes(fmt, rows, cols):
    return -(-rows // 128) * (_padded(fmt, cols) // (4 * BLOCK[fmt])) * 512


# ------------------------------------------------------------------------------------- plain form
def _tables(device):
    """What each byte stands for: two E2M1 codes, an E4M3 code, an E8M0 scale."""
    mag = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
    e2m1 = torch.cat([mag, -mag])
    byte = torch.arange(256)
    exp, frac = (byte >> 3) & 15, (byte & 7).float()
    e4m3 = torch.where(exp == 0, frac * 2.0 ** -9, (1 + frac / 8) * torch.exp2((exp - 7).float())) * torch.where(byte < 128, 1.0, -1.0)
    e4m3[(byte & 127) == 127] = float("nan")
    e8m0 = torch.exp2((byte - 127).double()).float()
    e8m0[255] = float("nan")
    return {"pair": torch.stack([e2m1[byte & 15], e2m1[byte >> 4]], 1).to(device), "e4m3": e4m3.to(device), "e8m0": e8m0.to(device)}


def _untile(fmt, scales, rows, k):
    """Scales in rows x blocks."""
    blocks = k // BLOCK[fmt]
    return scales.view(-(-rows // 128), blocks // 4, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-1, blocks)[:rows]


def _tile(scales, rows, blocks):
    """The same back into tiles; rows behind the last are zero."""
    full = torch.zeros(-(-rows // 128) * 128, blocks, dtype=torch.uint8, device=scales.device)
    full[:rows] = scales
    return full.view(-1, 4, 32, blocks // 4, 4).permute(0, 3, 2, 1, 4).reshape(-1).contiguous()


def _decode(fmt, codes, scales, t):
    """rows x k values in f32, without the tensor's scale."""
    rows = codes.shape[0]
    v = t["e4m3"][codes.int()] if fmt == "mxfp8" else t["pair"][codes.int()].reshape(rows, -1)
    s = t["e4m3" if fmt == "nvfp4" else "e8m0"][_untile(fmt, scales, rows, v.shape[1]).int()]
    return (v.view(rows, -1, BLOCK[fmt]) * s[:, :, None]).view(rows, -1)


def _quantized(fmt, x, g):
    """f32 rows x cols -> element values and block scales (f32, in rows x blocks x BLOCK and rows x blocks x 1)."""
    rows, cols = x.shape
    x = torch.nn.functional.pad(x, (0, _padded(fmt, cols) - cols)).view(rows, -1, BLOCK[fmt])
    amax = x.abs().amax(2, keepdim=True)
    if fmt == "nvfp4":
        s = (amax * (1.0 / (6.0 * g))).clamp(max=448.0).to(torch.float8_e4m3fn).float()
        q = torch.where(s > 0, x / (s * g), 0.0)
    else:
        # the exponent of the largest value, less that of the format's largest
        e = ((amax.view(torch.int32) >> 23) - (8 if fmt == "mxfp8" else 2)).clamp(min=0)
        s = ((e << 23) | torch.where(e == 0, 1 << 22, 0)).int().view(torch.float32)
        q = x * ((254 - e) << 23).int().view(torch.float32)
    if fmt == "mxfp8":
        return q.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).float(), s
    a = q.abs()
    i = (a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
    v = torch.where(i < 5, i * 0.5, i - 2.0) + torch.where(i == 7, 1.0, 0.0)
    return torch.copysign(v, q), s


def _quantized_values(fmt, x, g):
    v, s = _quantized(fmt, x, g)
    return (v * s * g).view(x.shape[0], -1)[:, : x.shape[1]]


def _encode(fmt, x, g):
    """Codes and tiled scales of f32 rows: what a user has in hand from the quantisation."""
    v, s = _quantized(fmt, x, g)
    rows = x.shape[0]
    if fmt == "mxfp8":
        codes = v.to(torch.float8_e4m3fn).view(torch.uint8).view(rows, -1)
    else:
        a = v.abs()
        i = torch.where(a < 3, a * 2, torch.where(a == 6, a + 1, a + 2)).to(torch.uint8) | (torch.signbit(v).to(torch.uint8) << 3)
        i = i.view(rows, -1, 2)
        codes = i[:, :, 0] | (i[:, :, 1] << 4)
    byte = s.to(torch.float8_e4m3fn).view(torch.uint8) if fmt == "nvfp4" else (s.view(torch.int32) >> 23).to(torch.uint8)
    return codes.contiguous(), _tile(byte.view(rows, -1), rows, byte.shape[1])


def _plain(s):
    op, fmt = s["op"], s["fmt"]
    if op == "quantize":
        return _quantized_values(fmt, s["x"].float(), s["g"]).to(torch.bfloat16)
    if op == "rmsnorm":
        h = s["x"].float()
        if s["residual"] is not None:
            h = h + s["residual"].float()
        y = h * torch.rsqrt(h.square().mean(1, keepdim=True) + s["eps"]) * s["weight"].float()
        v = _quantized_values(fmt, y, 1.0).to(torch.bfloat16)
        return [v] if s["residual"] is None else [v, h.to(s["x"].dtype)]
    if op == "matmul":
        a = _decode(fmt, s["a"], s["a_scales"], s["tables"])
        b = _decode(fmt, s["b"], s["b_scales"], s["tables"])
        return (s["alpha"] * (a @ b.T)).to(s["c"].dtype)
    w = _decode(fmt, s["w"], s["w_scales"], s["tables"])
    return (s["alpha"] * (s["x"].float() @ w[:, : s["x"].shape[1]].T)).to(s["y"].dtype)


# ------------------------------------------------------------------------------------- own calls
def _own(s):
    import lyth_b200 as lb

    op, fmt = s["op"], {"mxfp8": lb.MX_FP8, "mxfp4": lb.MX_FP4, "nvfp4": lb.MX_NVFP4}[s["fmt"]]
    if op == "quantize":
        lb.quantize_mx(fmt, s["x"], s["codes"], s["scales"], tensor_scale=s["g"])
        lb.dequantize_mx(fmt, s["codes"], s["scales"], s["values"], tensor_scale=s["g"])
        return s["values"]
    if op == "rmsnorm":
        lb.rmsnorm_mx(fmt, s["x"], s["weight"], s["codes"], s["scales"], residual=s["residual"], residual_out=s["h"], eps=s["eps"])
        lb.dequantize_mx(fmt, s["codes"], s["scales"], s["values"])
        return [s["values"]] if s["residual"] is None else [s["values"], s["h"]]
    if op == "matmul":
        lb.matmul_mx(fmt, s["a"], s["a_scales"], s["b"], s["b_scales"], s["c"], alpha=s["alpha"])
        return s["c"]
    lb.gemv_mx(fmt, s["x"], s["w"], s["w_scales"], s["y"], alpha=s["alpha"])
    return s["y"]


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    op, fmt, ty = case["op"], case["fmt"], DTYPE[case["ty"]]

    def normal(rows, cols, sigma):
        return torch.randn(rows, cols, generator=gen, device=dev) * sigma

    def activations(rows, cols):
        """Normal values, a few columns of each row block much larger, as a residual stream has them."""
        loud = 1 + 15 * (torch.rand(cols, generator=gen, device=dev) < 0.01)
        return normal(rows, cols, 1.0) * loud

    s = {"op": op, "fmt": fmt, "g": 1.0}
    if op in ("quantize", "rmsnorm"):
        rows, cols = case["rows"], case["cols"]
        s["codes"] = torch.empty(rows, _row_bytes(fmt, cols), dtype=torch.uint8, device=dev)
        s["scales"] = torch.empty(_scale_bytes(fmt, rows, cols), dtype=torch.uint8, device=dev)
        s["values"] = torch.empty(rows, cols, dtype=torch.bfloat16, device=dev)
    if op == "quantize":
        s["x"] = normal(rows, cols + case["pad"], 0.02).to(ty)[:, :cols]
        s["g"] = WEIGHT_SCALE if fmt == "nvfp4" else 1.0
    elif op == "rmsnorm":
        s["x"] = activations(rows, cols).to(ty)
        s["residual"] = activations(rows, cols).to(ty) if case["residual"] else None
        s["h"] = torch.empty(rows, cols, dtype=ty, device=dev) if case["residual"] else None
        s["weight"] = (1 + 0.1 * torch.randn(cols, generator=gen, device=dev)).to(ty)
        s["eps"] = 1e-5
    else:
        m, n, k = case["m"], case["n"], case["k"]
        gw = WEIGHT_SCALE if fmt == "nvfp4" else 1.0
        w, w_scales = _encode(fmt, normal(n, k, 0.02), gw)
        s["tables"] = _tables(dev)
        if op == "matmul":
            ga = ACTIVATION_SCALE if fmt == "nvfp4" else 1.0
            s["a"], s["a_scales"] = _encode(fmt, activations(m, k), ga)
            s["b"], s["b_scales"], s["alpha"] = w, w_scales, ga * gw
            s["c"] = torch.empty(m, n, dtype=ty, device=dev)
        else:
            s["x"], s["w"], s["w_scales"], s["alpha"] = activations(m, k).to(ty), w, w_scales, gw
            s["y"] = torch.empty(m, n, dtype=ty, device=dev)
    return s


# ------------------------------------------------------------------------------------- cost
def work(case):
    op, fmt, size = case["op"], case["fmt"], {"f32": 4, "f16": 2, "bf16": 2}[case["ty"]]

    def held(rows, cols):
        return rows * (_row_bytes(fmt, cols) + _padded(fmt, cols) // BLOCK[fmt])

    if op == "quantize":
        n = case["rows"] * case["cols"]
        # read x, write codes and scales; the values read them back and are written as bf16
        return {"bytes": n * size + 2 * held(case["rows"], case["cols"]) + 2 * n, "flops": 4 * n}
    if op == "rmsnorm":
        n = case["rows"] * case["cols"]
        return {"bytes": n * size * (3 if case["residual"] else 1) + case["cols"] * size + 2 * held(case["rows"], case["cols"]) + 2 * n, "flops": 8 * n}
    m, n, k = case["m"], case["n"], case["k"]
    if op == "matmul":
        return {"bytes": held(m, k) + held(n, k) + m * n * size, "flops": 2 * m * n * k}
    return {"bytes": m * k * size + held(n, k) + m * n * size, "flops": 2 * m * n * k}


# ------------------------------------------------------------------------------------- definition in 64 bits
def _levels(fmt):
    """The non-negative values of a code, ascending by code."""
    if fmt == "mxfp8":
        return [(i % 8) / 8 * 2.0 ** -6 if i < 8 else (1 + i % 8 / 8) * 2.0 ** (i // 8 - 7) for i in range(127)]
    return [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _nearest(levels, v):
    """The level nearest to v >= 0, ties to the even code, values behind the last to the last."""
    lv = torch.tensor(levels, dtype=torch.float64, device=v.device)
    hi = torch.searchsorted(lv, v.contiguous()).clamp(1, len(levels) - 1)
    lo = hi - 1
    up, down = lv[hi] - v, v - lv[lo]
    return lv[torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)]


def _exact_quantized(fmt, x, g):
    b, out = BLOCK[fmt], torch.zeros_like(x)
    whole = torch.zeros(x.shape[0], _padded(fmt, x.shape[1]), dtype=torch.float64, device=x.device)
    whole[:, : x.shape[1]] = x
    whole = whole.unflatten(1, (-1, b))
    top = whole.abs().max(2).values.unsqueeze(2)
    if fmt == "nvfp4":
        scale = _nearest(_levels("mxfp8"), top / 6 / g) * g
    else:
        scale = torch.ldexp(torch.ones_like(top), ((torch.frexp(top).exponent - 1).clamp(min=-126) - (8 if fmt == "mxfp8" else 2)).clamp(min=-127))
    ratio = torch.where(scale > 0, whole.abs() / torch.where(scale > 0, scale, 1), 0)
    out[:] = (torch.sign(whole) * _nearest(_levels(fmt), ratio) * scale).flatten(1)[:, : x.shape[1]]
    return out


def _exact_values(fmt, codes, scales, rows, cols):
    """Row-major values of codes and tiled scales, found byte by byte from the layout's definition."""
    dev, b = codes.device, BLOCK[fmt]
    j = torch.arange(cols, device=dev)
    r = torch.arange(rows, device=dev)[:, None]
    if fmt == "mxfp8":
        c, sign = codes[:, j].long() & 127, codes[:, j] >= 128
    else:
        c = (codes[:, j // 2].long() >> (4 * (j % 2))) & 15
        c, sign = c & 7, c >= 8
    v = torch.tensor(_levels(fmt), dtype=torch.float64, device=dev)[c]
    blk = j // b
    tiles = codes.shape[1] * (1 if fmt == "mxfp8" else 2) // (4 * b)
    at = ((r // 128) * tiles + blk // 4) * 512 + (r % 32) * 16 + (r % 128 // 32) * 4 + blk % 4
    byte = scales[at].long()
    if fmt == "nvfp4":
        scale = torch.tensor(_levels("mxfp8"), dtype=torch.float64, device=dev)[byte]
    else:
        scale = torch.exp2((byte - 127).double())
    return torch.where(sign, -v, v) * scale


def exact(case, seed):
    s = prepare(case, seed)
    op, fmt = case["op"], case["fmt"]
    if op == "quantize":
        return _exact_quantized(fmt, s["x"].double(), s["g"])
    if op == "rmsnorm":
        h = s["x"].double() if s["residual"] is None else s["x"].double() + s["residual"].double()
        y = h / (h.pow(2).sum(1, keepdim=True) / h.shape[1] + s["eps"]).sqrt() * s["weight"].double()
        v = _exact_quantized(fmt, y, 1.0)
        return [v] if s["residual"] is None else [v, h]
    if op == "matmul":
        a = _exact_values(fmt, s["a"], s["a_scales"], case["m"], case["k"])
        b = _exact_values(fmt, s["b"], s["b_scales"], case["n"], case["k"])
        return torch.einsum("mk,nk->mn", a, b) * s["alpha"]
    w = _exact_values(fmt, s["w"], s["w_scales"], case["n"], case["k"])
    return torch.einsum("mk,nk->mn", s["x"].double(), w) * s["alpha"]
