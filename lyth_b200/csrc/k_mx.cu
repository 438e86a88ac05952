// Quantisation to and from the block-scaled formats (mx.cuh), and the RMS norm that adds the
// residual and quantises its output in the same pass.
//
// All three are bound by HBM: a value is read once, its code (4 or 8 bits) and a 16th to a 32nd of a
// scale byte are written. A thread holds sixteen consecutive values: an NVFP4 block, or half an MX
// block whose other half is the neighbouring lane's (mx_quantize), so no value is read twice and
// shared memory is used only for the norm's row sum. Measured: 14336 x 4096 bf16 to NVFP4 27.1 us (150
// MB, 5.6 TB/s), back 24.0 (6.3); f32 24.6 us of 8192 x 4096 (6.2); the norm of 8192 x 4096 bf16 with a
// residual to MXFP8 38.3 us (236 MB, 6.2 TB/s). Rows that do not start on 32 bytes cost up to twice the
// norm's time (8192 x 4099: 67 us), in the instructions that shift them.
#include "mx.cuh"

namespace lyth {

constexpr int kMxThreads = 256;

// Chunks (16 columns) are one flat range, rows back to back, kMxThreads * U of them to a block: a
// warp's 32 chunks may lie in several short rows, and a scale word's chunks never straddle a row
// because a row holds whole words. One division finds a thread's first chunk (32-bit where the range
// allows); the next ones are a constant step on.
struct MxWalk {
    uint64_t row;
    uint32_t c;
    LYTH_D MxWalk(uint64_t flat, uint32_t cpr, bool narrow) {
        if (narrow) {
            row = (uint32_t)flat / cpr;
            c = (uint32_t)flat - (uint32_t)row * cpr;
        } else {
            row = flat / cpr;
            c = (uint32_t)(flat - row * cpr);
        }
    }
    LYTH_D void step(uint32_t rows, uint32_t chunks, uint32_t cpr) {
        row += rows;
        c += chunks;
        if (c >= cpr) { c -= cpr; row++; }
    }
};
struct MxFlat {
    uint64_t rows, ld;
    uint32_t cols, cpr;             // chunks per row
    uint32_t step_rows, step_c;     // kMxThreads chunks on
    bool narrow;                    // every flat index fits 32 bits
};

// U: chunks of a thread, all loaded before the first is used.
template <int FMT, int TY, bool VEC, int U>
__global__ void __launch_bounds__(kMxThreads)
    mx_quantize_kernel(const typename MxElem<TY>::type *__restrict__ x, MxFlat f, float inv6g, float g,
                       uint8_t *__restrict__ codes, uint8_t *__restrict__ scales) {
    grid_next();
    const uint32_t words = f.cpr * 16 / Mx<FMT>::kWord;
    const uint64_t row_bytes = (uint64_t)f.cpr * 2 * Mx<FMT>::kBits;
    grid_wait();
    x = after_wait(x);
    const void *hi = x + (f.rows - 1) * f.ld + f.cols;
    MxWalk w((uint64_t)blockIdx.x * (kMxThreads * U) + threadIdx.x, f.cpr, f.narrow);
    uint64_t row[U];
    uint32_t c[U], in[U][kMxWords<TY>];
#pragma unroll
    for (int u = 0; u < U; u++) {
        row[u] = w.row;
        c[u] = w.c;
        if (w.row < f.rows) {
            mx_load<TY, VEC>(x + w.row * f.ld, w.c, f.cols, x, hi, in[u]);
        } else {
#pragma unroll
            for (int i = 0; i < kMxWords<TY>; i++) in[u][i] = 0;
        }
        w.step(f.step_rows, f.step_c, f.cpr);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        float v[16];
        mx_widen<TY>(in[u], v);
        mx_quantize<FMT>(v, mx_top_words<TY>(in[u]), row[u] < f.rows, c[u], codes + row[u] * row_bytes,
                         scales + mx_scale_row(row[u], words), inv6g, g);
    }
}

template <int FMT, int TY, bool VEC, int U>
__global__ void __launch_bounds__(kMxThreads)
    mx_dequantize_kernel(const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scales, MxFlat f, float g,
                         typename MxElem<TY>::type *__restrict__ out) {
    const uint32_t words = f.cpr * 16 / Mx<FMT>::kWord;
    constexpr int kLanes = Mx<FMT>::kBlock / 16, kW = Mx<FMT>::kBits / 2;  // lanes of a block, words of a chunk
    const uint64_t flat = (uint64_t)blockIdx.x * (kMxThreads * U) + threadIdx.x;
    grid_next();
    MxWalk w(flat, f.cpr, f.narrow);
    grid_wait();
    codes = after_wait(codes);
    scales = after_wait(scales);
    uint64_t row[U];
    uint32_t c[U], in[U][kW], byte[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        row[u] = w.row;
        c[u] = w.c;
        byte[u] = 0;
#pragma unroll
        for (int i = 0; i < kW; i++) in[u][i] = 0;
        if (w.row < f.rows) {
            const uint8_t *at = codes + (flat + u * kMxThreads) * 4 * kW;
            const uint32_t blk = w.c / kLanes;
            byte[u] = scales[mx_scale_row(w.row, words) + (uint64_t)(blk / 4) * 512 + (blk & 3)];
            if constexpr (FMT == LYTH_MX_FP8) {
                const uint4 t = *reinterpret_cast<const uint4 *>(at);
                in[u][0] = t.x; in[u][1] = t.y; in[u][2] = t.z; in[u][3] = t.w;
            } else {
                const uint2 t = *reinterpret_cast<const uint2 *>(at);
                in[u][0] = t.x; in[u][1] = t.y;
            }
        }
        w.step(f.step_rows, f.step_c, f.cpr);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        uint32_t h[8], o[kMxWords<TY>];
        const float s = mx_scales2<FMT>(byte[u]).x;
        if constexpr (FMT == LYTH_MX_NVFP4 && TY != 0) {
            mx_nvfp4_back<TY>(in[u][0], in[u][1], s, g, o);
            mx_store<TY, VEC>(out + row[u] * f.ld, c[u], f.cols, row[u] < f.rows, o);
            continue;
        }
        if constexpr (FMT == LYTH_MX_FP8) {
#pragma unroll
            for (int i = 0; i < 4; i++) e4m3x4_f16(in[u][i], h[2 * i], h[2 * i + 1]);
        } else {
            uint32_t a[4];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                e2m1x8_f16(in[u][i], a);
#pragma unroll
                for (int j = 0; j < 4; j++) h[4 * i + j] = a[j];
            }
        }
        float v[16];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            float2 t = mx_mul2(f16x2_f32(h[i]), make_float2(s, s));
            if constexpr (FMT == LYTH_MX_NVFP4) t = mx_mul2(t, make_float2(g, g));
            v[2 * i] = t.x;
            v[2 * i + 1] = t.y;
        }
        mx_narrow<TY>(v, o);
        mx_store<TY, VEC>(out + row[u] * f.ld, c[u], f.cols, row[u] < f.rows, o);
    }
}

// h = x + residual (f32; written rounded to the type when residual_out is given),
// y = h * rsqrt(mean(h^2) + eps) * weight, codes and scales of y.
//
// blockDim.x threads (whole warps) own a row, blockDim.y rows share a block. V > 0: a thread's V
// chunks of h stay in registers between the sum and the scaling, so a row is read once. V = 0
// (rows wider than 1024 threads x 2 chunks): the second pass reads x and the residual again, and
// writes residual_out only then, since it may be either of them.
template <int FMT, int TY, int V, bool VEC>
__global__ void __launch_bounds__(1024)
    mx_rmsnorm_kernel(const typename MxElem<TY>::type *x, const typename MxElem<TY>::type *residual,
                      typename MxElem<TY>::type *residual_out, const typename MxElem<TY>::type *__restrict__ weight,
                      uint64_t rows, uint32_t cols, uint64_t ldx, uint64_t ldr, uint64_t ldo, uint32_t cpr, float eps,
                      float inv6g, float g, uint8_t *__restrict__ codes, uint8_t *__restrict__ scales) {
    constexpr int N = kMxWords<TY>, kHeld = V > 0 ? V : 1;
    __shared__ float part[32];
    grid_next();
    grid_wait();
    x = after_wait(x);
    residual = after_wait(residual);
    weight = after_wait(weight);
    const uint32_t tpr = blockDim.x, warps = tpr >> 5;
    const uint32_t words = cpr * 16 / Mx<FMT>::kWord;
    const uint64_t row_bytes = (uint64_t)cpr * 2 * Mx<FMT>::kBits, step = (uint64_t)gridDim.x * blockDim.y;
    const void *x_hi = x + (rows - 1) * ldx + cols, *r_hi = residual ? residual + (rows - 1) * ldr + cols : nullptr;
    auto load = [&](uint64_t row, uint32_t c, uint32_t (&a)[N], uint32_t (&b)[N]) {
#pragma unroll
        for (int i = 0; i < N; i++) a[i] = b[i] = 0;
        if (row < rows && c < cpr) {
            mx_load<TY, VEC>(x + row * ldx, c, cols, x, x_hi, a);
            if (residual) mx_load<TY, VEC>(residual + row * ldr, c, cols, residual, r_hi, b);
        }
    };
    auto add = [&](const uint32_t (&a)[N], const uint32_t (&b)[N], float (&v)[16]) {
        mx_widen<TY>(a, v);
        if (residual) {
            float r[16];
            mx_widen<TY>(b, r);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float2 t = mx_add2(make_float2(v[2 * i], v[2 * i + 1]), make_float2(r[2 * i], r[2 * i + 1]));
                v[2 * i] = t.x;
                v[2 * i + 1] = t.y;
            }
        }
    };
    auto keep = [&](uint64_t row, uint32_t c, const float (&v)[16]) {
        if (residual_out) {
            uint32_t o[N];
            mx_narrow<TY>(v, o);
            mx_store<TY, VEC>(residual_out + row * ldo, c, cols, row < rows && c < cpr, o);
        }
    };
    auto load_weight = [&](uint32_t c, uint32_t (&w)[N]) {
#pragma unroll
        for (int i = 0; i < N; i++) w[i] = 0;
        if (c < cpr) mx_load<TY, VEC>(weight, c, cols, weight, weight + cols, w);
    };
    uint64_t row0 = (uint64_t)blockIdx.x * blockDim.y;
    for (; row0 < rows; row0 += step) {
        const uint64_t row = row0 + threadIdx.y;
        float ss = 0.0f;
        float h[kHeld][16];
        auto square = [&](const float (&v)[16]) {
            float2 t = make_float2(ss, 0.0f);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float2 u = make_float2(v[2 * i], v[2 * i + 1]);
                t = mx_fma2(u, u, t);
            }
            ss = __fadd_rn(t.x, t.y);
        };
        uint32_t w[kHeld][N];
        if constexpr (V > 0) {
#pragma unroll
            for (int j = 0; j < V; j++) {
                uint32_t a[N], b[N];
                load(row, threadIdx.x + j * tpr, a, b);
                add(a, b, h[j]);
                square(h[j]);
                keep(row, threadIdx.x + j * tpr, h[j]);
                load_weight(threadIdx.x + j * tpr, w[j]);
            }
        } else {
            for (uint32_t c = threadIdx.x; c < cpr; c += tpr) {
                uint32_t a[N], b[N];
                load(row, c, a, b);
                add(a, b, h[0]);
                square(h[0]);
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ss = __fadd_rn(ss, __shfl_xor_sync(0xFFFFFFFFu, ss, o));
        if (warps > 1) {
            const uint32_t w0 = threadIdx.y * warps;
            if ((threadIdx.x & 31) == 0) part[w0 + (threadIdx.x >> 5)] = ss;
            __syncthreads();
            ss = 0.0f;
            for (uint32_t i = 0; i < warps; i++) ss = __fadd_rn(ss, part[w0 + i]);
            __syncthreads();
        }
        const float scale = rsqrtf(__fadd_rn(__fdiv_rn(ss, (float)cols), eps));
        uint8_t *cr = codes + row * row_bytes, *sr = scales + mx_scale_row(row, words);
        // whole warps walk the chunks (mx_quantize shuffles); lanes behind the row store nothing, and
        // share no block or scale word with lanes inside it
        const int trips = V > 0 ? V : (int)((cpr + tpr - 1) / tpr);
#pragma unroll(kHeld)
        for (int j = 0; j < trips; j++) {
            const uint32_t c = threadIdx.x + (uint32_t)j * tpr;
            const bool live = row < rows && c < cpr;
            float(&v)[16] = h[V > 0 ? j : 0];
            if constexpr (V == 0) {
                uint32_t a[N], b[N];
                load(row, c, a, b);
                add(a, b, v);
                keep(row, c, v);
            }
            if constexpr (V == 0) load_weight(c, w[0]);
            float wt[16];
            mx_widen<TY>(w[V > 0 ? j : 0], wt);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float2 y = mx_mul2(mx_mul2(make_float2(v[2 * i], v[2 * i + 1]), make_float2(scale, scale)),
                                         make_float2(wt[2 * i], wt[2 * i + 1]));
                v[2 * i] = y.x;
                v[2 * i + 1] = y.y;
            }
            mx_quantize<FMT>(v, mx_top(v), live, c, cr, sr, inv6g, g);
        }
    }
}

}  // namespace lyth

using namespace lyth;

extern "C" uint64_t lyth_b200_mx_row_bytes(int fmt, uint32_t cols) {
    return mx_known(fmt) ? mx_code_bytes(fmt, mx_padded(fmt, cols)) : 0;
}

extern "C" uint64_t lyth_b200_mx_scale_bytes(int fmt, uint64_t rows, uint32_t cols) {
    return mx_known(fmt) ? (rows + 127) / 128 * (mx_padded(fmt, cols) / (4 * mx_block(fmt))) * 512 : 0;
}

// Chunks to blocks of kMxThreads * u.
static MxFlat mx_flat(int fmt, uint64_t rows, uint32_t cols, uint64_t ld, int u, unsigned &grid) {
    MxFlat f;
    f.rows = rows;
    f.ld = ld;
    f.cols = cols;
    f.cpr = (uint32_t)(mx_padded(fmt, cols) / kMxChunk);
    f.step_rows = kMxThreads / f.cpr;
    f.step_c = kMxThreads % f.cpr;
    const uint64_t per = (uint64_t)kMxThreads * u, blocks = (rows * f.cpr + per - 1) / per;  // 2^30 at most
    f.narrow = blocks * per <= 0xFFFFFFFFull;
    grid = (unsigned)blocks;
    return f;
}

// What every entry here asks of its sizes: known format and type, columns that a 32-bit index
// holds after padding, no more values than a grid and a byte offset hold (rows * k may pass 64 bits).
static int mx_shape(int fmt, int ty, uint64_t rows, uint32_t cols) {
    if (!mx_known(fmt) || !mx_ty_known(ty)) return LYTH_E_UNSUPPORTED;
    if (cols == 0 || cols > (1u << 30) || rows > (1ull << 40) || rows > (1ull << 42) / mx_padded(fmt, cols)) return LYTH_E_INVALID;
    return LYTH_OK;
}

extern "C" int lyth_b200_quantize_mx(int fmt, int ty, uint64_t rows, uint32_t cols, const void *x, uint64_t ldx,
                                     float tensor_scale, uint8_t *codes, uint8_t *scales, cudaStream_t s) {
    const int e = mx_shape(fmt, ty, rows, cols);
    if (e != LYTH_OK) return e;
    float inv6g;
    if (ldx < cols || !mx_tensor_scale(fmt, tensor_scale, inv6g)) return LYTH_E_INVALID;
    if (rows == 0) return LYTH_OK;
    if (!x || !codes || !scales) return LYTH_E_INVALID;
    if (!aligned16(codes) || !aligned16(scales) || !mx_elem_aligned(x, ty)) return LYTH_E_UNSUPPORTED;
    const bool vec = cols % 16 == 0 && aligned32(x) && ldx * mx_ty_bytes(ty) % 32 == 0;
    unsigned grid;
    const MxFlat f = mx_flat(fmt, rows, cols, ldx, vec ? 2 : 1, grid);
    LYTH_MX_DISPATCH(fmt, ty,
                     auto k = vec ? mx_quantize_kernel<FMT, TY, true, 2> : mx_quantize_kernel<FMT, TY, false, 1>;
                     return mx_launch(k, grid, kMxThreads, 0, s, 1, static_cast<const MxElem<TY>::type *>(x), f,
                                                inv6g, tensor_scale, codes, scales));
    return LYTH_E_UNSUPPORTED;
}

extern "C" int lyth_b200_dequantize_mx(int fmt, int ty, uint64_t rows, uint32_t cols, const uint8_t *codes,
                                       const uint8_t *scales, float tensor_scale, void *out, uint64_t ldo,
                                       cudaStream_t s) {
    const int e = mx_shape(fmt, ty, rows, cols);
    if (e != LYTH_OK) return e;
    float inv6g;
    if (ldo < cols || !mx_tensor_scale(fmt, tensor_scale, inv6g)) return LYTH_E_INVALID;
    if (rows == 0) return LYTH_OK;
    if (!out || !codes || !scales) return LYTH_E_INVALID;
    if (!aligned16(codes) || !aligned16(scales) || !mx_elem_aligned(out, ty)) return LYTH_E_UNSUPPORTED;
    const bool vec = cols % 16 == 0 && aligned32(out) && ldo * mx_ty_bytes(ty) % 32 == 0;
    unsigned grid;
    const MxFlat f = mx_flat(fmt, rows, cols, ldo, vec ? 2 : 1, grid);
    LYTH_MX_DISPATCH(fmt, ty,
                     auto k = vec ? mx_dequantize_kernel<FMT, TY, true, 2> : mx_dequantize_kernel<FMT, TY, false, 1>;
                     return mx_launch(k, grid, kMxThreads, 0, s, 1, codes, scales, f, tensor_scale,
                                                static_cast<MxElem<TY>::type *>(out)));
    return LYTH_E_UNSUPPORTED;
}

template <int FMT, int TY>
static int rmsnorm_launch(const void *x, const void *residual, void *residual_out, const void *weight, uint64_t rows,
                           uint32_t cols, uint64_t ldx, uint64_t ldr, uint64_t ldo, uint32_t cpr, bool vec, float eps,
                           float inv6g, float g, uint8_t *codes, uint8_t *scales, cudaStream_t s) {
    using T = typename MxElem<TY>::type;
    const T *xt = static_cast<const T *>(x), *rt = static_cast<const T *>(residual), *wt = static_cast<const T *>(weight);
    T *ot = static_cast<T *>(residual_out);
    // One chunk a thread is quickest for few rows (one 4096-wide bf16 row: 2.6 us, two chunks 2.9); two
    // chunks in blocks half as large carry more bytes in flight once the rows fill the machine (8192
    // rows: 39.1 against 42.1 us). Of f32 and of rows in shifted words two would spill.
    const bool many = TY != 0 && vec && cpr >= 128 && rows >= 4ull * device_sms();
    const int v = cpr <= 1024 && !many ? 1 : cpr <= 2048 ? 2 : 0;
    const uint32_t tpr = v ? ((cpr + v - 1) / v + 31) / 32 * 32 : 1024;
    const uint32_t per = tpr < 128 ? 128 / tpr : 1;
    const dim3 block(tpr, per);
    const uint64_t need = (rows + per - 1) / per;
    const unsigned grid = need < (1u << 30) ? (unsigned)need : (1u << 30);
    auto k = v == 1   ? (vec ? mx_rmsnorm_kernel<FMT, TY, 1, true> : mx_rmsnorm_kernel<FMT, TY, 1, false>)
             : v == 2 ? (vec ? mx_rmsnorm_kernel<FMT, TY, 2, true> : mx_rmsnorm_kernel<FMT, TY, 2, false>)
                      : (vec ? mx_rmsnorm_kernel<FMT, TY, 0, true> : mx_rmsnorm_kernel<FMT, TY, 0, false>);
    return mx_launch(k, grid, block, 0, s, 1, xt, rt, ot, wt, rows, cols, ldx, ldr, ldo, cpr, eps, inv6g, g, codes,
                               scales);
}

extern "C" int lyth_b200_rmsnorm_mx(int fmt, int ty, uint64_t rows, uint32_t cols, const void *x, uint64_t ldx,
                                    const void *residual, uint64_t ldr, void *residual_out, uint64_t ldo,
                                    const void *weight, float eps, float tensor_scale, uint8_t *codes,
                                    uint8_t *scales, cudaStream_t s) {
    const int e = mx_shape(fmt, ty, rows, cols);
    if (e != LYTH_OK) return e;
    float inv6g;
    if (ldx < cols || (residual && ldr < cols) || (residual_out && ldo < cols) || !(eps >= 0.0f) ||
        !mx_tensor_scale(fmt, tensor_scale, inv6g))
        return LYTH_E_INVALID;
    if (rows == 0) return LYTH_OK;
    if (!x || !weight || !codes || !scales) return LYTH_E_INVALID;
    if (!aligned16(codes) || !aligned16(scales) || !mx_elem_aligned(x, ty) || !mx_elem_aligned(residual, ty) ||
        !mx_elem_aligned(residual_out, ty) || !mx_elem_aligned(weight, ty))
        return LYTH_E_UNSUPPORTED;
    const uint32_t cpr = (uint32_t)(mx_padded(fmt, cols) / kMxChunk);
    const uint64_t size = mx_ty_bytes(ty);
    const bool vec = cols % 16 == 0 && aligned32(x) && ldx * size % 32 == 0 && aligned32(weight) &&
                     (!residual || (aligned32(residual) && ldr * size % 32 == 0)) &&
                     (!residual_out || (aligned32(residual_out) && ldo * size % 32 == 0));
    LYTH_MX_DISPATCH(fmt, ty,
                     return (rmsnorm_launch<FMT, TY>(x, residual, residual_out, weight, rows, cols, ldx, ldr, ldo, cpr,
                                                     vec, eps, inv6g, tensor_scale, codes, scales, s)));
    return LYTH_E_UNSUPPORTED;
}
