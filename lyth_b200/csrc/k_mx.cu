// Quantisation to and from the block-scaled formats (mx.cuh), and the RMS norm that adds the
// residual and quantises its output in the same pass.
//
// All three are bound by HBM: a value is read once, its code (4 or 8 bits) and a 16th to a 32nd of a
// scale byte are written. A thread holds eight consecutive values (one 128-bit load of a 16-bit
// type, two of f32); a block's scale needs the largest magnitude over 2 or 4 neighbouring lanes
// (mx_quantize8), so no value is read twice and shared memory is used only for the norm's row sum.
#include "mx.cuh"

namespace lyth {

constexpr int kMxThreads = 256;

// Chunks (8 columns) are walked as one flat range, rows back to back: a warp's 32 chunks may lie in
// several short rows, and a scale word's chunks never straddle a row because a row holds whole words.
// The (row, chunk) of a thread advances by a constant step, so the only division is the first.
struct MxWalk {
    uint64_t row;
    uint32_t c;
    LYTH_D MxWalk(uint64_t flat, uint32_t cpr) : row(flat / cpr), c((uint32_t)(flat % cpr)) {}
    LYTH_D void step(uint64_t rows, uint32_t chunks, uint32_t cpr) {
        row += rows;
        c += chunks;
        if (c >= cpr) { c -= cpr; row++; }
    }
};

template <int FMT, int TY>
__global__ void __launch_bounds__(kMxThreads)
    mx_quantize_kernel(const typename MxElem<TY>::type *__restrict__ x, uint64_t rows, uint32_t cols, uint64_t ldx,
                       uint32_t cpr, bool vec, float inv6g, float g, uint8_t *__restrict__ codes,
                       uint8_t *__restrict__ scales) {
    const uint64_t total = rows * cpr, stride = (uint64_t)gridDim.x * kMxThreads;
    const uint64_t step_rows = stride / cpr;
    const uint32_t step_c = (uint32_t)(stride % cpr);
    const uint32_t words = cpr * 8 / Mx<FMT>::kWord;
    const uint64_t row_bytes = (uint64_t)cpr * Mx<FMT>::kBits;
    uint64_t flat = (uint64_t)blockIdx.x * kMxThreads + threadIdx.x;
    MxWalk w(flat, cpr);
    // whole warps: the warp's first chunk decides, the last warp's spare lanes hold zeros
    for (uint64_t base = flat - (threadIdx.x & 31); base < total; base += stride) {
        const bool live = w.row < rows;
        float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (live) mx_load8<TY>(x + w.row * ldx, 8 * w.c, cols, vec, v);
        mx_quantize8<FMT>(v, live, w.c, codes + w.row * row_bytes, scales + mx_scale_row(w.row, words), inv6g, g);
        w.step(step_rows, step_c, cpr);
    }
}

template <int FMT, int TY>
__global__ void __launch_bounds__(kMxThreads)
    mx_dequantize_kernel(const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scales, uint64_t rows,
                         uint32_t cols, uint64_t ldo, uint32_t cpr, bool vec, float g,
                         typename MxElem<TY>::type *__restrict__ out) {
    const uint64_t total = rows * cpr, stride = (uint64_t)gridDim.x * kMxThreads;
    const uint64_t step_rows = stride / cpr;
    const uint32_t step_c = (uint32_t)(stride % cpr);
    const uint32_t words = cpr * 8 / Mx<FMT>::kWord;
    uint64_t flat = (uint64_t)blockIdx.x * kMxThreads + threadIdx.x;
    MxWalk w(flat, cpr);
    for (; flat < total; flat += stride, w.step(step_rows, step_c, cpr)) {
        if (8 * w.c >= cols) continue;
        const uint8_t *at = codes + flat * Mx<FMT>::kBits;
        uint32_t h[4];
        if constexpr (FMT == LYTH_MX_FP8) {
            const uint2 u = *reinterpret_cast<const uint2 *>(at);
            e4m3x4_f16(u.x, h[0], h[1]);
            e4m3x4_f16(u.y, h[2], h[3]);
        } else {
            e2m1x8_f16(*reinterpret_cast<const uint32_t *>(at), h);
        }
        constexpr int kLanes = Mx<FMT>::kBlock / 8;
        const uint32_t blk = w.c / kLanes;
        const uint8_t byte = scales[mx_scale_row(w.row, words) + (uint64_t)(blk / 4) * 512 + (blk & 3)];
        const float s = mx_scales2<FMT>(byte).x;
        float v[8];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = f16x2_f32(h[i]);
            v[2 * i] = __fmul_rn(f.x, s);
            v[2 * i + 1] = __fmul_rn(f.y, s);
        }
        if constexpr (FMT == LYTH_MX_NVFP4) {
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = __fmul_rn(v[i], g);
        }
        mx_store8<TY>(out + w.row * ldo, 8 * w.c, cols, vec, v);
    }
}

// h = x + residual (f32; written rounded to the type when residual_out is given),
// y = h * rsqrt(mean(h^2) + eps) * weight, codes and scales of y.
//
// blockDim.x threads (whole warps) own a row, blockDim.y rows share a block. V > 0: a thread's V
// chunks of h stay in registers between the sum and the scaling, so a row is read once. V = 0
// (rows wider than 1024 threads x 4 chunks): the second pass reads x and the residual again, and
// writes residual_out only then, since it may be either of them.
template <int FMT, int TY, int V>
__global__ void __launch_bounds__(1024)
    mx_rmsnorm_kernel(const typename MxElem<TY>::type *x, const typename MxElem<TY>::type *residual,
                      typename MxElem<TY>::type *residual_out, const typename MxElem<TY>::type *__restrict__ weight,
                      uint64_t rows, uint32_t cols, uint64_t ldx, uint64_t ldr, uint64_t ldo, uint32_t cpr, bool vec,
                      float eps, float inv6g, float g, uint8_t *__restrict__ codes, uint8_t *__restrict__ scales) {
    __shared__ float part[32];
    const uint32_t tpr = blockDim.x, warps = tpr >> 5;
    const uint32_t words = cpr * 8 / Mx<FMT>::kWord;
    const uint64_t row_bytes = (uint64_t)cpr * Mx<FMT>::kBits;
    for (uint64_t row0 = (uint64_t)blockIdx.x * blockDim.y; row0 < rows; row0 += (uint64_t)gridDim.x * blockDim.y) {
        const uint64_t row = row0 + threadIdx.y;
        const bool in = row < rows;
        const typename MxElem<TY>::type *xr = x + row * ldx;
        const typename MxElem<TY>::type *rr = residual ? residual + row * ldr : nullptr;
        typename MxElem<TY>::type *ro = residual_out ? residual_out + row * ldo : nullptr;
        float ss = 0.0f;
        float h[V > 0 ? V : 1][8];
        auto sum8 = [&](uint32_t c, float (&v)[8], bool live) {
            if (!live) {
#pragma unroll
                for (int i = 0; i < 8; i++) v[i] = 0.0f;
                return;
            }
            mx_load8<TY>(xr, 8 * c, cols, vec, v);
            if (rr) {
                float r[8];
                mx_load8<TY>(rr, 8 * c, cols, vec, r);
#pragma unroll
                for (int i = 0; i < 8; i++) v[i] = __fadd_rn(v[i], r[i]);
            }
        };
        if constexpr (V > 0) {
#pragma unroll
            for (int j = 0; j < V; j++) {
                const uint32_t c = threadIdx.x + j * tpr;
                sum8(c, h[j], in && c < cpr);
            }
#pragma unroll
            for (int j = 0; j < V; j++) {
                const uint32_t c = threadIdx.x + j * tpr;
                if (ro && in && 8 * c < cols) mx_store8<TY>(ro, 8 * c, cols, vec, h[j]);
#pragma unroll
                for (int i = 0; i < 8; i++) ss = __fmaf_rn(h[j][i], h[j][i], ss);
            }
        } else {
            for (uint32_t c = threadIdx.x; c < cpr; c += tpr) {
                sum8(c, h[0], in);
#pragma unroll
                for (int i = 0; i < 8; i++) ss = __fmaf_rn(h[0][i], h[0][i], ss);
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
        // whole warps walk the chunks (mx_quantize8 shuffles): the lanes behind the row hold zeros
        const int trips = V > 0 ? V : (int)((cpr + tpr - 1) / tpr);
#pragma unroll(V > 0 ? V : 1)
        for (int j = 0; j < trips; j++) {
            const uint32_t c = threadIdx.x + (uint32_t)j * tpr;
            const bool live = in && c < cpr;
            float(&v)[8] = h[V > 0 ? j : 0];
            if constexpr (V == 0) {
                sum8(c, v, live);
                if (ro && live && 8 * c < cols) mx_store8<TY>(ro, 8 * c, cols, vec, v);
            }
            float wt[8] = {0, 0, 0, 0, 0, 0, 0, 0};
            if (live) mx_load8<TY>(weight, 8 * c, cols, vec, wt);
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = live ? __fmul_rn(__fmul_rn(v[i], scale), wt[i]) : 0.0f;
            // columns behind `cols` stay zero even where the row's sum is not a number
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (8 * c + i >= cols) v[i] = 0.0f;
            mx_quantize8<FMT>(v, live, c, cr, sr, inv6g, g);
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

// What every entry here asks of its sizes: known format and type, columns that a 32-bit index
// holds after padding, rows whose chunks a 64-bit count holds.
static int mx_shape(int fmt, int ty, uint64_t rows, uint32_t cols) {
    if (!mx_known(fmt) || !mx_ty_known(ty)) return LYTH_E_UNSUPPORTED;
    if (cols == 0 || cols > (1u << 30) || rows > (1ull << 40)) return LYTH_E_INVALID;
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
    if (!aligned16(codes) || !aligned16(scales)) return LYTH_E_UNSUPPORTED;
    const uint32_t cpr = (uint32_t)(mx_padded(fmt, cols) / 8);
    const bool vec = aligned16(x) && ldx * mx_ty_bytes(ty) % 16 == 0;
    const unsigned grid = stream_grid(rows * cpr, kMxThreads);
    LYTH_MX_DISPATCH(fmt, ty,
                     mx_quantize_kernel<FMT, TY><<<grid, kMxThreads, 0, s>>>(
                         static_cast<const MxElem<TY>::type *>(x), rows, cols, ldx, cpr, vec, inv6g, tensor_scale,
                         codes, scales));
    return last_launch_status();
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
    if (!aligned16(codes) || !aligned16(scales)) return LYTH_E_UNSUPPORTED;
    const uint32_t cpr = (uint32_t)(mx_padded(fmt, cols) / 8);
    const bool vec = aligned16(out) && ldo * mx_ty_bytes(ty) % 16 == 0;
    const unsigned grid = stream_grid(rows * cpr, kMxThreads);
    LYTH_MX_DISPATCH(fmt, ty,
                     mx_dequantize_kernel<FMT, TY><<<grid, kMxThreads, 0, s>>>(
                         codes, scales, rows, cols, ldo, cpr, vec, tensor_scale, static_cast<MxElem<TY>::type *>(out)));
    return last_launch_status();
}

template <int FMT, int TY>
static void rmsnorm_launch(const void *x, const void *residual, void *residual_out, const void *weight, uint64_t rows,
                           uint32_t cols, uint64_t ldx, uint64_t ldr, uint64_t ldo, uint32_t cpr, bool vec, float eps,
                           float inv6g, float g, uint8_t *codes, uint8_t *scales, cudaStream_t s) {
    using T = typename MxElem<TY>::type;
    const T *xt = static_cast<const T *>(x), *rt = static_cast<const T *>(residual), *wt = static_cast<const T *>(weight);
    T *ot = static_cast<T *>(residual_out);
    const int v = cpr <= 1024 ? 1 : cpr <= 4096 ? 4 : 0;
    uint32_t tpr = v ? ((cpr + v - 1) / v + 31) / 32 * 32 : 1024;
    const uint32_t per = tpr < 256 ? 256 / tpr : 1;
    const dim3 block(tpr, per);
    const uint64_t need = (rows + per - 1) / per;
    const unsigned grid = need < (1u << 30) ? (unsigned)need : (1u << 30);
#define LYTH_MX_NORM(V)                                                                                            \
    mx_rmsnorm_kernel<FMT, TY, V><<<grid, block, 0, s>>>(xt, rt, ot, wt, rows, cols, ldx, ldr, ldo, cpr, vec, eps, \
                                                         inv6g, g, codes, scales)
    if (v == 1) LYTH_MX_NORM(1);
    else if (v == 4) LYTH_MX_NORM(4);
    else LYTH_MX_NORM(0);
#undef LYTH_MX_NORM
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
    if (!aligned16(codes) || !aligned16(scales)) return LYTH_E_UNSUPPORTED;
    const uint32_t cpr = (uint32_t)(mx_padded(fmt, cols) / 8);
    const uint64_t size = mx_ty_bytes(ty);
    const bool vec = aligned16(x) && ldx * size % 16 == 0 && aligned16(weight) &&
                     (!residual || (aligned16(residual) && ldr * size % 16 == 0)) &&
                     (!residual_out || (aligned16(residual_out) && ldo * size % 16 == 0));
    LYTH_MX_DISPATCH(fmt, ty,
                     rmsnorm_launch<FMT, TY>(x, residual, residual_out, weight, rows, cols, ldx, ldr, ldo, cpr, vec,
                                             eps, inv6g, tensor_scale, codes, scales, s));
    return last_launch_status();
}
