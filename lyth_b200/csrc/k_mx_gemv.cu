// y = alpha * x W^T for a few rows of 16-bit x against block-scaled weights (mx.cuh): the product's
// form for one to eight tokens, bound by reading W once.
//
// W's codes go to f16 (exact) and through m16n8k16 tensor-core steps with W as the 16-row operand: the
// tcgen05 path needs both operands quantised and 128 rows of x, here x keeps its 16 bits. A lane reads
// 16 bytes along k of two rows (a quad of lanes 64 contiguous bytes of a row), so the four lanes of a
// quad hold different scale blocks within one step. The n = 8 side separates them: its columns are
// (token, lane of the quad), and x stands only where the column's lane is the lane that holds those k,
// zero elsewhere. A column's sum then is one lane's part, of one scale block, and is multiplied by
// that block's scale in f32 afterwards: four multiply-adds for the 64 codes a lane holds. Tensor-core
// work is four times what the product needs and is idle capacity here.
//
// Range: bf16 x is brought into f16 by one power of two for all of x in the block (its largest finite
// exponent to 2^14), undone in f32 at the end. Values below 2^-38 of the largest lose bits, which is
// below the rounding of the f32 sum; every other bf16 value keeps all its bits.
#include "mx.cuh"

namespace lyth {

constexpr int XV_WARPS = 8, XV_THREADS = 32 * XV_WARPS, XV_ROWS = 16;

struct XvArgs {
    const void *x;
    const uint8_t *w, *s;
    void *y;
    uint64_t ldx, ldy;
    uint32_t m, n, cols;
    uint32_t row_bytes, words;  // bytes of a row of codes; scale words along k
    uint32_t iters;             // steps of 64 bytes along k
    uint32_t chunk;             // steps whose x is in shared memory at once
    float alpha;
    bool vec;                   // rows of x start on 16 bytes
};

LYTH_D void xv_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 bytes of codes as pairs of f16 in k order: 16 registers of E2M1, 8 of E4M3.
template <int FMT>
LYTH_D void xv_decode(const uint4 &u, uint32_t (&h)[FMT == LYTH_MX_FP8 ? 8 : 16]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (FMT == LYTH_MX_FP8) {
            e4m3x4_f16(w[i], h[2 * i], h[2 * i + 1]);
        } else {
            uint32_t q[4];
            e2m1x8_f16(w[i], q);
#pragma unroll
            for (int j = 0; j < 4; j++) h[4 * i + j] = q[j];
        }
    }
}

// Row i (0..15) of tile t: four neighbouring rows of each 32-row quarter of a scale tile, whose
// sixteen scale words are contiguous.
LYTH_D uint64_t xv_row(uint64_t t, uint32_t i) { return (t >> 3) * 128 + (i & 3) * 32 + (t & 7) * 4 + (i >> 2); }

// PAIRS: token pairs (1, 2 or 4).
template <int FMT, int TY, int PAIRS>
__global__ void __launch_bounds__(XV_THREADS) mx_gemv_kernel(XvArgs p) {
    using T = typename MxElem<TY>::type;
    constexpr int kCodes = FMT == LYTH_MX_FP8 ? 16 : 32;  // codes of a lane per step
    constexpr int kStep = 4 * kCodes;                     // columns of a step
    constexpr int kUnits = kCodes / 8;                    // 16-byte units of f16 x of a lane per step
    extern __shared__ uint4 sx[];                         // [2 PAIRS][chunk][4 lanes][kUnits]
    __shared__ float s_part[XV_WARPS][2 * PAIRS][XV_ROWS];
    __shared__ uint32_t s_max[XV_WARPS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t units = p.chunk * 4 * kUnits;          // per token

    // x to shared memory as f16. Units are stored with their low bits exchanged (lane of the quad,
    // token) so that the eight lanes reading at once reach eight different 16-byte columns.
    float unscale = 1.0f;
    float scale = 1.0f;
    if constexpr (TY == LYTH_NARROW_BF16) {
        uint32_t top = 0;
        const uint32_t all = (p.cols + 7) / 8;
        for (uint64_t i = threadIdx.x; i < (uint64_t)p.m * all; i += XV_THREADS) {
            float v[8];
            mx_load8<TY>(static_cast<const T *>(p.x) + i / all * p.ldx, 8 * (uint32_t)(i % all), p.cols, p.vec, v);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const uint32_t e = (__float_as_uint(v[j]) >> 23) & 0xFFu;
                if (e < 255u) top = max(top, e);
            }
        }
        top = __reduce_max_sync(0xFFFFFFFFu, top);
        if (lane == 0) s_max[warp] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < XV_WARPS; i++) top = max(top, s_max[i]);
        // 2^(14 - e) and its inverse, e the largest exponent; kept within normal f32 numbers
        const int e = (int)top - 127, sh = min(14 - e, 126);
        scale = __uint_as_float((uint32_t)(sh + 127) << 23);
        unscale = __uint_as_float((uint32_t)(127 - sh) << 23);
    }
    const uint64_t tile = blockIdx.x;
    const uint64_t r0 = xv_row(tile, g), r1 = xv_row(tile, g + 8);
    const bool in0 = r0 < p.n, in1 = r1 < p.n;
    const uint8_t *w0 = p.w + r0 * p.row_bytes + 16 * t, *w1 = p.w + r1 * p.row_bytes + 16 * t;
    const uint8_t *s0 = p.s + mx_scale_row(r0, p.words), *s1 = p.s + mx_scale_row(r1, p.words);
    const bool mine = (g & 3) == t;  // this lane's x columns: token g / 4 of each pair
    float acc[PAIRS][2] = {};
    for (uint32_t c0 = 0; c0 < p.iters; c0 += p.chunk) {
        if (c0) __syncthreads();
        for (uint32_t i = threadIdx.x; i < 2 * PAIRS * units; i += XV_THREADS) {
            const uint32_t tok = i / units, u = i % units, l = (u / kUnits) & 3;
            float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
            if (tok < p.m) mx_load8<TY>(static_cast<const T *>(p.x) + tok * p.ldx, 8 * (c0 * 4 * kUnits + u), p.cols, p.vec, v);
    #pragma unroll
            for (int j = 0; j < 8; j++) v[j] = __fmul_rn(v[j], scale);
            const uint32_t sw = (kUnits == 4 ? l : 0u) ^ (tok & 1);
            sx[tok * units + (u ^ sw)] = make_uint4(mx_pack2<LYTH_NARROW_F16>(v[0], v[1]), mx_pack2<LYTH_NARROW_F16>(v[2], v[3]),
                                                    mx_pack2<LYTH_NARROW_F16>(v[4], v[5]), mx_pack2<LYTH_NARROW_F16>(v[6], v[7]));
        }
        __syncthreads();
    const uint32_t c1 = min(c0 + p.chunk, p.iters);
    for (uint32_t it = c0 + warp; it < c1; it += XV_WARPS) {
        const bool ink = it * 64 + 16 * t < p.row_bytes;
        uint4 u0 = make_uint4(0, 0, 0, 0), u1 = u0;
        if (in0 && ink) u0 = __ldcs(reinterpret_cast<const uint4 *>(w0 + (uint64_t)it * 64));
        if (in1 && ink) u1 = __ldcs(reinterpret_cast<const uint4 *>(w1 + (uint64_t)it * 64));
        // the scale word that holds this lane's two columns' blocks
        const uint32_t word = FMT == LYTH_MX_FP8 ? it >> 1 : FMT == LYTH_MX_FP4 ? it : 2 * it + (t & 1);
        uint32_t q0 = 0, q1 = 0;
        if (word < p.words) {
            if (in0) q0 = *reinterpret_cast<const uint32_t *>(s0 + (uint64_t)word * 512);
            if (in1) q1 = *reinterpret_cast<const uint32_t *>(s1 + (uint64_t)word * 512);
        }
        uint32_t h0[kCodes / 2], h1[kCodes / 2];
        xv_decode<FMT>(u0, h0);
        xv_decode<FMT>(u1, h1);
#pragma unroll
        for (int pr = 0; pr < PAIRS; pr++) {
            uint32_t b[kCodes / 2];
            const uint32_t tok = 2 * pr + (g >> 2);
#pragma unroll
            for (int j = 0; j < kUnits; j++) {
                uint4 v = make_uint4(0, 0, 0, 0);
                if (mine) v = sx[tok * units + ((((it - c0) * 4 + t) * kUnits + j) ^ ((kUnits == 4 ? t : 0) ^ (tok & 1)))];
                b[4 * j] = v.x; b[4 * j + 1] = v.y; b[4 * j + 2] = v.z; b[4 * j + 3] = v.w;
            }
            constexpr int kSub = FMT == LYTH_MX_NVFP4 ? 2 : 1;  // scale blocks of a lane per step
            float c[kSub][4] = {};
#pragma unroll
            for (int j = 0; j < kCodes / 4; j++)
                xv_mma(c[j * kSub / (kCodes / 4)], h0[2 * j], h1[2 * j], h0[2 * j + 1], h1[2 * j + 1], b[2 * j], b[2 * j + 1]);
            // columns 2t, 2t + 1: token t / 2 of the pair, quad lanes 2 (t % 2) and the next
            if constexpr (FMT == LYTH_MX_NVFP4) {
                const float2 a0 = mx_scales2<FMT>(q0), a1 = mx_scales2<FMT>(q0 >> 16);
                const float2 b0 = mx_scales2<FMT>(q1), b1 = mx_scales2<FMT>(q1 >> 16);
                acc[pr][0] = __fmaf_rn(c[0][0], a0.x, acc[pr][0]);
                acc[pr][0] = __fmaf_rn(c[1][0], a0.y, acc[pr][0]);
                acc[pr][0] = __fmaf_rn(c[0][1], a1.x, acc[pr][0]);
                acc[pr][0] = __fmaf_rn(c[1][1], a1.y, acc[pr][0]);
                acc[pr][1] = __fmaf_rn(c[0][2], b0.x, acc[pr][1]);
                acc[pr][1] = __fmaf_rn(c[1][2], b0.y, acc[pr][1]);
                acc[pr][1] = __fmaf_rn(c[0][3], b1.x, acc[pr][1]);
                acc[pr][1] = __fmaf_rn(c[1][3], b1.y, acc[pr][1]);
            } else if constexpr (FMT == LYTH_MX_FP4) {
                const float2 a = mx_scales2<FMT>(q0 >> (16 * (t & 1))), bb = mx_scales2<FMT>(q1 >> (16 * (t & 1)));
                acc[pr][0] = __fmaf_rn(c[0][0], a.x, acc[pr][0]);
                acc[pr][0] = __fmaf_rn(c[0][1], a.y, acc[pr][0]);
                acc[pr][1] = __fmaf_rn(c[0][2], bb.x, acc[pr][1]);
                acc[pr][1] = __fmaf_rn(c[0][3], bb.y, acc[pr][1]);
            } else {
                const uint32_t sh = 16 * (it & 1) + 8 * (t & 1);  // both columns in one block of 32
                const float a = mx_scales2<FMT>((q0 >> sh) & 0xFFu).x, bb = mx_scales2<FMT>((q1 >> sh) & 0xFFu).x;
                acc[pr][0] = __fmaf_rn(c[0][0], a, acc[pr][0]);
                acc[pr][0] = __fmaf_rn(c[0][1], a, acc[pr][0]);
                acc[pr][1] = __fmaf_rn(c[0][2], bb, acc[pr][1]);
                acc[pr][1] = __fmaf_rn(c[0][3], bb, acc[pr][1]);
            }
        }
    }
    }
#pragma unroll
    for (int pr = 0; pr < PAIRS; pr++)
#pragma unroll
        for (int i = 0; i < 2; i++) {
            acc[pr][i] = __fadd_rn(acc[pr][i], __shfl_xor_sync(0xFFFFFFFFu, acc[pr][i], 1));
            if ((t & 1) == 0) s_part[warp][2 * pr + (t >> 1)][g + 8 * i] = acc[pr][i];
        }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < p.m * XV_ROWS; i += XV_THREADS) {
        const uint32_t tok = i / XV_ROWS, r = i % XV_ROWS;
        const uint64_t row = xv_row(tile, r);
        if (row >= p.n) continue;
        float v = 0.0f;
#pragma unroll
        for (int k = 0; k < XV_WARPS; k++) v = __fadd_rn(v, s_part[k][tok][r]);
        static_cast<T *>(p.y)[tok * p.ldy + row] = MxElem<TY>::round(__fmul_rn(p.alpha, __fmul_rn(v, unscale)));
    }
}

template <int FMT, int TY, int PAIRS>
static int xv_launch(XvArgs p, cudaStream_t s) {
    // x of one step takes 2 PAIRS x 4 lanes x kUnits x 16 bytes; 64 KiB of it at once
    const uint32_t step_bytes = 2 * PAIRS * (FMT == LYTH_MX_FP8 ? 8 : 16) * 16;
    const uint32_t most = 64 * 1024 / step_bytes;
    p.chunk = p.iters < most ? p.iters : most;
    const size_t smem = (size_t)p.chunk * step_bytes;
    if (smem > 40 * 1024) {
        const cudaError_t e =
            cudaFuncSetAttribute(mx_gemv_kernel<FMT, TY, PAIRS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return status_of(e);
    }
    const unsigned grid = (unsigned)((p.n + 127) / 128 * 8);
    mx_gemv_kernel<FMT, TY, PAIRS><<<grid, XV_THREADS, smem, s>>>(p);
    return last_launch_status();
}

template <int FMT, int TY>
static int xv_pairs(const XvArgs &p, cudaStream_t s) {
    if (p.m <= 2) return xv_launch<FMT, TY, 1>(p, s);
    if (p.m <= 4) return xv_launch<FMT, TY, 2>(p, s);
    return xv_launch<FMT, TY, 4>(p, s);
}

}  // namespace lyth

using namespace lyth;

extern "C" int lyth_b200_gemv_mx(int fmt, int ty, uint32_t m, uint32_t n, uint32_t cols, const void *x, uint64_t ldx,
                                 const uint8_t *w, const uint8_t *w_scales, float alpha, void *y, uint64_t ldy,
                                 cudaStream_t s) {
    if (!mx_known(fmt) || (ty != LYTH_NARROW_F16 && ty != LYTH_NARROW_BF16) || m > LYTH_GEMV_MX_MAX_M)
        return LYTH_E_UNSUPPORTED;
    if (cols == 0 || cols > (1u << 30) || n > (1u << 31) || ldx < cols || ldy < n) return LYTH_E_INVALID;
    if (m == 0 || n == 0) return LYTH_OK;
    if (!x || !w || !w_scales || !y) return LYTH_E_INVALID;
    if (!aligned16(w) || !aligned16(w_scales)) return LYTH_E_UNSUPPORTED;
    const uint64_t k = mx_padded(fmt, cols);
    XvArgs p;
    p.x = x;
    p.w = w;
    p.s = w_scales;
    p.y = y;
    p.ldx = ldx;
    p.ldy = ldy;
    p.m = m;
    p.n = n;
    p.cols = cols;
    p.row_bytes = (uint32_t)mx_code_bytes(fmt, k);
    p.words = (uint32_t)(k / (4 * mx_block(fmt)));
    p.iters = (p.row_bytes + 63) / 64;
    p.alpha = alpha;
    p.vec = aligned16(x) && ldx * 2 % 16 == 0;
    const bool bf = ty == LYTH_NARROW_BF16;
    switch (fmt) {
        case LYTH_MX_FP8: return bf ? xv_pairs<LYTH_MX_FP8, LYTH_NARROW_BF16>(p, s) : xv_pairs<LYTH_MX_FP8, LYTH_NARROW_F16>(p, s);
        case LYTH_MX_FP4: return bf ? xv_pairs<LYTH_MX_FP4, LYTH_NARROW_BF16>(p, s) : xv_pairs<LYTH_MX_FP4, LYTH_NARROW_F16>(p, s);
        default: return bf ? xv_pairs<LYTH_MX_NVFP4, LYTH_NARROW_BF16>(p, s) : xv_pairs<LYTH_MX_NVFP4, LYTH_NARROW_F16>(p, s);
    }
}
