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
// work is four times what the product needs and is idle capacity for one or two tokens.
//
// What bounds the arithmetic of those is the conversion of codes (two codes an instruction, at half the issue
// rate), so everything around it is kept off the warps that convert: one block per SM, in roles:
//   producers (4 warps)  bring a stage -- 16 rows of W, up to 2048 bytes of each, and their scale words --
//                        into a ring of shared-memory stages, four rows a warp: a bulk copy per row (one
//                        lane each) and 16-byte asynchronous copies of the scales, completion on an
//                        mbarrier. (One warp for all sixteen rows needed 2000 cycles to issue a stage.)
//   consumers (16 warps) put x into shared memory as f16 once. Two teams of eight then take every other
//                        stage, a warp every eighth 64-byte step of it, so that one team's waits and sums
//                        lie under the other's conversions (all sixteen on one stage: 11.5 us, with the
//                        teams 10.6). The partial sums of a group stay in shared memory, where all meet once
//                        at the end and add them up in a fixed order. Where x does not fit, k is walked
//                        in chunks, x staged chunk by chunk.
// At the 96 registers that 640 threads leave, every bf16 instance spills (16 to 72 bytes of stores), no f16 one.
// Every mbarrier wait is bounded (mbar.cuh); one that runs out sets the device error flag and the
// block winds down. Loading and converting in the same warps, with four steps of loads in flight in
// registers, took 13.2 us for one token through 14336 x 4096 NVFP4 weights: 9.5 us without the loads,
// 10.6 us without the arithmetic. Now: one token through 14336 x 4096 NVFP4 10.6 us (33 MB, 3.1 TB/s),
// MXFP8 13.5 (4.5 TB/s), four tokens 15, eight 25, where the tensor-core steps bound it. Eight tokens as
// the columns of one step, W's codes times their scales in f16, took 18.6 (this then 25.7), but a token's sum then had other
// roundings than alone; taken for every count it cost one token 12.7 instead of 11.1.
//
// Range: bf16 x is brought into f16 by a power of two for each step's columns (128, of E4M3 weights 64
// neighbouring values of a token; their largest exponent to 2^14) and taken back in f32. Of those values,
// ones below 2^-31 of the largest lose bits (eight bits end at f16's 2^-24); every other product is exact
// before the f32 sums. A step's sum is below 2^28 and a multiple of 2^-33. E8M0 scales reach 2^-127 and
// 2^127, so the sum times the scale could leave f32 where the product does not: the power of two that
// takes x back comes in two factors, 2^-30 .. 2^30 of it before the scale and the rest after, and then
// neither end is passed before the product passes it (one token through 14336 x 4096 MXFP8 13.2 us with one
// factor and with two, eight 25.4 and 26.6; four through 4096 x 14336 MXFP4 17.4 and 18.4). NVFP4's scales
// end at 448 and 2^-9: one factor does.
#include <atomic>

#include "mbar.cuh"
#include "mx.cuh"

namespace lyth {

__device__ int g_xv_error = 0;

constexpr int XV_WARPS = 16;                        // consumers
constexpr int XV_TEAM = XV_WARPS / 2;               // a team takes every other stage
constexpr uint32_t XV_STAGES = 4;                   // of the ring: even, since a team owns every other one
constexpr int XV_PRODUCERS = 4;                     // warps, one per quad of a group
constexpr int XV_THREADS = 32 * (XV_WARPS + XV_PRODUCERS);
// f32 factors per token and step that take bf16 x back: two of E8M0 formats (see above), f16 x none.
template <int FMT, int TY>
constexpr uint32_t kXvBack = TY != LYTH_NARROW_BF16 ? 0 : FMT == LYTH_MX_NVFP4 ? 1 : 2;
// Groups whose partial sums are kept before they are added up: all of a block's, up to this many.
template <int PAIRS>
constexpr int kXvBatch = PAIRS == 4 ? 4 : 8;

struct XvArgs {
    const void *x;
    const uint8_t *w, *s;
    void *y;
    uint64_t ldx, ldy;
    uint32_t m, n, cols;
    uint32_t quads_each, quads_more;  // quads of a block; blocks that have one more
    uint32_t row_bytes, words;        // bytes of a row of codes; scale words along k
    uint32_t seg, segs;               // bytes of a row in a stage; stages along k
    uint32_t seg_words, stage_bytes;  // scale words of a row in a stage; 16 rows (pitch seg + 64) and the words
    uint32_t chunk, xsteps;           // segments, and steps, whose x is in shared memory at once
    float alpha;
    bool vec;                         // rows of x start on 16 bytes
};

LYTH_D void xv_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 bytes of shared memory where `on`, else v as it was.
LYTH_D void xv_load_x(uint4 &v, uint32_t at, bool on) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %5, 0;\n\t@p ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
                 : "+r"(v.x), "+r"(v.y), "+r"(v.z), "+r"(v.w)
                 : "r"(at), "r"((uint32_t)on)
                 : "memory");
}

// The eight codes of unit j of 16 bytes as four pairs of f16, in k order.
template <int FMT>
LYTH_D void xv_decode(const uint4 &u, int j, uint32_t (&h)[4]) {
    if constexpr (FMT == LYTH_MX_FP8) {
        e4m3x4_f16(j == 0 ? u.x : u.z, h[0], h[1]);
        e4m3x4_f16(j == 0 ? u.y : u.w, h[2], h[3]);
    } else {
        e2m1x8_f16(j == 0 ? u.x : j == 1 ? u.y : j == 2 ? u.z : u.w, h);
    }
}

// Eight values of x as four words of 16-bit pairs, zero behind `cols`.
template <int TY>
LYTH_D uint4 xv_load8(const typename MxElem<TY>::type *row, uint32_t col, uint32_t cols, bool vec) {
    if (vec && col + 8 <= cols) return *reinterpret_cast<const uint4 *>(row + col);
    const uint16_t *h = reinterpret_cast<const uint16_t *>(row);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t c = col + 2 * i, a = c < cols ? h[c] : 0u, b = c + 1 < cols ? h[c + 1] : 0u;
        w[i] = a | b << 16;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
// The largest exponent field among eight bf16 values that are numbers.
LYTH_D uint32_t xv_top(uint4 u) {
    const uint32_t a = __vmaxu2(__vmaxu2(u.x & 0x7FFF7FFFu, u.y & 0x7FFF7FFFu), __vmaxu2(u.z & 0x7FFF7FFFu, u.w & 0x7FFF7FFFu));
    uint32_t top = max(a & 0xFFFFu, a >> 16) >> 7;
    if (top == 255u) {  // an infinity or a NaN among them: look at each
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
        top = 0;
        for (int i = 0; i < 4; i++) {
            const uint32_t lo = (w[i] >> 7) & 0xFFu, hi = (w[i] >> 23) & 0xFFu;
            if (lo < 255u) top = max(top, lo);
            if (hi < 255u) top = max(top, hi);
        }
    }
    return top;
}
// Eight bf16 values times a power of two, in f16.
LYTH_D uint4 xv_f16(uint4 u, float scale) {
    uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = mx_mul2(mx_unpack2<LYTH_NARROW_BF16>(w[i]), make_float2(scale, scale));
        w[i] = mx_pack2<LYTH_NARROW_F16>(f.x, f.y);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

LYTH_D bool xv_wait(uint32_t bar, uint32_t parity) { return mbar_wait_warp(bar, parity, &g_xv_error); }

// Where a block is in its walk: batches of groups, chunks of k, groups, segments. All roles take the
// same steps.
struct XvWalk {
    uint64_t tile0;          // first scale tile (128 rows) of the batch; rows and quads count from it
    uint32_t lo, hi, last;   // the batch's quads, and the last row of W
    uint32_t groups;         // of the batch
};
template <int BATCH>
LYTH_D bool xv_batch(const XvArgs &p, uint32_t index, XvWalk &w) {
    const uint64_t q_lo = (uint64_t)blockIdx.x * p.quads_each + min(blockIdx.x, p.quads_more);
    const uint64_t q_hi = q_lo + p.quads_each + (blockIdx.x < p.quads_more ? 1 : 0);
    const uint64_t b_lo = q_lo + (uint64_t)index * (4 * BATCH);
    if (b_lo >= q_hi) return false;
    w.tile0 = b_lo >> 5;
    w.lo = (uint32_t)b_lo & 31u;
    w.hi = w.lo + (uint32_t)min(q_hi - b_lo, (uint64_t)(4 * BATCH));
    w.last = (uint32_t)min((uint64_t)p.n - 1 - w.tile0 * 128, (uint64_t)511);
    w.groups = (w.hi - w.lo + 3) / 4;
    return true;
}
LYTH_D uint32_t xv_row(uint32_t quad, uint32_t j) { return (quad >> 5) * 128 + (quad & 31) + 32 * j; }

// U steps (it, it + XV_TEAM, ..) of a warp in the stage at `at`, independent of one another until
// their sums meet in acc: acc[pair][row g, row g + 8] of token t / 2 of the pair. `words`: scale words
// that the row still has from the stage on. x_step: of step `it` in shared x.
template <int FMT, int TY, int PAIRS, int U>
LYTH_D void xv_steps(const uint8_t *at, uint32_t pitch, uint32_t it, uint32_t x_step, uint32_t g, uint32_t t, bool mine,
                     const uint32_t (&x_at)[PAIRS], const float *const (&xs_at)[PAIRS], uint32_t words,
                     uint4 (&xb)[4], float (&acc)[PAIRS][2]) {
    constexpr int kUnits = FMT == LYTH_MX_FP8 ? 2 : 4, kSub = FMT == LYTH_MX_NVFP4 ? 2 : 1;
    uint4 u0[U], u1[U];
    uint32_t q0[U], q1[U];
    float cc[U][PAIRS][kSub][4] = {};
#pragma unroll
    for (int s = 0; s < U; s++) {
        const uint32_t i = it + s * XV_TEAM;
        u0[s] = *reinterpret_cast<const uint4 *>(at + g * pitch + i * 64 + t * 16);
        u1[s] = *reinterpret_cast<const uint4 *>(at + (g + 8) * pitch + i * 64 + t * 16);
        // the scale word that holds this lane's two columns' blocks
        const uint32_t word = FMT == LYTH_MX_FP8 ? i >> 1 : FMT == LYTH_MX_FP4 ? i : 2 * i + (t & 1);
        q0[s] = *reinterpret_cast<const uint32_t *>(at + 16 * pitch + word * 64 + g * 4);
        q1[s] = *reinterpret_cast<const uint32_t *>(at + 16 * pitch + word * 64 + g * 4 + 32);
        if (FMT == LYTH_MX_NVFP4 && word >= words) q0[s] = q1[s] = 0;  // a row may end in half a step
    }
#pragma unroll
    for (int j = 0; j < kUnits; j++) {
#pragma unroll
        for (int s = 0; s < U; s++) {
            uint32_t h0[4], h1[4];
            xv_decode<FMT>(u0[s], j, h0);
            xv_decode<FMT>(u1[s], j, h1);
#pragma unroll
            for (int pr = 0; pr < PAIRS; pr++) {
                uint4 &v = xb[(s * PAIRS + pr) % 4];
                xv_load_x(v, x_at[pr] + (x_step + s * XV_TEAM) * (4 * kUnits * 16) + 64 * j, mine);
                xv_mma(cc[s][pr][j * kSub / kUnits], h0[0], h1[0], h0[1], h1[1], v.x, v.y);
                xv_mma(cc[s][pr][j * kSub / kUnits], h0[2], h1[2], h0[3], h1[3], v.z, v.w);
            }
        }
    }
#pragma unroll
    for (int s = 0; s < U; s++) {
        const uint32_t i = it + s * XV_TEAM;
        // columns 2t, 2t + 1: token t / 2 of the pair, quad lanes 2 (t % 2) and the next
        float2 f0[kSub], f1[kSub];  // this lane's scales, rows g and g + 8
        if constexpr (FMT == LYTH_MX_NVFP4) {
            const float2 a0 = mx_scales2<FMT>(q0[s]), a1 = mx_scales2<FMT>(q0[s] >> 16);
            const float2 b0 = mx_scales2<FMT>(q1[s]), b1 = mx_scales2<FMT>(q1[s] >> 16);
            f0[0] = make_float2(a0.x, a1.x);
            f0[1] = make_float2(a0.y, a1.y);
            f1[0] = make_float2(b0.x, b1.x);
            f1[1] = make_float2(b0.y, b1.y);
        } else if constexpr (FMT == LYTH_MX_FP4) {
            f0[0] = mx_scales2<FMT>(q0[s] >> (16 * (t & 1)));
            f1[0] = mx_scales2<FMT>(q1[s] >> (16 * (t & 1)));
        } else {  // both columns in one block of 32
            const uint32_t sh = 16 * (i & 1) + 8 * (t & 1);
            f0[0].x = f0[0].y = mx_scales2<FMT>((q0[s] >> sh) & 0xFFu).x;
            f1[0].x = f1[0].y = mx_scales2<FMT>((q1[s] >> sh) & 0xFFu).x;
        }
#pragma unroll
        for (int pr = 0; pr < PAIRS; pr++) {
            if constexpr (TY == LYTH_NARROW_BF16) {  // the step's sum, then back from x's f16 range
                float d0 = 0.0f, d1 = 0.0f, xs;
                float2 c0[kSub], c1[kSub];
#pragma unroll
                for (int k = 0; k < kSub; k++) {
                    c0[k] = make_float2(cc[s][pr][k][0], cc[s][pr][k][1]);
                    c1[k] = make_float2(cc[s][pr][k][2], cc[s][pr][k][3]);
                }
                if constexpr (kXvBack<FMT, TY> == 2) {
                    const float2 back = reinterpret_cast<const float2 *>(xs_at[pr])[x_step + s * XV_TEAM];
                    c0[0] = mx_mul2(c0[0], make_float2(back.x, back.x));
                    c1[0] = mx_mul2(c1[0], make_float2(back.x, back.x));
                    xs = back.y;
                } else {
                    xs = xs_at[pr][x_step + s * XV_TEAM];
                }
#pragma unroll
                for (int k = 0; k < kSub; k++) {
                    d0 = __fmaf_rn(c0[k].x, f0[k].x, d0);
                    d1 = __fmaf_rn(c1[k].x, f1[k].x, d1);
                    d0 = __fmaf_rn(c0[k].y, f0[k].y, d0);
                    d1 = __fmaf_rn(c1[k].y, f1[k].y, d1);
                }
                acc[pr][0] = __fmaf_rn(d0, xs, acc[pr][0]);
                acc[pr][1] = __fmaf_rn(d1, xs, acc[pr][1]);
            } else {
#pragma unroll
                for (int k = 0; k < kSub; k++) {
                    acc[pr][0] = __fmaf_rn(cc[s][pr][k][0], f0[k].x, acc[pr][0]);
                    acc[pr][1] = __fmaf_rn(cc[s][pr][k][2], f1[k].x, acc[pr][1]);
                    acc[pr][0] = __fmaf_rn(cc[s][pr][k][1], f0[k].y, acc[pr][0]);
                    acc[pr][1] = __fmaf_rn(cc[s][pr][k][3], f1[k].y, acc[pr][1]);
                }
            }
        }
    }
}

// Rows come in quads r, r + 32, r + 64, r + 96 of a scale tile, whose four scale words are contiguous.
// Quad q's row in quarter j is 128 (q / 32) + q % 32 + 32 j. A block owns a contiguous range of quads
// (the rows divide over the SMs to 4) in groups of four. PAIRS: token pairs (1, 2, 4).
template <int FMT, int TY, int PAIRS>
__global__ void __launch_bounds__(XV_THREADS, 1) mx_gemv_kernel(const __grid_constant__ XvArgs p) {
    using T = typename MxElem<TY>::type;
    constexpr int kUnits = FMT == LYTH_MX_FP8 ? 2 : 4;    // 16-byte units of f16 x of a lane per step
    constexpr int kU = PAIRS == 4 ? 1 : 2;                // steps a warp takes at once
    constexpr int kTokens = 2 * PAIRS;
    extern __shared__ __align__(128) uint8_t sm[];        // ring, x, partial sums
    __shared__ uint64_t bars[2 * XV_STAGES + 1];
    const uint32_t warp = warp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    const uint32_t xunits = p.xsteps * 4 * kUnits;        // 16-byte units of x per token
    const uint32_t pitch = p.seg + 64;                    // of rows in a stage: eight read at once hit all banks
    uint4 *sx = reinterpret_cast<uint4 *>(sm + XV_STAGES * p.stage_bytes);
    constexpr uint32_t kBack = kXvBack<FMT, TY>;
    // of bf16 x: [token][step][factor]; of two factors an odd number of pairs, so that two tokens' lie in
    // different banks
    const uint32_t bpitch = kBack == 2 ? (p.xsteps | 1) * 2 : p.xsteps * kBack;
    float *s_scale = reinterpret_cast<float *>(sx + p.m * (xunits + 4));
    float *s_part = s_scale + p.m * bpitch;               // [group][warp][token][row]
    auto full = [&](uint32_t s) { return smem_u32(bars + s); };
    auto empty = [&](uint32_t s) { return smem_u32(bars + XV_STAGES + s); };
    const uint32_t xbar = smem_u32(bars + 2 * XV_STAGES); // the consumers' meeting point
    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < XV_STAGES; s++) {
            mbar_init(full(s), 33 * XV_PRODUCERS);  // the producers' lanes (scales) and counts of bytes (rows)
            mbar_init(empty(s), XV_TEAM);
        }
        mbar_init(xbar, XV_WARPS);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    grid_next();
    grid_wait();

    if (warp >= XV_WARPS) {  // ------------------------------------------------------------------ producers
        uint32_t stage = 0, phase = 0;
        bool ok = true;
        XvWalk w;
        for (uint32_t b = 0; ok && xv_batch<kXvBatch<PAIRS>>(p, b, w); b++) {
            const uint8_t *w_base = p.w + w.tile0 * 128 * p.row_bytes, *s_base = p.s + w.tile0 * p.words * 512;
            for (uint32_t c0 = 0; ok && c0 < p.segs; c0 += p.chunk) {
                const uint32_t c1 = min(c0 + p.chunk, p.segs);
                for (uint32_t group = 0; ok && group < w.groups; group++) {
                    // a warp per quad: one lane brings its four rows, all lanes its scale words
                    const uint32_t pw = warp - XV_WARPS, quad = w.lo + 4 * group + pw, row = xv_row(quad, 0);
                    const bool has = quad < w.hi;
                    const uint32_t rows = !has || row > w.last ? 0u : min((w.last - row) / 32 + 1, 4u);
                    const uint8_t *src = w_base + (uint64_t)row * p.row_bytes;
                    const uint8_t *ssrc = s_base + (uint64_t)(quad >> 5) * p.words * 512 + (quad & 31) * 16;
                    for (uint32_t seg = c0; seg < c1; seg++) {
                        if (!xv_wait(empty(stage), phase ^ 1)) { ok = false; break; }
                        const uint32_t bytes = min(p.row_bytes - seg * p.seg, p.seg);
                        const uint32_t at = smem_u32(sm) + stage * p.stage_bytes;
                        if (elect_one()) {
                            mbar_expect_tx(full(stage), rows * bytes);
#pragma unroll
                            for (uint32_t j = 0; j < 4; j++)
                                if (j < rows)
                                    bulk_load(at + (pw * 4 + j) * pitch, src + seg * p.seg + (uint64_t)j * 32 * p.row_bytes, bytes,
                                              full(stage));
                        }
                        __syncwarp();
                        const uint32_t w0 = seg * p.seg_words, nw = min(p.words - w0, p.seg_words);
                        if (has)
                            for (uint32_t i = lane; i < nw; i += 32)
                                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at + 16 * pitch + i * 64 + pw * 16),
                                             "l"(ssrc + (uint64_t)(w0 + i) * 512)
                                             : "memory");
                        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(full(stage)) : "memory");
                        if (++stage == XV_STAGES) { stage = 0; phase ^= 1; }
                    }
                }
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        ring_drain(stage, phase, XV_STAGES, [&](uint32_t s, uint32_t parity) { xv_wait(full(s), parity); });
    } else {  // ------------------------------------------------------------------------------- consumers
        const uint32_t g = lane >> 2, t = lane & 3;
        // x in shared memory: [token][step][unit][lane of the quad], tokens 64 bytes apart modulo 128, so
        // that the eight lanes reading at once (two tokens, four quad lanes) reach all 32 banks. Lanes
        // that hold no column keep zeros in xb: their loads are predicated off. Columns of tokens behind
        // m are token m - 1 again and are not stored.
        const bool mine = (g & 3) == t;
        uint4 xb[4] = {};
        uint32_t x_at[PAIRS];
#pragma unroll
        for (int pr = 0; pr < PAIRS; pr++)
            x_at[pr] = smem_u32(sx + min(2u * pr + (g >> 2), p.m - 1) * (xunits + 4) + t);
        const float *xs_at[PAIRS];  // of this lane's columns' token
#pragma unroll
        for (int pr = 0; pr < PAIRS; pr++) xs_at[pr] = s_scale + min(2u * pr + (t >> 1), p.m - 1) * bpitch;
        const T *x = static_cast<const T *>(p.x);
        uint32_t stage = 0, phase = 0;
        bool ok = true, staged = false;
        uint32_t xphase = 0;
        auto meet = [&]() {
            __syncwarp();
            if (lane == 0) mbar_arrive(xbar);
            const bool met = xv_wait(xbar, xphase);
            xphase ^= 1;
            return met;
        };
        XvWalk w;
        for (uint32_t b = 0; ok && xv_batch<kXvBatch<PAIRS>>(p, b, w); b++) {
            for (uint32_t c0 = 0; ok && c0 < p.segs; c0 += p.chunk) {
                if (!staged || p.chunk < p.segs) {
                    // (a bounded meeting: a warp that gave up a wait has left)
                    if (staged && !(ok = meet())) break;
                    const uint32_t first = c0 * (p.seg / 64) * 4 * kUnits;
                    // Units of x, token after token, four of a thread's loads in flight; whole warps, since a
                    // step's units (16, of E4M3 codes 8) lie in neighbouring lanes and share a power of two.
                    const uint32_t all = p.m * xunits;
#pragma unroll 1
                    for (uint32_t i0 = threadIdx.x; i0 - lane < all; i0 += 4 * 32 * XV_WARPS) {
                        uint4 v[4];
                        uint32_t tok[4], u[4];
#pragma unroll
                        for (int h = 0; h < 4; h++) {
                            const uint32_t i = i0 + h * 32 * XV_WARPS;
                            tok[h] = p.m == 1 ? 0u : i / xunits;
                            u[h] = i - tok[h] * xunits;
                            v[h] = make_uint4(0, 0, 0, 0);
                            if (i < all) v[h] = xv_load8<TY>(x + tok[h] * p.ldx, 8 * (first + u[h]), p.cols, p.vec);
                        }
#pragma unroll
                        for (int h = 0; h < 4; h++) {
                            const bool in = i0 + h * 32 * XV_WARPS < all;
                            const uint32_t owner = u[h] / kUnits;  // step and quad lane
                            if constexpr (TY == LYTH_NARROW_BF16) {
                                uint32_t top = xv_top(v[h]);
#pragma unroll
                                for (int o = 1; o < 4 * kUnits; o *= 2) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
                                // 2^(14 - e), e the largest exponent; it and its inverse, whole or in two
                                // factors, are normal f32 numbers
                                const int sh = min(14 - ((int)top - 127), 126);
                                v[h] = xv_f16(v[h], __uint_as_float((uint32_t)(127 + sh) << 23));
                                const int near = kBack == 2 ? max(-30, min(30, -sh)) : 0;
                                float *back = s_scale + tok[h] * bpitch + owner / 4 * kBack;
                                if (in && u[h] % (4 * kUnits) == 0) {
                                    if constexpr (kBack == 2) *back++ = __uint_as_float((uint32_t)(127 + near) << 23);
                                    *back = __uint_as_float((uint32_t)(127 - sh - near) << 23);
                                }
                            }
                            if (in) sx[tok[h] * (xunits + 4) + owner / 4 * (4 * kUnits) + u[h] % kUnits * 4 + owner % 4] = v[h];
                        }
                    }
                    if (!(ok = meet())) break;
                    staged = true;
                }
                const uint32_t c1 = min(c0 + p.chunk, p.segs);
                for (uint32_t group = 0; ok && group < w.groups; group++) {
                    float acc[PAIRS][2] = {};
                    for (uint32_t seg = c0; seg < c1; seg++) {
                        if ((stage & 1) != warp / XV_TEAM) {  // the other team's
                            if (++stage == XV_STAGES) { stage = 0; phase ^= 1; }
                            continue;
                        }
                        if (!xv_wait(full(stage), phase)) { ok = false; break; }
                        const uint8_t *at = sm + stage * p.stage_bytes;
                        const uint32_t steps = (min(p.row_bytes - seg * p.seg, p.seg) + 63) / 64;
                        const uint32_t words = p.words - seg * p.seg_words, x_base = (seg - c0) * (p.seg / 64);
                        uint32_t it = warp % XV_TEAM;
                        for (; it + (kU - 1) * XV_TEAM < steps; it += kU * XV_TEAM)
                            xv_steps<FMT, TY, PAIRS, kU>(at, pitch, it, x_base + it, g, t, mine, x_at, xs_at, words, xb, acc);
                        if constexpr (kU > 1)
                            for (; it < steps; it += XV_TEAM)
                                xv_steps<FMT, TY, PAIRS, 1>(at, pitch, it, x_base + it, g, t, mine, x_at, xs_at, words, xb, acc);
                        __syncwarp();
                        if (lane == 0) mbar_arrive(empty(stage));
                        if (++stage == XV_STAGES) { stage = 0; phase ^= 1; }
                    }
                    if (!ok) break;
                    // this warp's part of the group, of its own from chunk to chunk
                    float *part = s_part + (group * XV_WARPS + warp) * (kTokens * 16);
#pragma unroll
                    for (int pr = 0; pr < PAIRS; pr++)
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            const float v = __fadd_rn(acc[pr][i], __shfl_xor_sync(0xFFFFFFFFu, acc[pr][i], 1));
                            float *to = part + (2 * pr + (t >> 1)) * 16 + g + 8 * i;
                            if ((t & 1) == 0) *to = c0 ? __fadd_rn(*to, v) : v;
                        }
                }
            }
            if (!ok || !(ok = meet())) break;
#pragma unroll 1
            for (uint32_t i = threadIdx.x; i < w.groups * p.m * 16; i += 32 * XV_WARPS) {
                const uint32_t group = i / 16 % w.groups, tok = i / 16 / w.groups, r = i & 15;
                const uint32_t quad = w.lo + 4 * group + (r >> 2), row = xv_row(quad, r & 3);
                const float *part = s_part + (group * XV_WARPS * kTokens + tok) * 16 + r;
                float v = 0.0f;
#pragma unroll
                for (int k = 0; k < XV_WARPS; k++) v = __fadd_rn(v, part[k * kTokens * 16]);
                if (quad < w.hi && row <= w.last)
                    static_cast<T *>(p.y)[tok * p.ldy + w.tile0 * 128 + row] =
                        MxElem<TY>::round(__fmul_rn(p.alpha, v));
            }
            if (w.hi - w.lo == 4 * kXvBatch<PAIRS> && !(ok = meet())) break;  // before the next batch's sums
        }
    }
}

template <int FMT, int TY, int PAIRS>
static int xv_launch(XvArgs p, cudaStream_t s) {
    const uint32_t quads = p.n / 128 * 32 + (p.n % 128 < 32 ? p.n % 128 : 32u);
    const uint32_t sms = (uint32_t)device_sms(), grid = quads < sms ? quads : sms;
    p.quads_each = quads / grid;
    p.quads_more = quads % grid;
    // Shared memory: the partial sums, the ring, and as much of x as there is room for. A stage is 2048 bytes
    // a row; where all of x does not fit beside four of them, 1536 or 1024 (4 rows of x, 4096 x 14336 MXFP4:
    // 1536 15.9 us, six stages of 1024 18.7), and beyond that x is walked in chunks (at least a stage's: 8
    // tokens x 1024 E2M1 bytes are 32 KiB).
    const uint32_t groups = (p.quads_each + (p.quads_more ? 1 : 0) + 3) / 4;
    const size_t sums = (size_t)(groups < (uint32_t)kXvBatch<PAIRS> ? groups : kXvBatch<PAIRS>) * XV_WARPS * 2 * PAIRS * 16 * sizeof(float);
    const size_t step_x = (size_t)p.m * ((FMT == LYTH_MX_FP8 ? 8 : 16) * 16 + kXvBack<FMT, TY> * sizeof(float));
    const uint32_t steps = (p.row_bytes + 63) / 64;
    const size_t pads = p.m * (64 + (kXvBack<FMT, TY> == 2 ? 8 : 0)), room = 226 * 1024 - sums - pads;
    auto ring = [&](uint32_t seg) {
        p.seg = seg;
        p.segs = (p.row_bytes + seg - 1) / seg;
        p.seg_words = seg / 64 * 2 / (FMT == LYTH_MX_FP8 ? 4 : FMT == LYTH_MX_FP4 ? 2 : 1);
        p.stage_bytes = 16 * (seg + 64) + p.seg_words * 64;
        return (size_t)XV_STAGES * p.stage_bytes;
    };
    size_t held = ring(2048);
    if (held + steps * step_x > room) held = ring(1536);
    if (held + steps * step_x > room) held = ring(1024);
    p.chunk = held + steps * step_x <= room ? p.segs : (uint32_t)((room - held) / (p.seg / 64 * step_x));
    p.xsteps = p.chunk == p.segs ? steps : p.chunk * (p.seg / 64);
    const size_t smem = held + p.xsteps * step_x + pads + sums;
    static std::atomic<bool> set[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return status_of(e);
    if (dev < 0 || dev >= 64 || !set[dev]) {
        e = cudaFuncSetAttribute(mx_gemv_kernel<FMT, TY, PAIRS>, cudaFuncAttributeMaxDynamicSharedMemorySize, 226 * 1024);
        if (e != cudaSuccess) return status_of(e);
        if (dev >= 0 && dev < 64) set[dev] = true;
    }
    return mx_launch(mx_gemv_kernel<FMT, TY, PAIRS>, grid, XV_THREADS, smem, s, 1, p);
}

template <int FMT, int TY>
static int xv_pairs(const XvArgs &p, cudaStream_t s) {
    if (p.m <= 2) return xv_launch<FMT, TY, 1>(p, s);
    if (p.m <= 4) return xv_launch<FMT, TY, 2>(p, s);
    return xv_launch<FMT, TY, 4>(p, s);
}

int xv_take_device_error() {
    int v = 0;
    const cudaError_t e = cudaMemcpyFromSymbol(&v, g_xv_error, sizeof(int));
    if (e != cudaSuccess) return status_of(e);
    if (!v) return LYTH_OK;
    const int zero = 0;
    cudaMemcpyToSymbol(g_xv_error, &zero, sizeof(int));
    return LYTH_E_TIMEOUT;
}

}  // namespace lyth

using namespace lyth;

extern "C" int lyth_b200_gemv_mx(int fmt, int ty, uint32_t m, uint32_t n, uint32_t cols, const void *x, uint64_t ldx,
                                 const uint8_t *w, const uint8_t *w_scales, float alpha, void *y, uint64_t ldy,
                                 cudaStream_t s) {
    if (!mx_known(fmt) || (ty != LYTH_NARROW_F16 && ty != LYTH_NARROW_BF16) || m > LYTH_GEMV_MX_MAX_M)
        return LYTH_E_UNSUPPORTED;
    if (cols == 0 || cols > (1u << 24) || n > (1u << 31) || ldx < cols || ldy < n) return LYTH_E_INVALID;
    if (m == 0 || n == 0) return LYTH_OK;
    if (!x || !w || !w_scales || !y) return LYTH_E_INVALID;
    if (!aligned16(w) || !aligned16(w_scales) || !mx_elem_aligned(x, ty) || !mx_elem_aligned(y, ty))
        return LYTH_E_UNSUPPORTED;
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
    p.alpha = alpha;
    p.vec = aligned16(x) && ldx * 2 % 16 == 0;
    const bool bf = ty == LYTH_NARROW_BF16;
    switch (fmt) {
        case LYTH_MX_FP8: return bf ? xv_pairs<LYTH_MX_FP8, LYTH_NARROW_BF16>(p, s) : xv_pairs<LYTH_MX_FP8, LYTH_NARROW_F16>(p, s);
        case LYTH_MX_FP4: return bf ? xv_pairs<LYTH_MX_FP4, LYTH_NARROW_BF16>(p, s) : xv_pairs<LYTH_MX_FP4, LYTH_NARROW_F16>(p, s);
        default: return bf ? xv_pairs<LYTH_MX_NVFP4, LYTH_NARROW_BF16>(p, s) : xv_pairs<LYTH_MX_NVFP4, LYTH_NARROW_F16>(p, s);
    }
}
