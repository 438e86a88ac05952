// Product of two block-scaled matrices on the sm_100a tensor cores: C = alpha * A * B^T with A
// (m x k) and B (n x k) in one of mx.cuh's formats, f32 accumulation in tensor memory, C in f32,
// f16 or bf16. tcgen05.mma .block_scale multiplies the codes and applies both operands' block scales
// inside the contraction, so nothing is dequantised.
//
// Two forms, chosen by the number of 128 x 128 tiles: up to one per SM, single SMs whose clusters share k
// (mx_mma1_kernel); more, CTA pairs on tiles of 256 x 192 to 384 (mx_mma2_kernel). Both stage steps of 128 bytes
// along k (128 E4M3 or 256 E2M1 codes) of A and B in a shared-memory ring (TMA, 128-byte swizzle, no
// multicast) with both operands' scale tiles (512 bytes per 128 rows x 4 blocks, already in the order
// tensor memory wants), move the scales to tensor memory and issue one MMA per 32 bytes of k.
// Ragged edges: rows behind m or n arrive as zeros (tensor-map fill) or carry any scale, and are not
// stored; k is whole scale words, so the last step's MMAs are only fewer. Every wait is bounded.
#include <cuda.h>

#include <atomic>

#include "mbar.cuh"
#include "mx.cuh"

namespace lyth {

__device__ int g_mx_error = 0;

constexpr int XM_BM = 128, XM_BN = 128, XM_STAGES = 6;
constexpr int XM_OP_BYTES = 128 * 128;         // one operand's box: 128 rows x 128 bytes
constexpr int XM_TMEM_COLS = 512;              // the pair form: two accumulators, then the scales
constexpr int X1_TMEM_COLS = 256;              // the single-SM form: an accumulator, then the scales
constexpr uint32_t X1_PITCH = XM_BN + 4;

// Scale tiles (4 blocks along k) in one 128-byte step.
template <int FMT>
struct Xm {
    static constexpr int kTiles = FMT == LYTH_MX_FP8 ? 1 : FMT == LYTH_MX_FP4 ? 2 : 4;
    static constexpr int kStageBytes = 2 * XM_OP_BYTES + 2 * kTiles * 512;
    static constexpr size_t kSmem = 1024 + (size_t)XM_STAGES * kStageBytes + 256;
};

// Instruction descriptor of the block-scaled kinds: B scale id at bits 4-5, A type at 7-9, B type at
// 10-12 (E4M3 0 of mxf8f6f4, E2M1 1 of the 4-bit kinds), both operands K-major, N >> 3 at 17-22,
// scale type at 23 (E8M0 1, E4M3 0), M >> 7 at 27-28, A scale id at 29-30. The scale id says which
// bytes of the 32-bit scale cells an MMA uses: one (E4M3 codes), two, or all four (NVFP4).
template <int FMT>
LYTH_D uint32_t xm_idesc(int n, int m, int j) {
    const uint32_t ty = FMT == LYTH_MX_FP8 ? 0u : 1u;
    const uint32_t id = FMT == LYTH_MX_FP8 ? (uint32_t)j : FMT == LYTH_MX_FP4 ? (uint32_t)(j & 1) * 2u : 0u;
    return (id << 4) | (ty << 7) | (ty << 10) | ((uint32_t)(n >> 3) << 17) |
           ((FMT == LYTH_MX_NVFP4 ? 0u : 1u) << 23) | ((uint32_t)(m >> 7) << 27) | (id << 29);
}

// Every role is a whole warp in step: its lanes wait together, take one decision by vote, and one elected
// lane issues. The operands of TMA and MMA instructions then stay in uniform registers; a loop of a
// single lane (`if (lane == 0)`) had the compiler gather them for each instruction, 880 cycles for the
// four MMAs and two waits of a step and 550 for its four copies, which bound the kernels.
LYTH_D bool xm_wait(uint32_t bar, uint32_t parity) { return mbar_wait_warp(bar, parity, &g_mx_error); }
LYTH_D void xm_prefetch(const CUtensorMap *map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)map) : "memory");
}

// Shared-memory descriptor: K-major rows of 128 bytes with the 128-byte swizzle (8-row groups 1024
// bytes apart).
LYTH_D uint64_t xm_desc_op(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | 1ull << 16 | 64ull << 32 | 1ull << 46 | 2ull << 61;
}

template <int FMT>
LYTH_D void xm_mma(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t acc) {
#define LYTH_XM_MMA(KIND)                                                                                  \
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"                                         \
                 "tcgen05.mma.cta_group::1." KIND " [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),       \
                 "l"(da), "l"(db), "r"(idesc), "r"(sfa), "r"(sfb), "r"(acc)                                \
                 : "memory")
    if constexpr (FMT == LYTH_MX_FP8) LYTH_XM_MMA("kind::mxf8f6f4.block_scale.scale_vec::1X");
    else if constexpr (FMT == LYTH_MX_FP4) LYTH_XM_MMA("kind::mxf4.block_scale.scale_vec::2X");
    else LYTH_XM_MMA("kind::mxf4nvf4.block_scale.scale_vec::4X");
#undef LYTH_XM_MMA
}
LYTH_D void xm_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
LYTH_D void xm_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
LYTH_D void xm_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
LYTH_D void xm_tma(uint32_t dst, const CUtensorMap *map, int c0, int c1, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            dst),
        "l"((uint64_t)map), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
}
LYTH_D void xm_ld32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

struct XmArgs {
    const uint8_t *sa, *sb;  // scale tiles
    uint64_t m, n, ldc;
    uint32_t row_bytes;      // bytes of a row of codes
    uint32_t words;          // scale tiles along k
    float alpha;
    bool vec, vec4;          // rows of C start on 32 bytes; on four elements
};

// A lane's row of C, stored 32 columns at a time from left to right. Rows that start on 32 bytes are
// stored in 256-bit pieces, whole sectors. Others too: a lane shifts its row to the aligned pieces, the
// end of one chunk completing the next one's first piece; what is left of the first and of the last
// piece goes out in the few powers of two that make it up. 1500 x 5000 x 1000 MXFP4 to bf16, rows 16
// bytes off: 14.0 us, first and last bytes by elements 18.2, all through shared memory, so that sixteen
// lanes stored a row's neighbouring elements, 28.9; rows that start on 32 bytes 10.
struct XmRow {
    uint32_t held[8];  // the last chunk of 32 bytes, whose last `delta` bytes are not stored yet
    bool any = false;
};
// a where `on`, else b: in registers (the compiler makes an array in local memory of a chain of choices).
LYTH_D uint32_t xm_select(uint32_t on, uint32_t a, uint32_t b) {
    uint32_t r;
    asm("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %3, 0;\n\tselp.b32 %0, %1, %2, p;\n\t}" : "=r"(r) : "r"(a), "r"(b), "r"(on));
    return r;
}
// The aligned piece that ends `delta` bytes short of chunk w's end and starts with chunk h's last ones.
LYTH_D void xm_piece(const uint32_t (&h)[8], const uint32_t (&w)[8], uint32_t delta, uint32_t (&out)[8]) {
    uint32_t v[12];
#pragma unroll
    for (int i = 0; i < 12; i++) {
        const uint32_t lo = i < 8 ? h[i] : w[i - 8], hi = i < 4 ? h[i + 4] : w[i - 4];
        v[i] = (32 - delta) & 16 ? hi : lo;
    }
    mx_shift<8>(v, (32 - delta) & 15);
#pragma unroll
    for (int i = 0; i < 8; i++) out[i] = delta ? v[i] : w[i];
}
// The word of a piece that holds byte b.
LYTH_D uint32_t xm_word(const uint32_t (&w)[8], uint32_t b) {
    const uint32_t a0 = xm_select(b & 4, w[1], w[0]), a1 = xm_select(b & 4, w[3], w[2]);
    const uint32_t a2 = xm_select(b & 4, w[5], w[4]), a3 = xm_select(b & 4, w[7], w[6]);
    return xm_select(b & 16, xm_select(b & 8, a3, a2), xm_select(b & 8, a1, a0));
}
// Bytes from .. 31 of the piece at `at`.
LYTH_D void xm_store_end(char *at, const uint32_t (&w)[8], uint32_t from) {
    const uint32_t n = 32 - from;
    if (n & 2) {
        *reinterpret_cast<uint16_t *>(at + from) = (uint16_t)(xm_word(w, from) >> 16);
    }
    if (n & 4) {
        const uint32_t a = (from + 3) & ~3u;
        *reinterpret_cast<uint32_t *>(at + a) = xm_word(w, a);
    }
    if (n & 8) {
        const bool up = n >= 16;  // words 2 and 3, else 6 and 7
        *reinterpret_cast<uint2 *>(at + (up ? 8 : 24)) = up ? make_uint2(w[2], w[3]) : make_uint2(w[6], w[7]);
    }
    if (n & 16) *reinterpret_cast<uint4 *>(at + 16) = make_uint4(w[4], w[5], w[6], w[7]);
    if (n & 32) mx_st32(at, w);
}
// Bytes 0 .. n - 1 of the piece at `at`, n below 32.
LYTH_D void xm_store_start(char *at, const uint32_t (&w)[8], uint32_t n) {
    if (n & 16) *reinterpret_cast<uint4 *>(at) = make_uint4(w[0], w[1], w[2], w[3]);
    if (n & 8) {
        const bool up = n & 16;
        *reinterpret_cast<uint2 *>(at + (up ? 16 : 0)) = up ? make_uint2(w[4], w[5]) : make_uint2(w[0], w[1]);
    }
    if (n & 4) {
        const uint32_t a = n & ~7u;
        *reinterpret_cast<uint32_t *>(at + a) = xm_word(w, a);
    }
    if (n & 2) {
        const uint32_t a = n & ~3u;
        *reinterpret_cast<uint16_t *>(at + a) = (uint16_t)xm_word(w, a);
    }
}
// Columns col .. col + 31 of a warp's rows row0 .. (a row a lane), `last` of those that this warp stores.
template <int TY>
LYTH_D void xm_store32(typename MxElem<TY>::type *C, uint64_t row0, uint64_t col, const XmArgs &p, XmRow &h, bool last,
                       const uint32_t (&r)[32]) {
    constexpr uint32_t E = TY == 0 ? 4 : 2, kCols = 32 / E;
    const uint32_t lane = threadIdx.x & 31;
    if (col >= p.n || row0 + lane >= p.m) return;
    const uint32_t left = p.n - col < 32 ? (uint32_t)(p.n - col) : 32u;
    char *to = reinterpret_cast<char *>(C + (row0 + lane) * p.ldc + col);
    const uint32_t delta = (uint32_t)(reinterpret_cast<uintptr_t>(to) & 31u);
    uint32_t out[8];
#pragma unroll
    for (uint32_t q = 0; q < 32 / kCols; q++) {
        if (q * kCols >= left) break;
        uint32_t w[8];
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) {
            const uint32_t j = q * kCols + i * (4 / E);
            if constexpr (TY == 0) w[i] = __float_as_uint(__fmul_rn(p.alpha, __uint_as_float(r[j])));
            else w[i] = mx_pack2<TY>(__fmul_rn(p.alpha, __uint_as_float(r[j])), __fmul_rn(p.alpha, __uint_as_float(r[j + 1])));
        }
        const uint32_t bytes = min(left - q * kCols, kCols) * E;
        if (p.vec && bytes == 32) {
            mx_st32(to, w);
        } else {
            xm_piece(h.held, w, delta, out);
            if (bytes == 32) {
                if (h.any) mx_st32(to - delta, out);
                else xm_store_end(to - delta, out, delta);
#pragma unroll
                for (int i = 0; i < 8; i++) h.held[i] = w[i];
                h.any = true;
            } else {  // the row's end
                uint32_t n = delta + bytes;
                char *at = to - delta;
                if (h.any || delta == 0) {
                    if (n >= 32) {
                        mx_st32(at, out);
                        xm_piece(w, w, delta, out);
                        at += 32;
                        n -= 32;
                    }
                    xm_store_start(at, out, n);
                } else {  // and its start
#pragma unroll
                    for (uint32_t i = 0; i < 32; i += E) {
                        if (i < bytes) {
                            if constexpr (E == 4) *reinterpret_cast<uint32_t *>(to + i) = w[i / 4];
                            else *reinterpret_cast<uint16_t *>(to + i) = (uint16_t)(w[i / 4] >> (8 * (i & 2)));
                        }
                    }
                }
                h.any = false;
            }
        }
        to += 32;
    }
    if (h.any && (last || col + 32 >= p.n)) {
        xm_piece(h.held, h.held, delta, out);
        xm_store_start(to - delta, out, delta);
        h.any = false;
    }
}

// ---------------------------------------------------------------------------------------------
// The single-SM form, for products of at most one 128 x 128 tile per SM: a cluster of 1, 2 or 4 CTAs
// takes a tile, each a contiguous share of k, so that few tiles still fill the machine; their
// accumulators meet in shared memory and every CTA adds up a share of the columns over the cluster, in
// rank order. One token batch of 32 through 14336 x 4096 is 112 tiles; through 4096 x 14336, 32 tiles
// of four shares. NVFP4, 34 MB: 9.9 us, MXFP4 10.0, 3.4 TB/s; first copies and the epilogue are about four
// of them, and a quarter of the SMs have no tile.
//   warp 0     producer: boxes of A (only the rows that exist), B and both operands' scales.
//   warp 1     issues the MMAs.
//   warps 2-9  scales from shared to tensor memory as below, four warps the even steps and four the odd
//              (a step takes one set of four 600 cycles, the MMAs of it 260), then the epilogue.
constexpr int X1_SETS = 4, X1_THREADS = 320;

LYTH_D void x1_st4(uint32_t taddr, uint4 v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr), "r"(v.x), "r"(v.y),
                 "r"(v.z), "r"(v.w)
                 : "memory");
}
LYTH_D void xm_tma3(uint32_t dst, const CUtensorMap *map, int c0, int c1, int c2, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
        "[%5];" ::"r"(dst),
        "l"((uint64_t)map), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
        : "memory");
}

template <int FMT, int TY>
__global__ void __launch_bounds__(X1_THREADS, 1)
    mx_mma1_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                   const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSB,
                   typename MxElem<TY>::type *C, XmArgs p, uint32_t klog, uint32_t a_rows) {
    constexpr int T = Xm<FMT>::kTiles, S = XM_STAGES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *sA = smem, *sB = sA + S * XM_OP_BYTES, *sSA = sB + S * XM_OP_BYTES, *sSB = sSA + S * T * 512;
    uint64_t *bars = reinterpret_cast<uint64_t *>(sSB + S * T * 512);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * S + X1_SETS + 1);
    auto full = [&](int s) { return smem_u32(bars + s); };
    auto empty = [&](int s) { return smem_u32(bars + S + s); };
    auto sready = [&](int b) { return smem_u32(bars + 2 * S + b); };
    const uint32_t done = smem_u32(bars + 2 * S + X1_SETS);

    const int warp = (int)warp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    const uint32_t ks = 1u << klog, rank = blockIdx.x & (ks - 1), tile = blockIdx.x >> klog;
    const uint32_t tiles_m = (uint32_t)((p.m + XM_BM - 1) / XM_BM), tm = tile % tiles_m, tn = tile / tiles_m;
    const uint32_t all = (p.row_bytes + 127) / 128, k0 = all * rank / ks, k1 = all * (rank + 1) / ks;

    grid_next();
    if (threadIdx.x == 32) {
        xm_prefetch(&tmA);
        xm_prefetch(&tmB);
        xm_prefetch(&tmSA);
        xm_prefetch(&tmSB);
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < S; s++) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
        }
        for (int b = 0; b < X1_SETS; b++) mbar_init(sready(b), 4);  // the four warps of the step
        mbar_init(done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(X1_TMEM_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    xm_fence_before();
    __syncthreads();
    xm_fence_after();
    const uint32_t tmem_base = warp_uniform(*tmem_slot);
    grid_wait();
    bool ok = true;

    if (warp == 0) {
        uint32_t stage = 0, phase = 0;
        for (uint32_t kb = k0; kb < k1; kb++) {
            if (!xm_wait(empty(stage), phase ^ 1)) { ok = false; break; }
            if (elect_one()) {
                mbar_expect_tx(full(stage), a_rows * 128 + XM_OP_BYTES + 2 * T * 512);
                xm_tma3(smem_u32(sSA + stage * T * 512), &tmSA, 0, (int)(kb * T), (int)tm, full(stage));
                xm_tma3(smem_u32(sSB + stage * T * 512), &tmSB, 0, (int)(kb * T), (int)tn, full(stage));
                xm_tma(smem_u32(sA + stage * XM_OP_BYTES), &tmA, (int)(kb * 128), (int)(tm * XM_BM), full(stage));
                xm_tma(smem_u32(sB + stage * XM_OP_BYTES), &tmB, (int)(kb * 128), (int)(tn * XM_BN), full(stage));
            }
            __syncwarp();
            if (++stage == S) { stage = 0; phase ^= 1; }
        }
        ring_drain(stage, phase, S, [&](uint32_t s, uint32_t parity) { xm_wait(full(s), parity); });
    } else if (warp == 1) {
        uint32_t stage = 0, phase = 0, set = 0, sphase = 0;
        for (uint32_t kb = k0; kb < k1; kb++) {
            // the scale warps have seen this step's copies land (`full`) before they arrive here
            if (!xm_wait(sready(set), sphase)) { ok = false; break; }
            xm_fence_after();
            const uint32_t left = p.row_bytes - kb * 128;
            const int mmas = left < 128 ? (int)(left / 32) : 4;
            const uint32_t sfa = tmem_base + XM_BN + set * 8 * T, sfb = sfa + 4 * T;
            const uint64_t a = xm_desc_op(smem_u32(sA + stage * XM_OP_BYTES)), b = xm_desc_op(smem_u32(sB + stage * XM_OP_BYTES));
            if (elect_one()) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    if (j < mmas)  // 32 bytes of k on: two units of the descriptor's address
                        xm_mma<FMT>(tmem_base, a + 2 * j, b + 2 * j, xm_idesc<FMT>(XM_BN, XM_BM, j),
                                    sfa + 4 * (j * T / 4), sfb + 4 * (j * T / 4), ((kb - k0) | (uint32_t)j) != 0);
                }
                xm_commit(empty(stage));
                if (kb + 1 == k1) xm_commit(done);
            }
            __syncwarp();
            if (++stage == S) { stage = 0; phase ^= 1; }
            if (++set == X1_SETS) { set = 0; sphase ^= 1; }
        }
    } else {
        const uint32_t quad = (uint32_t)(warp & 3);  // the TMEM lane quadrant this warp may access
        const uint32_t half = (uint32_t)(warp - 2) >> 2;  // of the steps, then of the columns
        uint32_t stage = half, phase = 0, set = half, old = half, old_phase = 0;
        for (uint32_t kb = k0 + half; kb < k1; kb += 2) {
            if (!xm_wait(full(stage), phase)) { ok = false; break; }
            uint4 sa[T], sb[T];  // read while the set may still be in use
#pragma unroll
            for (int t = 0; t < T; t++) {
                sa[t] = *reinterpret_cast<const uint4 *>(sSA + (stage * T + t) * 512 + lane * 16);
                sb[t] = *reinterpret_cast<const uint4 *>(sSB + (stage * T + t) * 512 + lane * 16);
            }
            // the set is free once the MMAs of the step X1_SETS back, whose commit frees its stage, are done
            if (kb - k0 >= X1_SETS) {
                if (!xm_wait(empty(old), old_phase)) { ok = false; break; }
                if ((old += 2) >= S) { old -= S; old_phase ^= 1; }
            }
            xm_fence_after();
            const uint32_t at = tmem_base + ((quad * 32) << 16) + XM_BN + set * 8 * T;
#pragma unroll
            for (int t = 0; t < T; t++) {
                x1_st4(at + 4 * t, sa[t]);
                x1_st4(at + 4 * T + 4 * t, sb[t]);
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            xm_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(sready(set));
            if ((stage += 2) >= S) { stage -= S; phase ^= 1; }
            if ((set += 2) >= X1_SETS) set -= X1_SETS;
        }
        if (ok) ok = xm_wait(done, 0);
        xm_fence_after();
        // the accumulators: straight to C, or to shared memory (the ring, whose last MMA is done) for the
        // cluster's sum; rows of 132 floats keep a warp's 128-bit accesses apart
        const uint32_t r = quad * 32 + lane;
        float *mine = reinterpret_cast<float *>(smem) + r * X1_PITCH;
        if (ok && tm * (uint64_t)XM_BM + quad * 32 < p.m) {
            XmRow h;
#pragma unroll 1
            for (uint32_t c = 2 * half; c < 2 * half + 2; c++) {
                uint32_t v[32];
                xm_ld32(tmem_base + ((quad * 32) << 16) + c * 32, v);
                if (ks == 1) {
                    xm_store32<TY>(C, (uint64_t)tm * XM_BM + quad * 32, (uint64_t)tn * XM_BN + c * 32, p, h, c & 1, v);
                    __syncwarp();
                } else {
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        *reinterpret_cast<uint4 *>(mine + c * 32 + 4 * i) = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
                }
            }
        }
    }
    if (ks > 1) {
        cluster_sync_all();
        // this CTA's columns of the sum, over the cluster in rank order
        const uint32_t width = XM_BN >> klog, rows = (uint32_t)min((uint64_t)XM_BM, p.m - tm * (uint64_t)XM_BM);
        const uint32_t glog = 5 - klog, items = rows << glog;  // four columns an item
        // eight loads of a thread in flight: 8 / ks items from each of the ks CTAs
        for (uint32_t i0 = threadIdx.x; i0 < items; i0 += X1_THREADS << (3 - klog)) {
            float4 v[8];
#pragma unroll
            for (uint32_t q = 0; q < 8; q++) {
                const uint32_t i = i0 + (q >> klog) * X1_THREADS;
                if (i < items) {
                    const uint32_t at = smem_u32(smem) + ((i >> glog) * X1_PITCH + rank * width + (i & ((1u << glog) - 1)) * 4) * 4;
                    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                                 : "=f"(v[q].x), "=f"(v[q].y), "=f"(v[q].z), "=f"(v[q].w)
                                 : "r"(mapa_shared(at, q & (ks - 1)))
                                 : "memory");
                }
            }
            float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (uint32_t q = 0; q < 8; q++) {
                sum.x = __fadd_rn(sum.x, v[q].x);
                sum.y = __fadd_rn(sum.y, v[q].y);
                sum.z = __fadd_rn(sum.z, v[q].z);
                sum.w = __fadd_rn(sum.w, v[q].w);
                if ((q & (ks - 1)) == ks - 1) {
                    const uint32_t i = i0 + (q >> klog) * X1_THREADS;
                    if (i < items) {
                        const float f[4] = {__fmul_rn(p.alpha, sum.x), __fmul_rn(p.alpha, sum.y), __fmul_rn(p.alpha, sum.z),
                                            __fmul_rn(p.alpha, sum.w)};
                        const uint64_t n0 = (uint64_t)tn * XM_BN + rank * width + (i & ((1u << glog) - 1)) * 4;
                        typename MxElem<TY>::type *to = C + ((uint64_t)tm * XM_BM + (i >> glog)) * p.ldc + n0;
                        if (p.vec4 && n0 + 4 <= p.n) {
                            if constexpr (TY == 0) *reinterpret_cast<float4 *>(to) = make_float4(f[0], f[1], f[2], f[3]);
                            else *reinterpret_cast<uint2 *>(to) = make_uint2(mx_pack2<TY>(f[0], f[1]), mx_pack2<TY>(f[2], f[3]));
                        } else {
#pragma unroll
                            for (int j = 0; j < 4; j++)
                                if (n0 + j < p.n) to[j] = MxElem<TY>::round(f[j]);
                        }
                    }
                    sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                }
            }
        }
        cluster_sync_all();  // no CTA leaves while another reads its sums
    }
    xm_fence_before();
    __syncthreads();
    if (warp == 1) {
        xm_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(X1_TMEM_COLS)
                     : "memory");
    }
}

// ---------------------------------------------------------------------------------------------
// The 2-SM form: a CTA pair computes a 256 x 192 tile with tcgen05.mma.cta_group::2. Each CTA stages
// its 128 rows of A and 96 of the tile's 192 rows of B, so a 128-byte step moves 28 KiB into an SM for
// the work that takes the 128 x 128 form 42 KiB: at 4 bits it is this traffic that bounds, 47 bytes a
// cycle into an SM measured, not the tensor cores. 192 columns leave room in tensor memory for two
// accumulators (2 x 192) beside the sets of scales. NT = 1: the accumulators take turns, and the
// epilogue of a tile runs beside the next. NT = 2: a tile of 256 x 384 uses both, a third less traffic
// for the work, with the epilogue partly exposed. BN = 256: one accumulator of 256 columns, the epilogue
// exposed. Chosen by the rounds that each leaves (launch rule).
// Measured: 4096 x 14336 x 4096 NVFP4 105 us (4.6 PFLOP/s), MXFP4 99; 4096^3 NVFP4 34.5 us (4.0), MXFP4
// 33, MXFP8 57 (2.4 PFLOP/s).
//
//   both CTAs, warp 0    producer: its halves of A and B as boxes that complete on the leader's `full`
//                        barrier; its 128 rows' A scales and the B scales of all 192 columns (the pair's
//                        MMA reads them in each CTA's tensor memory) on its own `sfull`. No multicast.
//   both CTAs, warps 6-9 scales: from shared to tensor memory, each warp its 32-lane quadrant (the four
//                        quadrants hold the same scales), then an arrival on the leader's `sready`.
//                        tcgen05.cp does this without warps, but in the MMAs' queue: a copy of one tile
//                        took 60 cycles of it, twelve of them (NVFP4) twice the time of the step's MMAs.
//   leader, warp 1       issues the MMAs; one commit frees the stage, and the set of scales in tensor
//                        memory, in both CTAs.
//   both CTAs, warps 2-5 epilogue of this CTA's 128 rows.
// B scale tiles are 128 rows and a tile of 192 starts on a multiple of 64: two scale tiles cover it, and
// an odd start reads from two tensor-memory columns (64 rows) on.
constexpr int X2_THREADS = 320;

// BN: columns of an accumulator, 192 or 256. NT: accumulators of a tile.
template <int FMT, int NT, int BN>
struct X2 {
    static constexpr int kTiles = Xm<FMT>::kTiles;
    static constexpr int kAccs = BN == 192 ? 2 : 1;                  // accumulators in tensor memory
    static constexpr int kHalf = BN / 2, kBBytes = kHalf * 128;      // this CTA's rows of B for one accumulator
    static constexpr uint32_t kSfCol = kAccs * BN;                   // the scales' first column
    static constexpr int kBTiles = NT + 1;                           // of 128 rows, that hold the tile's columns
    static constexpr int kSfBytes = (1 + kBTiles) * kTiles * 512;
    static constexpr int kStageBytes = XM_OP_BYTES + NT * kBBytes + kSfBytes;
    static constexpr int kSetCols = 4 * kTiles * (1 + kBTiles);      // a step's scales in tensor memory
    static constexpr int kSets = (512 - kSfCol) / kSetCols < 4 ? (512 - kSfCol) / kSetCols : 4;
    static_assert(NT <= kAccs, "a tile's accumulators are held at once");
    static constexpr int kStages = (227 * 1024 - 1280) / kStageBytes;
    static constexpr size_t kSmem = 1280 + (size_t)kStages * kStageBytes;  // 256 bytes of barriers past the ring
    static_assert((3 * kStages + 4 + 4 + 1) * 8 <= 256, "barriers and the tensor-memory address");
};

LYTH_D void x2_tma2(uint32_t dst, const CUtensorMap *map, int c0, int c1, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
        "%3}], [%4];" ::"r"(dst),
        "l"((uint64_t)map), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
}
template <int FMT>
LYTH_D void x2_mma(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t acc) {
#define LYTH_X2_MMA(KIND)                                                                                  \
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"                                         \
                 "tcgen05.mma.cta_group::2." KIND " [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),       \
                 "l"(da), "l"(db), "r"(idesc), "r"(sfa), "r"(sfb), "r"(acc)                                \
                 : "memory")
    if constexpr (FMT == LYTH_MX_FP8) LYTH_X2_MMA("kind::mxf8f6f4.block_scale.scale_vec::1X");
    else if constexpr (FMT == LYTH_MX_FP4) LYTH_X2_MMA("kind::mxf4.block_scale.scale_vec::2X");
    else LYTH_X2_MMA("kind::mxf4nvf4.block_scale.scale_vec::4X");
#undef LYTH_X2_MMA
}
LYTH_D void x2_commit(uint32_t bar) {  // on this barrier in both CTAs
    const uint16_t mask = 3;
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
        "h"(mask)
        : "memory");
}

template <int FMT, int TY, int NT, int BN>
__global__ void __launch_bounds__(X2_THREADS, 1)
    mx_mma2_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                   const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSB,
                   typename MxElem<TY>::type *C, XmArgs p) {
    using L = X2<FMT, NT, BN>;
    constexpr int T = L::kTiles, S = L::kStages, kSets = L::kSets, NB = L::kBTiles;
    constexpr bool kTurns = NT < L::kAccs;  // tiles take the accumulators in turn
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *sA = smem, *sB = sA + S * XM_OP_BYTES, *sSA = sB + S * NT * L::kBBytes, *sSB = sSA + S * T * 512;
    uint64_t *bars = reinterpret_cast<uint64_t *>(sSB + S * NB * T * 512);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 3 * S + 4 + 4);
    auto full = [&](int s) { return smem_u32(bars + s); };
    auto empty = [&](int s) { return smem_u32(bars + S + s); };
    auto sfull = [&](int s) { return smem_u32(bars + 2 * S + s); };
    auto tfull = [&](int b) { return smem_u32(bars + 3 * S + b); };
    auto tempty = [&](int b) { return smem_u32(bars + 3 * S + 2 + b); };
    auto sready = [&](int b) { return smem_u32(bars + 3 * S + 4 + b); };

    const int warp = (int)warp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    const uint32_t crank = blockIdx.x & 1, pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;  // clusters of 2 along x
    const uint64_t tiles_m = (p.m + 255) / 256, tiles_n = (p.n + NT * BN - 1) / (NT * BN), ntiles = tiles_m * tiles_n;
    const uint32_t steps = (p.row_bytes + 127) / 128;

    grid_next();
    if (threadIdx.x == 32) {
        xm_prefetch(&tmA);
        xm_prefetch(&tmB);
        xm_prefetch(&tmSA);
        xm_prefetch(&tmSB);
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < S; s++) {
            mbar_init(full(s), 2);  // the two producers' arrivals (the leader's barrier is the one used)
            mbar_init(empty(s), 1);
            mbar_init(sfull(s), 1);
        }
        for (int b = 0; b < kSets; b++) mbar_init(sready(b), 8);  // four scale warps in each CTA (the leader's)
        for (int b = 0; b < 2; b++) {
            mbar_init(tfull(b), 1);
            mbar_init(tempty(b), 8);  // four epilogue warps in each CTA (the leader's is the one used)
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(XM_TMEM_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    xm_fence_before();
    cluster_sync_all();
    xm_fence_after();
    const uint32_t tmem_base = warp_uniform(*tmem_slot);
    grid_wait();

    if (warp == 0) {
        uint32_t stage = 0, phase = 0;
        bool ok = true;
        const uint32_t lead = warp_uniform(mapa_shared(full(0), 0));  // the leader's `full` barriers
        for (uint64_t tile = pair; tile < ntiles && ok; tile += npairs) {
            const uint32_t tm = (uint32_t)(tile % tiles_m), tn = (uint32_t)(tile / tiles_m);
            const int m0 = (int)(tm * 256 + 128 * crank), n0 = (int)(tn * (NT * BN));
            for (uint32_t kb = 0; kb < steps; kb++) {
                if (!xm_wait(empty(stage), phase ^ 1)) { ok = false; break; }
                const uint32_t lf = lead + 8 * stage;
                if (elect_one()) {
                    mbar_expect_tx(sfull(stage), L::kSfBytes);
                    xm_tma3(smem_u32(sSA + stage * T * 512), &tmSA, 0, (int)(kb * T), m0 >> 7, sfull(stage));
                    xm_tma3(smem_u32(sSB + stage * NB * T * 512), &tmSB, 0, (int)(kb * T), n0 >> 7, sfull(stage));
                    mbar_expect_tx_cluster(lf, XM_OP_BYTES + NT * L::kBBytes);
                    x2_tma2(smem_u32(sA + stage * XM_OP_BYTES), &tmA, (int)(kb * 128), m0, lf);
#pragma unroll
                    for (int h = 0; h < NT; h++)
                        x2_tma2(smem_u32(sB + (stage * NT + h) * L::kBBytes), &tmB, (int)(kb * 128),
                                n0 + h * BN + L::kHalf * (int)crank, lf);
                }
                __syncwarp();
                if (++stage == S) { stage = 0; phase ^= 1; }
            }
        }
        // This CTA's scale copies; its halves of A and B are waited for on the leader's barriers, by the
        // warp that issues the MMAs.
        ring_drain(stage, phase, S, [&](uint32_t s, uint32_t parity) { xm_wait(sfull(s), parity); });
        // Tail: every stage released by the MMA's commit, so no arrival is still on its way to this
        // CTA's barriers when it leaves.
        if (ok)
            for (int s = 0; s < S; s++) {
                if (!xm_wait(empty(stage), phase ^ 1)) break;
                if (++stage == S) { stage = 0; phase ^= 1; }
            }
    } else if (warp == 1) {
        if (crank == 0) {
            uint32_t stage = 0, phase = 0, local = 0, set = 0, sphase = 0;
            bool ok = true;
            for (uint64_t tile = pair; tile < ntiles && ok; tile += npairs, local++) {
                // one accumulator a tile, in turn; or both
                const uint32_t ab = kTurns ? local & 1 : 0u, aphase = kTurns ? (local >> 1) & 1 : local & 1;
                const uint32_t shift = kTurns ? ((uint32_t)(tile / tiles_m) & 1) * 2 : 0u;  // 192 tn is 64 mod 128
                for (uint32_t kb = 0; kb < steps; kb++) {
                    if (!xm_wait(full(stage), phase) || !xm_wait(sready(set), sphase)) { ok = false; break; }
                    const uint32_t left = p.row_bytes - kb * 128;
                    const int mmas = left < 128 ? (int)(left / 32) : 4;
                    const uint32_t sfa = tmem_base + L::kSfCol + set * L::kSetCols, sfb = sfa + 4 * T + shift;
                    const uint64_t a = xm_desc_op(smem_u32(sA + stage * XM_OP_BYTES));
                    const uint64_t b = xm_desc_op(smem_u32(sB + stage * NT * L::kBBytes));
#pragma unroll
                    for (int h = 0; h < NT; h++) {
                        if (kb == 0 && !xm_wait(tempty(ab + h), aphase ^ 1)) { ok = false; break; }
                        xm_fence_after();
                        if (elect_one()) {
#pragma unroll
                            for (int j = 0; j < 4; j++) {
                                if (j < mmas)  // columns 192 h on: six words of scales
                                    x2_mma<FMT>(tmem_base + (ab + h) * BN, a + 2 * j, b + h * (L::kBBytes / 16) + 2 * j,
                                                xm_idesc<FMT>(BN, 256, j), sfa + 4 * (j * T / 4),
                                                sfb + 4 * NB * (j * T / 4) + 6 * h, (kb | (uint32_t)j) != 0);
                            }
                            if (h == NT - 1) x2_commit(empty(stage));
                            if (kb + 1 == steps) x2_commit(tfull(ab + h));
                        }
                        __syncwarp();
                    }
                    if (!ok) break;
                    if (++stage == S) { stage = 0; phase ^= 1; }
                    if (++set == kSets) { set = 0; sphase ^= 1; }
                }
            }
            // After a timed-out wait, give the stages the producers may have in flight a bounded
            // chance to land (both CTAs' copies complete on these barriers) before the pair leaves.
            if (!ok) {
                for (int s = 0; s < S; s++) {
                    xm_wait(full(stage), phase);
                    if (++stage == S) { stage = 0; phase ^= 1; }
                }
            }
        }
    } else if (warp >= 6) {
        const uint32_t quad = (uint32_t)(warp & 3);  // the TMEM lane quadrant this warp may write
        uint32_t stage = 0, phase = 0, set = 0, lead[kSets];
        for (int b = 0; b < kSets; b++) lead[b] = mapa_shared(sready(b), 0);
        uint32_t step = 0, old = 0, old_phase = 0;  // steps so far; the stage and phase of the one kSets back
        bool ok = true;
        for (uint64_t tile = pair; tile < ntiles && ok; tile += npairs) {
            for (uint32_t kb = 0; kb < steps; kb++) {
                if (!xm_wait(sfull(stage), phase)) { ok = false; break; }
                // a tile is 16 bytes a lane: its words of four columns; read while the set may still be in use
                const uint8_t *a = sSA + stage * T * 512 + lane * 16, *b = sSB + stage * NB * T * 512 + lane * 16;
                uint4 sa[T], sb[T][NB];
#pragma unroll
                for (int t = 0; t < T; t++) {
                    sa[t] = *reinterpret_cast<const uint4 *>(a + t * 512);
#pragma unroll
                    for (int h = 0; h < NB; h++) sb[t][h] = *reinterpret_cast<const uint4 *>(b + (h * T + t) * 512);
                }
                // the set is free once the MMAs of the step kSets back, whose commit frees its stage, are done
                if (step >= (uint32_t)kSets) {
                    if (!xm_wait(empty(old), old_phase)) { ok = false; break; }
                    if (++old == S) { old = 0; old_phase ^= 1; }
                } else {
                    step++;
                }
                xm_fence_after();
                const uint32_t at = tmem_base + ((quad * 32) << 16) + L::kSfCol + set * L::kSetCols;
#pragma unroll
                for (int t = 0; t < T; t++) {
                    x1_st4(at + 4 * t, sa[t]);
#pragma unroll
                    for (int h = 0; h < NB; h++) x1_st4(at + 4 * T + 4 * NB * t + 4 * h, sb[t][h]);
                }
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                xm_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(lead[set]);
                if (++stage == S) { stage = 0; phase ^= 1; }
                if (++set == kSets) set = 0;
            }
        }
    } else {
        const uint32_t quad = (uint32_t)(warp & 3);  // the TMEM lane quadrant this warp may read
        const uint32_t lead_tempty[2] = {mapa_shared(tempty(0), 0), mapa_shared(tempty(1), 0)};
        uint32_t local = 0;
        bool ok = true;
        for (uint64_t tile = pair; tile < ntiles && ok; tile += npairs, local++) {
            const uint64_t row0 = tile % tiles_m * 256 + 128 * crank + quad * 32, n0 = tile / tiles_m * (NT * BN);
#pragma unroll 1
            for (uint32_t h = 0; h < NT; h++) {
                const uint32_t ab = kTurns ? local & 1 : h, aphase = kTurns ? (local >> 1) & 1 : local & 1;
                if (!xm_wait(tfull(ab), aphase)) { ok = false; break; }
                xm_fence_after();
                XmRow held;
#pragma unroll 1
                for (int c = 0; c < BN / 32; c++) {
                    uint32_t r[32];
                    xm_ld32(tmem_base + ab * BN + ((quad * 32) << 16) + c * 32, r);
                    xm_store32<TY>(C, row0, n0 + h * BN + c * 32, p, held, c + 1 == BN / 32, r);
                    __syncwarp();
                }
                xm_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(lead_tempty[ab]);
            }
        }
    }
    __syncwarp();
    xm_fence_before();
    cluster_sync_all();
    if (warp == 1) {
        xm_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(XM_TMEM_COLS)
                     : "memory");
    }
}

// Codes as a 2-D byte tensor: a 128-byte (the swizzle span) x box_rows box, zeros outside.
static bool xm_map(CUtensorMap *map, const void *base, uint64_t row_bytes, uint64_t rows, uint32_t box_rows) {
    PFN_encode_tiled enc = tensor_map_encoder();
    if (!enc) return false;
    cuuint64_t dims[2] = {row_bytes, rows};
    cuuint64_t strides[1] = {row_bytes};
    cuuint32_t box[2] = {128, box_rows};
    cuuint32_t estr[2] = {1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Scale tiles as a 3-D tensor of words: 128 (512 bytes) x tiles along k x tiles of 128 rows.
static bool xm_map_sf(CUtensorMap *map, const void *base, uint64_t words, uint64_t rows, uint32_t box_words,
                      uint32_t box_tiles) {
    PFN_encode_tiled enc = tensor_map_encoder();
    if (!enc) return false;
    cuuint64_t dims[3] = {128, words, (rows + 127) / 128};
    cuuint64_t strides[2] = {512, words * 512};
    cuuint32_t box[3] = {128, box_words, box_tiles};
    cuuint32_t estr[3] = {1, 1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, const_cast<void *>(base), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int FMT, int TY, int NT, int BN>
static int x2_launch(const uint8_t *a, const uint8_t *b, void *c, const XmArgs &p, cudaStream_t s) {
    using L = X2<FMT, NT, BN>;
    constexpr int T = L::kTiles;
    CUtensorMap ta, tb, tsa, tsb;
    if (!xm_map(&ta, a, p.row_bytes, p.m, 128) || !xm_map(&tb, b, p.row_bytes, p.n, L::kHalf) ||
        !xm_map_sf(&tsa, p.sa, p.words, p.m, T, 1) || !xm_map_sf(&tsb, p.sb, p.words, p.n, T, L::kBTiles))
        return LYTH_E_UNSUPPORTED;
    static std::atomic<int> fit_of[64];  // pairs resident at once, asked once per device (0: not yet)
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return status_of(e);
    int pairs = dev >= 0 && dev < 64 ? fit_of[dev].load() : 0;
    if (pairs == 0) {
        pairs = device_sms() / 2;
        e = cudaFuncSetAttribute(mx_mma2_kernel<FMT, TY, NT, BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::kSmem);
        if (e != cudaSuccess) return status_of(e);
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 2;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cudaLaunchConfig_t cfg = {};
        cfg.blockDim = dim3(X2_THREADS);
        cfg.dynamicSmemBytes = L::kSmem;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        cfg.gridDim = dim3(2u * (unsigned)pairs);
        int fit = 0;
        if (cudaOccupancyMaxActiveClusters(&fit, mx_mma2_kernel<FMT, TY, NT, BN>, &cfg) != cudaSuccess || fit < 1) fit = pairs;
        cudaGetLastError();
        if (fit < pairs) pairs = fit;
        if (dev >= 0 && dev < 64) fit_of[dev] = pairs;
    }
    const uint64_t tiles = (p.m + 255) / 256 * ((p.n + NT * BN - 1) / (NT * BN));
    if ((uint64_t)pairs > tiles) pairs = (int)tiles;
    return mx_launch(mx_mma2_kernel<FMT, TY, NT, BN>, 2u * (unsigned)pairs, X2_THREADS, L::kSmem, s, 2, ta, tb, tsa, tsb,
                               static_cast<typename MxElem<TY>::type *>(c), p);
}

template <int FMT, int TY>
static int x1_launch(const uint8_t *a, const uint8_t *b, void *c, const XmArgs &p, cudaStream_t s) {
    constexpr int T = Xm<FMT>::kTiles;
    const uint32_t a_rows = p.m < 128 ? ((uint32_t)p.m + 7) / 8 * 8 : 128u;
    CUtensorMap ta, tb, tsa, tsb;
    if (!xm_map(&ta, a, p.row_bytes, p.m, a_rows) || !xm_map(&tb, b, p.row_bytes, p.n, XM_BN) ||
        !xm_map_sf(&tsa, p.sa, p.words, p.m, T, 1) || !xm_map_sf(&tsb, p.sb, p.words, p.n, T, 1))
        return LYTH_E_UNSUPPORTED;
    static std::atomic<bool> done[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return status_of(e);
    if (dev < 0 || dev >= 64 || !done[dev]) {
        e = cudaFuncSetAttribute(mx_mma1_kernel<FMT, TY>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Xm<FMT>::kSmem);
        if (e != cudaSuccess) return status_of(e);
        if (dev >= 0 && dev < 64) done[dev] = true;
    }
    // shares of k: as many as keep every SM to one CTA and a share at least four steps long, four at most
    // (100 x 512 x 8192 NVFP4, 4 tiles: 11.7, 10.3, 8.5 and, with eight, 8.9 us; 16 x 1024 x 1024, four
    // steps: 4.4 us whole, 5.0 in two)
    const uint32_t tiles = (uint32_t)((p.m + XM_BM - 1) / XM_BM * ((p.n + XM_BN - 1) / XM_BN));
    const uint32_t steps = (p.row_bytes + 127) / 128;
    uint32_t klog = 0;
    while (klog < 2 && tiles << (klog + 1) <= (uint32_t)device_sms() && steps >> (klog + 1) >= 4) klog++;
    return mx_launch(mx_mma1_kernel<FMT, TY>, tiles << klog, X1_THREADS, Xm<FMT>::kSmem, s, 1u << klog, ta, tb, tsa,
                               tsb, static_cast<typename MxElem<TY>::type *>(c), p, klog, a_rows);
}

int mx_take_device_error() {
    int v = 0;
    const cudaError_t e = cudaMemcpyFromSymbol(&v, g_mx_error, sizeof(int));
    if (e != cudaSuccess) return status_of(e);
    if (!v) return LYTH_OK;
    const int zero = 0;
    cudaMemcpyToSymbol(g_mx_error, &zero, sizeof(int));
    return LYTH_E_TIMEOUT;
}

}  // namespace lyth

using namespace lyth;

extern "C" int lyth_b200_matmul_mx(int fmt, int ty, uint32_t m, uint32_t n, uint32_t cols, const uint8_t *a,
                                   const uint8_t *a_scales, const uint8_t *b, const uint8_t *b_scales, float alpha,
                                   void *c, uint64_t ldc, cudaStream_t s) {
    if (!mx_known(fmt) || !mx_ty_known(ty)) return LYTH_E_UNSUPPORTED;
    if (cols == 0 || cols > (1u << 30) || m > 0x7FFFFE00u || n > 0x7FFFFE00u || ldc < n) return LYTH_E_INVALID;
    if (m == 0 || n == 0) return LYTH_OK;
    if (!a || !a_scales || !b || !b_scales || !c) return LYTH_E_INVALID;
    if (!aligned16(a) || !aligned16(a_scales) || !aligned16(b) || !aligned16(b_scales) || !mx_elem_aligned(c, ty))
        return LYTH_E_UNSUPPORTED;
    const uint64_t k = mx_padded(fmt, cols);
    XmArgs p;
    p.sa = a_scales;
    p.sb = b_scales;
    p.m = m;
    p.n = n;
    p.ldc = ldc;
    p.row_bytes = (uint32_t)mx_code_bytes(fmt, k);
    p.words = (uint32_t)(k / (4 * mx_block(fmt)));
    p.alpha = alpha;
    p.vec = aligned32(c) && ldc * mx_ty_bytes(ty) % 32 == 0;
    p.vec4 = ((uintptr_t)c & (4 * mx_ty_bytes(ty) - 1)) == 0 && ldc % 4 == 0;
    // one tile per SM at most: single SMs, else pairs. us on single SMs and on pairs, NVFP4, k 4096: 32 x 18944
    // (148 tiles) 10.3 and 13.6, 32 x 19072 (149) 15.7 and 15.0; 1024 x 2304 (144) 7.7 and 9.9, 1024 x 2432 (152)
    // 13.8 and 9.7. (Where few rows fill a second round of single SMs well it is the other way: 32 x 28672 x
    // 8192, 224 tiles, 28.2 and 30.5.)
    const uint64_t tiles = ((uint64_t)m + XM_BM - 1) / XM_BM * (((uint64_t)n + XM_BN - 1) / XM_BN);
    if (tiles > (uint64_t)device_sms()) {
        // The tiles' width by the rounds that all pairs make over them: of 192, 256 or 384 columns, a column
        // of the wider ones taking 0.9 and 0.85 (NVFP4; 0.93 and 0.9 of the others) of one of the first, since
        // less is staged for the same work. With up to 128 rows of A the weights in flight count, 0.79 of 384.
        // us for 192, 256, 384: 4096 x 14336 x 4096 NVFP4 117, 107, 105 (17, 13, 9 rounds); 1024 x 4096 x 4096
        // 16.0, 11.4, 15.1 (2, 1, 1); 4096^3 MXFP4 33.0, 33.0, 36.5 (5, 4, 3); 2048 x 4096 x 4096 MXFP8 32.7,
        // 29.5, 39.6 (3, 2, 2); 16 x 128256 x 4096 MXFP8 152, 134, 120 (10, 7, 5).
        const uint64_t pairs = (uint64_t)device_sms() / 2, rows = ((uint64_t)m + 255) / 256;
        const bool nv = fmt == LYTH_MX_NVFP4;
        auto cost = [&](uint64_t width, uint64_t column) {
            return (rows * ((n + width - 1) / width) + pairs - 1) / pairs * width * column;
        };
        const uint64_t c192 = cost(192, 200), c256 = cost(256, nv ? 179 : 186);
        const uint64_t c384 = cost(384, m <= 128 ? 158 : nv ? 170 : 181);
        if (c256 < c192 && c256 < c384) {
            LYTH_MX_DISPATCH(fmt, ty, return (x2_launch<FMT, TY, 1, 256>(a, b, c, p, s)));
        }
        if (c384 < c192) {
            LYTH_MX_DISPATCH(fmt, ty, return (x2_launch<FMT, TY, 2, 192>(a, b, c, p, s)));
        }
        LYTH_MX_DISPATCH(fmt, ty, return (x2_launch<FMT, TY, 1, 192>(a, b, c, p, s)));
    }
    LYTH_MX_DISPATCH(fmt, ty, return (x1_launch<FMT, TY>(a, b, c, p, s)));
    return LYTH_E_UNSUPPORTED;
}
