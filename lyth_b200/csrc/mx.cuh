// Block-scaled ("microscaled") formats shared by the quantisation, norm, product and GEMV kernels.
//
//   LYTH_MX_FP8     E4M3 codes, blocks of 32 columns, scale 2^(byte - 127) (E8M0)
//   LYTH_MX_FP4     E2M1 codes, blocks of 32 columns, scale 2^(byte - 127) (E8M0)
//   LYTH_MX_NVFP4   E2M1 codes, blocks of 16 columns, scale E4M3, times one f32 scale per tensor
//
// (the OCP Microscaling specification v1.0 for the first two). A row of `cols` values is held as
// k >= cols codes, k the next multiple of four blocks, so a row's scales are whole 32-bit words.
// Codes are row-major (4 bits: even column in the low half of the byte). Scales lie in tiles of 128
// rows x 4 blocks (512 bytes), the order the tensor cores take them from tensor memory: row r,
// block b of a tile at (r % 32) * 16 + (r / 32) * 4 + b; the tiles of 128 rows follow one another
// along k, then the next 128 rows.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace lyth {

template <int FMT>
struct Mx {
    static constexpr int kBlock = FMT == LYTH_MX_NVFP4 ? 16 : 32;      // columns per scale
    static constexpr int kBits = FMT == LYTH_MX_FP8 ? 8 : 4;           // bits per code
    static constexpr int kWord = 4 * kBlock;                           // columns per 32-bit scale word
    static constexpr int kEmax = FMT == LYTH_MX_FP8 ? 8 : 2;           // exponent of the largest code
};

inline uint32_t mx_block(int fmt) { return fmt == LYTH_MX_NVFP4 ? 16u : 32u; }
inline bool mx_known(int fmt) { return fmt == LYTH_MX_FP8 || fmt == LYTH_MX_FP4 || fmt == LYTH_MX_NVFP4; }
// Columns held for a row of `cols`: the next multiple of four blocks.
inline uint64_t mx_padded(int fmt, uint64_t cols) {
    const uint64_t w = 4ull * mx_block(fmt);
    return (cols + w - 1) / w * w;
}
inline uint64_t mx_code_bytes(int fmt, uint64_t k) { return fmt == LYTH_MX_FP8 ? k : k / 2; }

// ---- launches that overlap. A kernel here may be placed on the SMs while the one before it in the stream
// still runs its last blocks: all that touches no tensor (barriers, tensor memory, indexes) comes before
// grid_wait(), which returns once every earlier grid of the stream is complete and its writes are visible;
// grid_next() lets the following kernel do the same. Every thread that reads or writes global memory
// waits, and loads are not hoisted above it: pointers pass through grid_wait, or the loads are volatile.
LYTH_D void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
template <typename T>
LYTH_D T *after_wait(T *p) {  // p, as a value that exists only once the wait is over
    asm volatile("" : "+l"(p)::"memory");
    return p;
}
LYTH_D void grid_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Host: a launch with that leave, as clusters of `cluster` blocks; its status.
template <typename... P, typename... A>
inline int mx_launch(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, unsigned cluster,
                             A... args) {
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
    if (e != cudaSuccess) cudaGetLastError();  // reported here, not by the next call
    return status_of(e);
}

// ---- element types of the unquantised side: 0 f32, LYTH_NARROW_F16, LYTH_NARROW_BF16.
template <int TY> struct MxElem;
template <> struct MxElem<0> {
    using type = float;
    LYTH_D static float round(float v) { return v; }
};
template <> struct MxElem<LYTH_NARROW_F16> {
    using type = __half;
    LYTH_D static __half round(float v) { return __float2half_rn(v); }
};
template <> struct MxElem<LYTH_NARROW_BF16> {
    using type = __nv_bfloat16;
    LYTH_D static __nv_bfloat16 round(float v) { return __float2bfloat16_rn(v); }
};
inline bool mx_ty_known(int ty) { return ty == 0 || ty == LYTH_NARROW_F16 || ty == LYTH_NARROW_BF16; }
inline uint64_t mx_ty_bytes(int ty) { return ty == 0 ? 4 : 2; }
// Pointers of the unquantised side start on an element (null does).
inline bool mx_elem_aligned(const void *p, int ty) { return ((uintptr_t)p & (mx_ty_bytes(ty) - 1)) == 0; }

// Two f32 as one register of 16-bit values, a in the low half.
template <int TY>
LYTH_D uint32_t mx_pack2(float a, float b) {
    if constexpr (TY == LYTH_NARROW_F16) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}
template <int TY>
LYTH_D float2 mx_unpack2(uint32_t u) {
    if constexpr (TY == LYTH_NARROW_F16) {
        return __half22float2(*reinterpret_cast<const __half2 *>(&u));
    } else {
        return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
    }
}

// ---- rows of the unquantised side, 16 values ("a chunk") at a time.
// A chunk is 8 words of a 16-bit type, 16 of f32. VEC: every row starts on 32 bytes and is whole
// chunks, which move in 256-bit accesses (two 128-bit stores 32 bytes apart per lane write every
// 32-byte sector twice by halves: 14336 x 4096 values back from NVFP4 to bf16 in 40 us, now 25).
// Other rows start anywhere and are moved in aligned 16-byte accesses all the same: a load reads the
// aligned words around the chunk and shifts them, a store lets each lane complete its first aligned
// word with its neighbour's tail (333 x 4101 values back to bf16: 3.0 us, by elements 6.4).
constexpr int kMxChunk = 16;
template <int TY>
constexpr int kMxWords = TY == 0 ? 16 : 8;

LYTH_D void mx_ld32(const void *p, uint32_t *w) {
    asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                 : "l"(p));
}
LYTH_D void mx_st32(void *p, const uint32_t *w) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                 "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}
inline bool aligned32(const void *p) { return ((uintptr_t)p & 31u) == 0; }

// Words `delta` bytes (0 .. 15, a multiple of the element) into w[0 .. N + 3], N of them.
template <int N>
LYTH_D void mx_shift(uint32_t (&w)[N + 4], uint32_t delta) {
    if (delta & 8) {
#pragma unroll
        for (int i = 0; i < N + 2; i++) w[i] = w[i + 2];
    }
    if (delta & 4) {
#pragma unroll
        for (int i = 0; i < N + 1; i++) w[i] = w[i + 1];
    }
    if (delta & 2) {
#pragma unroll
        for (int i = 0; i < N; i++) w[i] = __funnelshift_r(w[i], w[i + 1], 16);
    }
}

// Chunk c of a row as words; zero behind `cols`. lo and hi bound the matrix (its first byte, one past
// its last): the aligned words may hold bytes of a neighbouring row or of the gap between rows, which
// are dropped, but nothing outside the matrix is read. Plain loads: an output may alias the input.
template <int TY, bool VEC>
LYTH_D void mx_load(const typename MxElem<TY>::type *row, uint32_t c, uint32_t cols, const void *lo, const void *hi,
                    uint32_t (&out)[kMxWords<TY>]) {
    constexpr int N = kMxWords<TY>, E = TY == 0 ? 4 : 2;
    if constexpr (VEC) {
        if (16 * c < cols) {
#pragma unroll
            for (int i = 0; i < N; i += 8) mx_ld32(reinterpret_cast<const char *>(row + 16 * c) + 4 * i, out + i);
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) out[i] = 0;
        }
        return;
    }
    const uint32_t left = cols > 16 * c ? cols - 16 * c : 0u;
    const char *p = reinterpret_cast<const char *>(row + 16ull * c);
    if (left == 0) {
#pragma unroll
        for (int i = 0; i < N; i++) out[i] = 0;
        return;
    }
    const uint32_t delta = (uint32_t)(reinterpret_cast<uintptr_t>(p) & 15u);
    const char *q = p - delta;
    const uint32_t need = 4 * N + (delta ? 16 : 0);
    if (q >= static_cast<const char *>(lo) && q + need <= static_cast<const char *>(hi)) {
        uint32_t w[N + 4];
#pragma unroll
        for (int i = 0; i < N / 4 + 1; i++) {
            uint4 u = make_uint4(0, 0, 0, 0);
            if (i < N / 4 || delta) u = *reinterpret_cast<const uint4 *>(q + 16 * i);
            w[4 * i] = u.x; w[4 * i + 1] = u.y; w[4 * i + 2] = u.z; w[4 * i + 3] = u.w;
        }
        mx_shift<N>(w, delta);
#pragma unroll
        for (int i = 0; i < N; i++) out[i] = w[i];
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) {
            if constexpr (TY == 0) {
                out[i] = (uint32_t)i < left ? reinterpret_cast<const uint32_t *>(p)[i] : 0u;
            } else {
                const uint16_t *h = reinterpret_cast<const uint16_t *>(p);
                const uint32_t a = 2u * i < left ? h[2 * i] : 0u, b = 2u * i + 1 < left ? h[2 * i + 1] : 0u;
                out[i] = a | b << 16;
            }
        }
        return;
    }
    if (left < 16) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            if constexpr (E == 4) {
                if ((uint32_t)i >= left) out[i] = 0;
            } else {
                if (2u * i >= left) out[i] = 0;
                else if (2u * i + 1 >= left) out[i] &= 0xFFFFu;
            }
        }
    }
}

// Chunk c of a row from words. Called by whole warps (it shuffles unless VEC), lane l + 1 holding the
// chunk after lane l's where both lie in one row. Lanes not `live`, and elements behind `cols`, store
// nothing.
template <int TY, bool VEC>
LYTH_D void mx_store(typename MxElem<TY>::type *row, uint32_t c, uint32_t cols, bool live,
                     const uint32_t (&w)[kMxWords<TY>]) {
    constexpr int N = kMxWords<TY>, E = TY == 0 ? 4 : 2;
    if constexpr (VEC) {
        if (live && 16 * c < cols) {
#pragma unroll
            for (int i = 0; i < N; i += 8) mx_st32(reinterpret_cast<char *>(row + 16 * c) + 4 * i, w + i);
        }
        return;
    }
    const uint32_t left = live && cols > 16 * c ? cols - 16 * c : 0u, lane = threadIdx.x & 31;
    char *p = reinterpret_cast<char *>(row + 16ull * c);
    const uint32_t delta = (uint32_t)(reinterpret_cast<uintptr_t>(p) & 15u);
    const bool whole = left >= 16;
    uint32_t to = left < 16 ? left * E : 0;  // the chunk's first bytes, stored by elements
    const uint32_t whole_of = __ballot_sync(0xFFFFFFFFu, whole);
    // the neighbours' chunks continue this one exactly when they are in the same row
    const bool prev = whole && c > 0 && lane > 0 && (whole_of >> (lane - 1) & 1);
    const uint32_t c_next = __shfl_down_sync(0xFFFFFFFFu, c, 1);
    const bool next = whole && lane < 31 && (whole_of >> (lane + 1) & 1) && c_next == c + 1;
    uint32_t v[N + 4];  // the previous lane's last 16 bytes, then this lane's
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = __shfl_up_sync(0xFFFFFFFFu, w[N - 4 + i], 1);
#pragma unroll
    for (int i = 0; i < N; i++) v[4 + i] = w[i];
    if (whole) {
        // the words that start at p - delta are 16 - delta bytes in; delta 0 leaves this lane's own
        mx_shift<N>(v, (16 - delta) & 15);
        char *q = p - delta;
#pragma unroll
        for (int i = 0; i < N / 4; i++) {
            uint4 u = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
            if (delta == 0) u = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
            if (i > 0 || prev || delta == 0) reinterpret_cast<uint4 *>(q)[i] = u;
        }
        if (delta && !prev) to = 16 - delta;
        if (delta && !next) {  // this lane's last delta bytes
#pragma unroll
            for (int i = 0; i < 16 / E; i++) {
                const uint32_t at = 4 * N - 16 + i * E;
                if (at >= 4 * N - delta) {
                    if constexpr (E == 4) reinterpret_cast<uint32_t *>(p)[at / 4] = w[at / 4];
                    else reinterpret_cast<uint16_t *>(p)[at / 2] = (uint16_t)(w[at / 4] >> (8 * (at & 2)));
                }
            }
        }
    }
    if (to) {
#pragma unroll
        for (int i = 0; i < 4 * N / E; i++) {
            const uint32_t at = i * E;
            if (at < to) {
                if constexpr (E == 4) reinterpret_cast<uint32_t *>(p)[i] = w[i];
                else reinterpret_cast<uint16_t *>(p)[i] = (uint16_t)(w[at / 4] >> (8 * (at & 2)));
            }
        }
    }
}

// Words to f32 values and back (one rounding).
template <int TY>
LYTH_D void mx_widen(const uint32_t (&w)[kMxWords<TY>], float (&v)[16]) {
    if constexpr (TY == 0) {
#pragma unroll
        for (int i = 0; i < 16; i++) v[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float2 f = mx_unpack2<TY>(w[i]);
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
}
template <int TY>
LYTH_D void mx_narrow(const float (&v)[16], uint32_t (&w)[kMxWords<TY>]) {
    if constexpr (TY == 0) {
#pragma unroll
        for (int i = 0; i < 16; i++) w[i] = __float_as_uint(v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) w[i] = mx_pack2<TY>(v[2 * i], v[2 * i + 1]);
    }
}
// The largest magnitude of three values, NaN if one is.
LYTH_D float mx_max3(float a, float b, float c) {
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// The bits of the largest magnitude among the chunk's values (above any number's if one is NaN); of
// 16-bit types two at a time on the stored patterns, which order alike.
LYTH_D uint32_t mx_top(const float (&v)[16]) {
    float t[5];
#pragma unroll
    for (int i = 0; i < 5; i++) t[i] = mx_max3(v[3 * i], v[3 * i + 1], v[3 * i + 2]);
    const float u = mx_max3(t[0], t[1], t[2]), w = mx_max3(t[3], t[4], v[15]);
    return __float_as_uint(mx_max3(u, w, w)) & 0x7FFFFFFFu;
}
template <int TY>
LYTH_D uint32_t mx_top_words(const uint32_t (&w)[kMxWords<TY>]) {
    uint32_t top = 0;
    if constexpr (TY == 0) {
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; i++) v[i] = __uint_as_float(w[i]);
        return mx_top(v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) top = __vmaxu2(top, w[i] & 0x7FFF7FFFu);
        const uint32_t h = max(top & 0xFFFFu, top >> 16);
        return __float_as_uint(mx_unpack2<TY>(h).x);
    }
}

// ---- code conversions (round to nearest even, saturating)
LYTH_D uint32_t e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
// Four values to four E4M3 codes, the first in the lowest byte.
LYTH_D uint32_t e4m3x4(float2 v0, float2 v1) {
    uint32_t r;
    asm("{\n\t.reg .b16 a, b;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 b, %4, %3;\n\t"
        "mov.b32 %0, {a, b};\n\t}"
        : "=r"(r)
        : "f"(v0.x), "f"(v0.y), "f"(v1.x), "f"(v1.y));
    return r;
}
// Eight values to eight E2M1 codes, the first in the lowest four bits.
LYTH_D uint32_t e2m1x8(float2 v0, float2 v1, float2 v2, float2 v3) {
    uint32_t r;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(r)
        : "f"(v0.x), "f"(v0.y), "f"(v1.x), "f"(v1.y), "f"(v2.x), "f"(v2.y), "f"(v3.x), "f"(v3.y));
    return r;
}
// A register of eight E2M1 codes as four pairs of f16 (exact: every code is an f16 value).
LYTH_D void e2m1x8_f16(uint32_t w, uint32_t (&h)[4]) {
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "mov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(w));
}
// A register of four E4M3 codes as two pairs of f16 (exact).
LYTH_D void e4m3x4_f16(uint32_t w, uint32_t &lo, uint32_t &hi) {
    asm("{\n\t.reg .b16 a, b;\n\t"
        "mov.b32 {a, b}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
}
LYTH_D float2 f16x2_f32(uint32_t h) { return __half22float2(*reinterpret_cast<const __half2 *>(&h)); }
// The scales of the two bytes in the low half of `w`, as f32 (0xFF of E8M0 and 0x7F of E4M3 are NaN).
template <int FMT>
LYTH_D float2 mx_scales2(uint32_t w) {
    uint32_t r;
    const uint16_t h = (uint16_t)w;
    if constexpr (FMT == LYTH_MX_NVFP4) {
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(h));
        return f16x2_f32(r);
    } else {
        asm("cvt.rn.bf16x2.ue8m0x2 %0, %1;" : "=r"(r) : "h"(h));
        return make_float2(__uint_as_float(r << 16), __uint_as_float(r & 0xFFFF0000u));
    }
}

// Where row r's scale word for columns 0 .. kWord-1 lies; the words along k are 512 bytes apart.
// `words` = k / kWord.
LYTH_D uint64_t mx_scale_row(uint64_t r, uint32_t words) {
    return (r >> 7) * words * 512ull + (r & 31) * 16 + ((r >> 5) & 3) * 4;
}

// Two independent f32 sums, products or multiply-adds, each rounded as the scalar one.
LYTH_D float2 mx_mul2(float2 a, float2 b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;"
        : "=l"(d)
        : "l"(*reinterpret_cast<uint64_t *>(&a)), "l"(*reinterpret_cast<uint64_t *>(&b)));
    return *reinterpret_cast<float2 *>(&d);
}
LYTH_D float2 mx_mul2_rz(float2 a, float2 b) {
    uint64_t d;
    asm("mul.rz.f32x2 %0, %1, %2;"
        : "=l"(d)
        : "l"(*reinterpret_cast<uint64_t *>(&a)), "l"(*reinterpret_cast<uint64_t *>(&b)));
    return *reinterpret_cast<float2 *>(&d);
}
LYTH_D float2 mx_add2(float2 a, float2 b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(d)
        : "l"(*reinterpret_cast<uint64_t *>(&a)), "l"(*reinterpret_cast<uint64_t *>(&b)));
    return *reinterpret_cast<float2 *>(&d);
}
LYTH_D float2 mx_fma2(float2 a, float2 b, float2 c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(d)
        : "l"(*reinterpret_cast<uint64_t *>(&a)), "l"(*reinterpret_cast<uint64_t *>(&b)),
          "l"(*reinterpret_cast<uint64_t *>(&c)));
    return *reinterpret_cast<float2 *>(&d);
}

// Two products rounded to odd: cut, and the last bit set where the cut lost something (or is NaN). Rounding that
// to a shorter type is rounding the product itself to it. The products' last bits are f32 numbers here.
LYTH_D float2 mx_mul2_odd(float2 a, float b) {
    const float2 v = mx_mul2_rz(a, make_float2(b, b)), lost = mx_fma2(a, make_float2(-b, -b), v);
    return make_float2(__uint_as_float(__float_as_uint(v.x) | (lost.x != 0.0f)),
                       __uint_as_float(__float_as_uint(v.y) | (lost.y != 0.0f)));
}
// The sixteen values of an NVFP4 block in a 16-bit type, each code * s * g rounded once (code * s is exact, and f32
// before the type would be a second rounding). A block has eight magnitudes: they are rounded once for all, and
// the values looked up by byte: 14336 x 4096 to bf16 24.0 us, as with two roundings; each value by itself 29.1.
template <int TY>
LYTH_D void mx_nvfp4_back(uint32_t w0, uint32_t w1, float s, float g, uint32_t (&out)[8]) {
    uint32_t m[4];  // the magnitudes of codes 2 i and 2 i + 1
    if constexpr (TY == LYTH_NARROW_BF16) {
        // 2^-110 .. 2^112, normal numbers of bf16: s g and 3 s g rounded, the others steps of the exponent from them
        const float2 v = mx_mul2_odd(make_float2(s, __fmul_rn(s, 3.0f)), g);
        const uint32_t p = mx_pack2<TY>(v.x, v.y);
        const bool number = s != 0.0f && s == s;  // else all are zero, or NaN
        m[0] = number ? (p << 16) - 0x00800000u : p;
        m[1] = number ? p - 0x00800000u : p;
        m[2] = number ? p + 0x00000080u : p;
        m[3] = number ? p + 0x00800100u : p;
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            constexpr float kCode[8] = {0.0f, 0.5f, 1.0f, 1.5f, 2.0f, 3.0f, 4.0f, 6.0f};
            const float2 v = mx_mul2_odd(mx_mul2(make_float2(kCode[2 * i], kCode[2 * i + 1]), make_float2(s, s)), g);
            m[i] = mx_pack2<TY>(v.x, v.y);
        }
    }
    const uint32_t lo0 = __byte_perm(m[0], m[1], 0x6420), lo1 = __byte_perm(m[2], m[3], 0x6420);
    const uint32_t hi0 = __byte_perm(m[0], m[1], 0x7531), hi1 = __byte_perm(m[2], m[3], 0x7531);
#pragma unroll
    for (int i = 0; i < 4; i++) {  // four codes each
        const uint32_t w = (i & 2 ? w1 : w0) >> (16 * (i & 1));
        const uint32_t sign = __byte_perm(w << 4, w, 0x5140);  // of code j in bit 7 of byte j
        const uint32_t lo = __byte_perm(lo0, lo1, w & 0x7777u);
        const uint32_t hi = __byte_perm(hi0, hi1, w & 0x7777u) ^ (sign & 0x80808080u);
        out[2 * i] = __byte_perm(lo, hi, 0x5140);
        out[2 * i + 1] = __byte_perm(lo, hi, 0x7362);
    }
}

// Quantise the sixteen values of chunk c (columns 16 c ..) of a row, `top` the bits of their largest
// magnitude (mx_top), and store its codes and, from the first lane of each scale word, the word.
// Called by whole warps; consecutive lanes hold consecutive chunks and a scale word's chunks (8, NVFP4
// 4) sit in lanes aligned to it, so what the lanes of a block and of a word share is a butterfly.
// Lanes that are not `live` hold zeros and store nothing.
//
// Scale: MX, the exponent of the largest value less that of the largest code, which is exact; NVFP4,
// the largest value over 6 tensor scales, rounded to E4M3. A block that holds an infinity or a NaN
// gets the NaN scale and zero codes, so that what it stands for is NaN and not a number.
template <int FMT>
LYTH_D void mx_quantize(const float (&v)[16], uint32_t top, bool live, uint32_t c, uint8_t *codes_row,
                        uint8_t *scales_row, float inv6g, float g) {
    if constexpr (Mx<FMT>::kBlock == 32) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
    const bool bad = top >= 0x7F800000u;
    uint32_t byte;
    float2 q[8];
    if constexpr (FMT == LYTH_MX_NVFP4) {
        byte = e4m3x2(__fmul_rn(__uint_as_float(top), inv6g), 0.0f) & 0x7Fu;
        // 1 / d in two parts, the first rounded down: v r + (v r_lo) is v / d to 2^-46, rounded once, so
        // values halfway between two codes are halfway here too (v r alone misses some of them when d
        // is 13, 14 or 15 eighths of a power of two). d is rounded itself unless g is a power of two; then
        // a quotient is off by less than 2^-22. r_lo >= 0 keeps the sign of a zero.
        const float d = __fmul_rn(mx_scales2<FMT>(byte).x, g), r = byte == 0 ? 0.0f : __frcp_rd(d);
        const float r_lo = __fmul_rn(__fmaf_rn(-d, r, 1.0f), r);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float2 u = make_float2(v[2 * i], v[2 * i + 1]);
            q[i] = mx_fma2(u, make_float2(r, r), mx_mul2(u, make_float2(r_lo, r_lo)));
        }
        if (bad) byte = 0x7Fu;
    } else {
        const int e = (int)(top >> 23) - Mx<FMT>::kEmax;
        byte = e > 0 ? (uint32_t)e : 0u;
        const float r = __uint_as_float((254u - byte) << 23);  // 2^(127 - byte): the division is exact
#pragma unroll
        for (int i = 0; i < 8; i++) q[i] = mx_mul2(make_float2(v[2 * i], v[2 * i + 1]), make_float2(r, r));
        if (bad) byte = 0xFFu;
    }
    constexpr int kLanes = Mx<FMT>::kBlock / 16;  // lanes of a block
    uint32_t word = byte << (8 * ((c / kLanes) & 3));
    word |= __shfl_xor_sync(0xFFFFFFFFu, word, kLanes);
    word |= __shfl_xor_sync(0xFFFFFFFFu, word, 2 * kLanes);
    if (!live) return;
    if constexpr (FMT == LYTH_MX_FP8) {
        uint4 u = make_uint4(e4m3x4(q[0], q[1]), e4m3x4(q[2], q[3]), e4m3x4(q[4], q[5]), e4m3x4(q[6], q[7]));
        if (bad) u = make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4 *>(codes_row + 16ull * c) = u;
    } else {
        uint2 u = make_uint2(e2m1x8(q[0], q[1], q[2], q[3]), e2m1x8(q[4], q[5], q[6], q[7]));
        if (bad) u = make_uint2(0, 0);
        *reinterpret_cast<uint2 *>(codes_row + 8ull * c) = u;
    }
    if (c % (4 * kLanes) == 0)
        *reinterpret_cast<uint32_t *>(scales_row + (uint64_t)(c / (4 * kLanes)) * 512) = word;
}

// Host: the constants of an NVFP4 tensor scale (1 for the MX formats, whose scale it must be).
// Scales outside 2^-100 .. 2^100 are refused: products with a block scale would leave f32.
inline bool mx_tensor_scale(int fmt, float g, float &inv6g) {
    if (fmt != LYTH_MX_NVFP4) {
        inv6g = 1.0f;
        return g == 1.0f;
    }
    if (!(g >= 7.8886091e-31f && g <= 1.2676506e30f)) return false;
    inv6g = (float)(1.0 / (6.0 * (double)g));
    return true;
}

// Calls `f` with the format and the element type as compile-time constants.
#define LYTH_MX_DISPATCH_TY(fmt_const, ty, ...)                                   \
    switch (ty) {                                                                 \
        case 0: { constexpr int FMT = fmt_const, TY = 0; __VA_ARGS__; break; }     \
        case LYTH_NARROW_F16: { constexpr int FMT = fmt_const, TY = LYTH_NARROW_F16; __VA_ARGS__; break; } \
        default: { constexpr int FMT = fmt_const, TY = LYTH_NARROW_BF16; __VA_ARGS__; break; }            \
    }
#define LYTH_MX_DISPATCH(fmt, ty, ...)                                            \
    switch (fmt) {                                                                \
        case LYTH_MX_FP8: LYTH_MX_DISPATCH_TY(LYTH_MX_FP8, ty, __VA_ARGS__); break; \
        case LYTH_MX_FP4: LYTH_MX_DISPATCH_TY(LYTH_MX_FP4, ty, __VA_ARGS__); break; \
        default: LYTH_MX_DISPATCH_TY(LYTH_MX_NVFP4, ty, __VA_ARGS__); break;        \
    }

}  // namespace lyth
