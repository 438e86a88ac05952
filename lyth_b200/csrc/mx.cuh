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

// ---- element types of the unquantised side: 0 f32, LYTH_NARROW_F16, LYTH_NARROW_BF16.
template <int TY> struct MxElem;
template <> struct MxElem<0> {
    using type = float;
    LYTH_D static float load(const float *p) { return *p; }
    LYTH_D static float round(float v) { return v; }
};
template <> struct MxElem<LYTH_NARROW_F16> {
    using type = __half;
    LYTH_D static float load(const __half *p) { return __half2float(*p); }
    LYTH_D static __half round(float v) { return __float2half_rn(v); }
};
template <> struct MxElem<LYTH_NARROW_BF16> {
    using type = __nv_bfloat16;
    LYTH_D static float load(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
    LYTH_D static __nv_bfloat16 round(float v) { return __float2bfloat16_rn(v); }
};
inline bool mx_ty_known(int ty) { return ty == 0 || ty == LYTH_NARROW_F16 || ty == LYTH_NARROW_BF16; }
inline uint64_t mx_ty_bytes(int ty) { return ty == 0 ? 4 : 2; }

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

// Eight consecutive values of a row, `col` a multiple of 8, zero behind `cols`. `vec`: every row
// starts on 16 bytes. Plain loads: an output may alias the input of the same positions.
template <int TY>
LYTH_D void mx_load8(const typename MxElem<TY>::type *row, uint32_t col, uint32_t cols, bool vec, float (&v)[8]) {
    if (vec && col + 8 <= cols) {
        if constexpr (TY == 0) {
            const float4 a = *reinterpret_cast<const float4 *>(row + col);
            const float4 b = *reinterpret_cast<const float4 *>(row + col + 4);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
            v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
            const uint4 u = *reinterpret_cast<const uint4 *>(row + col);
            const float2 a = mx_unpack2<TY>(u.x), b = mx_unpack2<TY>(u.y), c = mx_unpack2<TY>(u.z),
                         d = mx_unpack2<TY>(u.w);
            v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
            v[4] = c.x; v[5] = c.y; v[6] = d.x; v[7] = d.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = col + i < cols ? MxElem<TY>::load(row + col + i) : 0.0f;
    }
}
template <int TY>
LYTH_D void mx_store8(typename MxElem<TY>::type *row, uint32_t col, uint32_t cols, bool vec, const float (&v)[8]) {
    if (vec && col + 8 <= cols) {
        if constexpr (TY == 0) {
            *reinterpret_cast<float4 *>(row + col) = make_float4(v[0], v[1], v[2], v[3]);
            *reinterpret_cast<float4 *>(row + col + 4) = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            *reinterpret_cast<uint4 *>(row + col) = make_uint4(mx_pack2<TY>(v[0], v[1]), mx_pack2<TY>(v[2], v[3]),
                                                               mx_pack2<TY>(v[4], v[5]), mx_pack2<TY>(v[6], v[7]));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (col + i < cols) row[col + i] = MxElem<TY>::round(v[i]);
    }
}

// ---- code conversions (round to nearest even, saturating)
LYTH_D uint32_t e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
// Eight values to eight E2M1 codes, v[0] in the lowest four bits.
LYTH_D uint32_t e2m1x8(const float (&v)[8]) {
    uint32_t r;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
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

// Quantise the eight values of chunk `chunk` (columns 8*chunk ..) of a row and store its codes and,
// from the first lane of each scale word, the word. Called by whole warps; consecutive lanes hold
// consecutive chunks and a scale word's chunks (16, NVFP4 8) sit in lanes aligned to it, so the
// block's largest magnitude and the word itself are butterflies over neighbouring lanes. Lanes that
// are not `live` hold zeros and store nothing.
//
// The magnitudes are compared as integers (NaN above infinity above every number). Scale: MX, the
// exponent of the largest value less that of the largest code, which is exact; NVFP4, the largest
// value over 6 tensor scales, rounded to E4M3. A block that holds an infinity or a NaN gets the NaN
// scale and zero codes, so that what it stands for is NaN and not a number.
template <int FMT>
LYTH_D void mx_quantize8(const float (&v)[8], bool live, uint32_t chunk, uint8_t *codes_row, uint8_t *scales_row,
                         float inv6g, float g) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
    if constexpr (Mx<FMT>::kBlock == 32) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
    const bool bad = top >= 0x7F800000u;
    uint32_t byte;
    float mul, d = 1.0f;
    if constexpr (FMT == LYTH_MX_NVFP4) {
        byte = e4m3x2(__fmul_rn(__uint_as_float(top), inv6g), 0.0f) & 0x7Fu;
        d = __fmul_rn(mx_scales2<FMT>(byte).x, g);
        mul = byte == 0 ? 0.0f : __fdiv_rn(1.0f, d);
        if (bad) byte = 0x7Fu;
    } else {
        const int e = (int)(top >> 23) - Mx<FMT>::kEmax;
        byte = e > 0 ? (uint32_t)e : 0u;
        mul = __uint_as_float((254u - byte) << 23);  // 2^(127 - byte): the division is exact
        if (bad) byte = 0xFFu;
    }
    if (bad) mul = 0.0f;
    float q[8];
#pragma unroll
    for (int i = 0; i < 8; i++) q[i] = bad ? 0.0f : __fmul_rn(v[i], mul);
    if constexpr (FMT == LYTH_MX_NVFP4) {
        // v / d correctly rounded (Markstein's step after a correctly rounded 1 / d), so that values
        // halfway between two codes are halfway here too. A saturated scale leaves quotients of any
        // size; they are cut first, to keep the remainder finite.
        if (byte == 0x7Eu) {
#pragma unroll
            for (int i = 0; i < 8; i++) q[i] = fminf(fmaxf(q[i], -64.0f), 64.0f);
        }
        if (!bad && byte != 0) {
#pragma unroll
            for (int i = 0; i < 8; i++)  // the sign is v's: -0 + 0 in the step would lose it
                q[i] = copysignf(__fmaf_rn(__fmaf_rn(-q[i], d, v[i]), mul, q[i]), v[i]);
        }
    }
    constexpr int kLanes = Mx<FMT>::kBlock / 8;  // lanes of a block
    uint32_t word = byte << (8 * ((chunk / kLanes) & 3));
    word |= __shfl_xor_sync(0xFFFFFFFFu, word, kLanes);
    word |= __shfl_xor_sync(0xFFFFFFFFu, word, 2 * kLanes);
    if (!live) return;
    if constexpr (FMT == LYTH_MX_FP8) {
        *reinterpret_cast<uint2 *>(codes_row + 8ull * chunk) =
            make_uint2(e4m3x2(q[0], q[1]) | e4m3x2(q[2], q[3]) << 16, e4m3x2(q[4], q[5]) | e4m3x2(q[6], q[7]) << 16);
    } else {
        *reinterpret_cast<uint32_t *>(codes_row + 4ull * chunk) = e2m1x8(q);
    }
    if (chunk % (4 * kLanes) == 0)
        *reinterpret_cast<uint32_t *>(scales_row + (uint64_t)(chunk / (4 * kLanes)) * 512) = word;
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
