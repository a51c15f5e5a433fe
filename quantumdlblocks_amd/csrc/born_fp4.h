// A paged key-value cache in 4 bits: its rows and how they are read.
//
// A row (one head of one token) is W = 32 nb columns, the head dim rounded up to
// whole blocks of 32 (zeros behind it).  A block is 16 bytes of 4-bit codes, the
// lower nibble first, and one scale byte e: value = code 2^(e - 127), the codes
// being sign, two exponent bits and one mantissa bit: 0, .5, 1, 1.5, 2, 3, 4, 6.
// e = 255: not a number; 253 and 254 are not written.
//
// Two significant bits and a power of two are exact in bf16, so every product
// here runs on the bf16 matrix pipe whatever the type of the queries: these are
// taken apart into bf16 parts that sum to them exactly (one for bf16, two for
// fp16, three for fp32), and so are the fp32 weights where they are not rounded.
//
// A token that cannot be held (an infinity, NaN or magnitude past 7 2^125 in it) has a block of scale
// 255: every query that sees it, and no other, gets NaN.  A weight of 0 times a
// NaN would reach the queries that do not see it, so V's bad blocks are read as
// zeros and K's block as NaN in their place.
#pragma once

#include <type_traits>

#include "born_common.h"
#include "born_packed.h"
#include "born_paged.h"

namespace qdl {

constexpr int kFp4Block = 32;
constexpr uint32_t kFp4Bad = 255;

// Strides in bytes: page, token, head; in 32 bits, so that an address takes one
// multiplication a stride.
struct Fp4Cache {
    uint8_t *k, *v, *ks, *vs;
    uint32_t kp, kt, kh, vp, vt, vh, ksp, kst, ksh, vsp, vst, vsh;
    int cache_pages;
    int page, page_shift, nb;  // tokens per page, its logarithm or -1; blocks of a row
};

// Row (page, token, head) of one of the tensors.
__device__ __forceinline__ uint64_t fp4_at(uint32_t page, uint32_t sp, uint32_t row, uint32_t st, uint32_t head, uint32_t sh) {
    return (uint64_t)page * sp + (uint64_t)row * st + (uint64_t)head * sh;
}

struct Fp4Pages {
    const int32_t* table;  // (B, pages)
    const int32_t* lens;   // (B)
    int64_t table_ld;
    int pages;
};

// Keys of sequence b, cut to its table.
__device__ __forceinline__ int fp4_len(const Fp4Cache& c, const Fp4Pages& t, int b) {
    return (int)min((int64_t)max(t.lens[b], 0), (int64_t)t.pages * c.page);
}

// Page index and row of key j >= 0.
__device__ __forceinline__ int fp4_page(const Fp4Cache& c, int j) { return c.page_shift >= 0 ? j >> c.page_shift : j / c.page; }

// The scale of a block as the conversions take it: fp32's exponent field.
__device__ __forceinline__ float fp4_scale(uint32_t e) { return __uint_as_float(e << 23); }

// Values 2 i and 2 i + 1 of a dword of codes, as a bf16 pair.
template <int I>
__device__ __forceinline__ uint32_t fp4_pair(uint32_t codes, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, I));
}
// All eight: the operand of a product over them.
__device__ __forceinline__ u32x4 fp4_eight(uint32_t codes, float scale) {
    return u32x4{fp4_pair<0>(codes, scale), fp4_pair<1>(codes, scale), fp4_pair<2>(codes, scale), fp4_pair<3>(codes, scale)};
}

// fp32 pairs as PARTS bf16 pairs whose sum they are (three: exactly).
template <int PARTS>
__device__ __forceinline__ void fp4_parts(float x, float y, uint32_t (&u)[PARTS]) {
#pragma unroll
    for (int i = 0; i < PARTS; ++i) {
        u[i] = BF16::pack(x, y);
        x -= BF16::lo(u[i]);
        y -= BF16::hi(u[i]);
    }
}

// bf16 parts of queries in E, and of the weights for outputs in E: with two the
// output's rounding is the only one of 16 bits, with three fp32 has none.
template <class E>
constexpr int kQParts = std::is_same<E, F32>::value ? 3 : std::is_same<E, F16>::value ? 2 : 1;
template <class E>
constexpr int kPParts = std::is_same<E, F32>::value ? 3 : 2;

// The same of values that bf16 may round to an infinity: its largest number first
// where they are finite, and nothing behind an infinity.
template <int PARTS>
__device__ __forceinline__ void fp4_large_parts(float x, float y, uint32_t (&u)[PARTS]) {
    auto first = [](float z) __attribute__((always_inline)) {
        return fabsf(z) >= 0x1.FFp127f && fabsf(z) < HUGE_VALF ? copysignf(0x1.FEp127f, z) : z;
    };
    u[0] = BF16::pack(first(x), first(y));
    uint32_t rest[PARTS - 1];
    fp4_parts<PARTS - 1>(fabsf(x) == HUGE_VALF ? 0.f : x - BF16::lo(u[0]), fabsf(y) == HUGE_VALF ? 0.f : y - BF16::hi(u[0]), rest);
#pragma unroll
    for (int i = 1; i < PARTS; ++i) u[i] = rest[i - 1];
}

// Eight values of a query from column `at` on (D - at of them, 0 behind), as operands.
template <class E>
__device__ __forceinline__ void fp4_query(const uint8_t* row, int at, int D, bool ok, bool neg, u32x4 (&q)[kQParts<E>]) {
    if constexpr (std::is_same<E, BF16>::value) {
        u32x4 y = {0u, 0u, 0u, 0u};
        if (ok && at < D) y = ldg16(row + 2 * at) ^ (neg ? 0x80008000u : 0u);
        q[0] = y;
    } else {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = 0.f;
        if (ok && at < D) {  // D: a multiple of 8
            if constexpr (std::is_same<E, F32>::value) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const u32x4 y = ldg16(row + 4 * at + 16 * h);
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[4 * h + i] = __uint_as_float(y[i]);
                }
            } else {
                const u32x4 y = ldg16(row + 2 * at);
#pragma unroll
                for (int i = 0; i < 4; ++i) x[2 * i] = E::lo(y[i]), x[2 * i + 1] = E::hi(y[i]);
            }
        }
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x[i] = neg ? -x[i] : x[i];
            top = fmaxf(top, fabsf(x[i]));
        }
        const bool large = top >= 0x1.FFp127f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t u[kQParts<E>];
            fp4_parts<kQParts<E>>(x[2 * i], x[2 * i + 1], u);
#pragma unroll
            for (int k = 0; k < kQParts<E>; ++k) q[k][i] = u[k];
        }
        if (!large) return;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t u[kQParts<E>];
            fp4_large_parts<kQParts<E>>(x[2 * i], x[2 * i + 1], u);
#pragma unroll
            for (int k = 0; k < kQParts<E>; ++k) q[k][i] = u[k];
        }
    }
}

template <class E>
__device__ __forceinline__ void fp4_store4(uint8_t* row, int col, f32x4v x) {
    if constexpr (std::is_same<E, F32>::value) {
        *reinterpret_cast<f32x4v*>(row + 4 * col) = x;
    } else {
        const u32x2 y = {E::pack(x[0], x[1]), E::pack(x[2], x[3])};
        *reinterpret_cast<u32x2*>(row + 2 * col) = y;
    }
}

}  // namespace qdl
