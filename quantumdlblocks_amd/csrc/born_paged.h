// Born attention of one new token per sequence over a paged key-value cache.
//
//   p_j = (s relu(sign(s) q.k_j))^2 for the sequence's visible keys j,
//   O = sum_j p_j v_j / (sum_j p_j + eps)
// for each query head; G = H / Hkv query heads read one key head.  Key j of
// sequence b lies in page table[b][j / page] at row j % page.
//
// What bounds it: reading K and V once.  The weights need no maximum, so the
// keys split freely: a workgroup takes one split of one (sequence, key head),
// its four waves every fourth 32 keys of it, and partial sums of numerators and
// denominators just add: the waves' in LDS, the splits' in the join kernel,
// both in a fixed order.
//
// Nothing is staged: K goes straight from memory into the A operand of S^T = K
// Q^T (16 keys, 32 columns each), up to 16 query heads of the group being its
// columns.  V comes as whole rows, 8 columns of a lane's keys per load, and the
// lane picks the A operand of O^T = V^T P^T out of its 8 x 8 values by byte
// permutes (half an operation per value), since the order of the columns is
// free: the m-th row of accumulator e is column 8 m + e.  The weights never
// leave the registers: the two 16-key products' C layout is the B operand of
// the 32-key one in the key order that the V loads use.
//
// No weight is rounded to 16 bits: its 16-bit form and that of what is left of it
// are two products with the same operand of V, which costs nothing beside the
// loads (us with one product and with two, by graph replay: bf16 64 sequences of
// 1024 keys, 8 key heads, D128 66.2 and 66.5; 16 of 4096, D256 115.9 and 116.3;
// 32 heads a key head, D64 35.4 and 35.7).  The denominator and the raw weights
// for key_weight take them in fp32; splits are written and joined in fp32.
//
// bf16, 32 sequences of 2048 to 14622 keys, 8 key heads D128: 808 MB in 162 us
// (5.0 TB/s) and a join of 5; one sequence of 1531 keys: 5.6 us and 2.9.
#pragma once

#include <type_traits>

#include "born_common.h"
#include "born_packed.h"

namespace qdl {

typedef float f32x4v __attribute__((ext_vector_type(4)));

struct PagedArgs {
    const void *q, *k, *v;
    void* out;
    const int32_t* table;  // (B, pages)
    const int32_t* lens;   // (B)
    const float* scale;
    float scale_value;
    int per_head_scale;
    int B, H, Hkv, G, D;
    int pages;             // table columns
    int64_t table_ld;
    int64_t cache_pages;   // pages of the cache: others are missing
    int page, page_shift;  // tokens per page; its logarithm, or -1
    int window;
    int nsplit, chunk;     // keys per split, a multiple of 128
    int gblocks;           // 16-head blocks of a group
    float eps;
    int64_t q_sb, q_sh, kp, kt, kh, vp, vt, vh;  // bytes
    float* part;           // (B, H, nsplit, D + 4): denominator, three unused, numerators; or nullptr (one split)
    float* weights;        // (B, Hkv, L) or nullptr: += sum over the group of p / Z
    int64_t w_sb, w_sh;    // elements
    int w_len;             // columns of weights
    float* raw;            // (B, H, raw_ld) workspace: p without s^2, keys from paged_base on, where weights are kept
    int64_t raw_ld;
};

__device__ __forceinline__ f32x4v mfma16_f32(float a, float b, f32x4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}
template <class E>
__device__ __forceinline__ f32x4v mfma16(u32x4 a, u32x4 b, f32x4v c) {
    if constexpr (std::is_same<E, F16>::value)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Visible keys of a sequence: [first, n).
struct PagedSpan {
    int first, n;
};
__device__ __forceinline__ PagedSpan paged_span(const PagedArgs& p, int b) {
    const int64_t room = (int64_t)p.pages * p.page;
    const int n = (int)min((int64_t)max(p.lens[b], 0), room);
    return {p.window > 0 ? max(0, n - p.window) : 0, n};
}

// Splits and raw weights count from here.
__device__ __forceinline__ int paged_base(PagedSpan sp) { return sp.first & ~31; }

// Page table entries and scalars that never change during a launch, read as
// scalar loads where the index is uniform.
typedef const __attribute__((address_space(4))) int32_t* ConstIntPtr;

// Row of key j: page and row in it; false for keys outside [first, n) and for
// pages that are none of the cache's.
__device__ __forceinline__ bool paged_row(const PagedArgs& p, ConstIntPtr table, PagedSpan sp, int j, int64_t& page, int& row) {
    const bool in = j >= sp.first && j < sp.n;
    const int jj = in ? j : 0;
    const int i = p.page_shift >= 0 ? jj >> p.page_shift : jj / p.page;
    row = jj - i * p.page;
    const int32_t t = in ? table[i] : -1;
    page = t;
    return t >= 0 && t < p.cache_pages;
}

// 1 / Z, without the s^2 of both; 0 for rows without weight.
__device__ __forceinline__ float paged_inverse(const PagedArgs& p, int h, float z) {
    const float s = arg_scale(p, h), den = z + (p.eps == 0.f ? 0.f : p.eps / (s * s));
    return s != 0.f ? packed_inverse(den) : 0.f;
}

// A operands of V^T: 16-bit, lane's 8 keys x 8 columns (x[k][...]) -> the keys
// of column e.
__device__ __forceinline__ u32x4 paged_column(const u32x4 (&x)[8], int e) {
    u32x4 a;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t lo = x[2 * i][e >> 1], hi = x[2 * i + 1][e >> 1];
        a[i] = __builtin_amdgcn_perm(hi, lo, (e & 1) ? 0x07060302u : 0x05040100u);
    }
    return a;
}

template <class E, int DP>
struct PagedCfg {
    static constexpr bool k32 = std::is_same<E, F32>::value;
    static constexpr int IT = kItem<E>;
    // K: 16-byte chunks of a row, four lanes of a key taking chunks 4 ks + j.
    static constexpr int KS = DP * IT / 64;
    // V: columns per lane and load (VC), blocks of 16 VC columns.
    static constexpr int VC = k32 ? 4 : DP == 64 ? 4 : 8, VB = DP / (16 * VC), NO = VB * VC;
    static constexpr int VW = VC * IT / 4;  // dwords of a V load
    // Two sets of 32 keys in registers, one loading while the other is used,
    // where two fit beside the accumulators.
    static constexpr int NBUF = 2 * 4 * KS + 8 * VW * VB <= 64 ? 2 : 1;
    static constexpr int WPE = IT * DP <= 256 ? 2 : 1;
};

// A wave's 32 keys.
template <class E, int DP>
struct PagedKeys {
    using C = PagedCfg<E, DP>;
    u32x4 k[2][C::KS];
    u32x4 v[C::VB][8];
    bool full, there[2];  // all 32 visible; the pages of each 16
};

__device__ __forceinline__ u32x4 paged_ldg(const uint8_t* p, int words) {
    if (words == 4) return ldg16(p);
    const u32x2 y = *reinterpret_cast<const u32x2*>(p);
    return u32x4{y[0], y[1], 0u, 0u};
}

// DP: 64, 128 or 256 columns; WEIGH: the raw weights are written too; P16:
// pages of a multiple of 16 tokens, so that 16 keys from a multiple of 16 lie in
// one page and their addresses are one scalar base and a lane's offset.
template <class E, int DP, bool WEIGH, bool P16>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(PagedCfg<E, DP>::WPE)))
void born_paged_kernel(PagedArgs p) {
    using C = PagedCfg<E, DP>;
    constexpr bool k32 = C::k32;
    constexpr int IT = C::IT, NW = 4, KS = C::KS, VC = C::VC, VB = C::VB, NO = C::NO, VW = C::VW;
    __shared__ float red[NW][16][DP + 4];
    __shared__ float zred[NW][16];

    const int gb = blockIdx.x % p.gblocks, rest = blockIdx.x / p.gblocks;
    const int hk = rest % p.Hkv, rest2 = rest / p.Hkv;
    const int split = rest2 % p.nsplit, b = rest2 / p.nsplit;
    const PagedSpan sp = paged_span(p, b);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int m = lane & 15, j4 = lane >> 4;
    const int heads = min(16, p.G - 16 * gb), h0 = hk * p.G + 16 * gb;
    const int base = paged_base(sp);
    const int s0 = base + split * p.chunk, s1 = min(sp.n, s0 + p.chunk);
    if (s0 >= s1 && split > 0) return;  // the join reads the filled splits only
    const ConstIntPtr table = (ConstIntPtr)(uintptr_t)(p.table + (int64_t)b * p.table_ld);
    const uint8_t* const kc = (const uint8_t*)p.k + (int64_t)hk * p.kh;
    const uint8_t* const vc = (const uint8_t*)p.v + (int64_t)hk * p.vh;

    // A lane's chunks of K and columns of V; past D they are read from the
    // row's start, K's made zeros and V's columns never stored.
    int ko[KS], vo[VB];
    uint32_t kmask[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        const int at = 16 * (4 * ks + j4);
        kmask[ks] = at < IT * p.D ? ~0u : 0u;
        ko[ks] = at < IT * p.D ? at : 0;
    }
#pragma unroll
    for (int vb = 0; vb < VB; ++vb) {
        const int col = 16 * VC * vb + VC * m;
        vo[vb] = col < p.D ? IT * col : 0;
    }
    const bool whole = p.D == DP;

    // Query head h0 + m in the columns of S^T.
    const bool okh = m < heads;
    const float sc = arg_scale(p, okh ? h0 + m : h0);
    const uint32_t flip = packed_flip<E>(sc);
    u32x4 qr[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        u32x4 x = {0u, 0u, 0u, 0u};
        if (okh && kmask[ks]) x = ldg16((const uint8_t*)p.q + (int64_t)b * p.q_sb + (int64_t)(h0 + m) * p.q_sh + ko[ks]) ^ flip;
        qr[ks] = x;
    }
    f32x4v acc[NO];
#pragma unroll
    for (int i = 0; i < NO; ++i) acc[i] = f32x4v{0.f, 0.f, 0.f, 0.f};
    float z = 0.f, cf = std::is_same<E, F16>::value ? kF16Start : 1.f;

    // Keys key0 + 16 t + m for K, key0 + 16 t + 4 j4 + i for V.
    auto load = [&](PagedKeys<E, DP>& x, int key0) __attribute__((always_inline)) {
        if constexpr (P16) {
            // Keys outside [first, n) and missing pages: the loads go to the
            // nearest visible key, or to page 0, and use() drops what they bring.
            const uint8_t *kp[2], *vp[2];
            int first[2];
            x.full = key0 >= sp.first && key0 + 32 <= sp.n;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int j = min(max(key0 + 16 * t, sp.first), sp.n - 1);
                const int i = __builtin_amdgcn_readfirstlane(p.page_shift >= 0 ? j >> p.page_shift : j / p.page);
                const int32_t page = table[i];
                x.there[t] = page >= 0 && page < p.cache_pages;
                x.full = x.full && x.there[t];
                const int64_t at = x.there[t] ? page : 0;
                kp[t] = kc + at * p.kp;
                vp[t] = vc + at * p.vp;
                first[t] = i * p.page;
            }
            auto row = [&](int t, int r) { return (uint32_t)(min(max(key0 + 16 * t + r, sp.first), sp.n - 1) - first[t]); };
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const uint32_t o = row(t, m) * (uint32_t)p.kt;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) x.k[t][ks] = ldg16(kp[t] + (o + (uint32_t)ko[ks]));
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t o = row(i >> 2, 4 * j4 + (i & 3)) * (uint32_t)p.vt;
#pragma unroll
                for (int vb = 0; vb < VB; ++vb) x.v[vb][i] = paged_ldg(vp[i >> 2] + (o + (uint32_t)vo[vb]), VW);
            }
            return;
        }
        x.full = true;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            int64_t page;
            int row;
            const bool ok = paged_row(p, table, sp, key0 + 16 * t + m, page, row);
            const uint8_t* at = kc + page * p.kp + (int64_t)row * p.kt;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                u32x4 y = {0u, 0u, 0u, 0u};
                if (ok) y = ldg16(at + ko[ks]);
                x.k[t][ks] = y;
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            int64_t page;
            int row;
            const bool ok = paged_row(p, table, sp, key0 + 16 * (i >> 2) + 4 * j4 + (i & 3), page, row);
            const uint8_t* at = vc + page * p.vp + (int64_t)row * p.vt;
#pragma unroll
            for (int vb = 0; vb < VB; ++vb) {
                u32x4 y = {0u, 0u, 0u, 0u};
                if (ok) y = paged_ldg(at + vo[vb], VW);
                x.v[vb][i] = y;
            }
        }
    };
    auto use = [&](PagedKeys<E, DP>& x, int key0) __attribute__((always_inline)) {
        if (!whole) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) x.k[t][ks] &= kmask[ks];
        }
        f32x4v s[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            s[t] = f32x4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                if constexpr (k32) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[t] = mfma16_f32(__uint_as_float(x.k[t][ks][i]), __uint_as_float(qr[ks][i]), s[t]);
                } else {
                    s[t] = mfma16<E>(x.k[t][ks], qr[ks], s[t]);
                }
            }
        }
        if (P16 && !x.full) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int key = key0 + 16 * (i >> 2) + 4 * j4 + (i & 3);
                const bool seen = x.there[i >> 2] && key >= sp.first && key < sp.n;
                if (!seen) s[i >> 2][i & 3] = 0.f;
#pragma unroll
                for (int vb = 0; vb < VB; ++vb) x.v[vb][i] &= seen ? ~0u : 0u;
            }
        }
        // Weights: relu(r)^2, keys 16 t + 4 j4 + r of the 32.
        float w[8];
        if constexpr (std::is_same<E, F16>::value) {
            float big = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) big = fmaxf(big, s[i >> 2][i & 3]);
            big = fmaxf(big, __shfl_xor(big, 16));
            big = fmaxf(big, __shfl_xor(big, 32));
            if (__ballot(big * cf > 255.f) != 0) {
                const float to = big * cf > 255.f ? f16_factor(big) : cf, by = (to / cf) * (to / cf);
                cf = to;
                z *= by;
#pragma unroll
                for (int i = 0; i < NO; ++i) acc[i] *= by;
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float a = relu_f32(s[i >> 2][i & 3]) * cf;
            w[i] = a * a;
        }
        if constexpr (WEIGH) {
            const float back = std::is_same<E, F16>::value ? 1.f / (cf * cf) : 1.f;
            if (okh) {
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const int at = key0 - base + 16 * t + 4 * j4;
                    float* to = p.raw + ((int64_t)b * p.H + h0 + m) * p.raw_ld + at;
                    const f32x4v y = {w[4 * t] * back, w[4 * t + 1] * back, w[4 * t + 2] * back, w[4 * t + 3] * back};
                    if (at < p.raw_ld) *reinterpret_cast<f32x4v*>(to) = y;  // raw_ld: a multiple of 32
                }
            }
        }
        if constexpr (k32) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                z += w[i];
#pragma unroll
                for (int vb = 0; vb < VB; ++vb)
#pragma unroll
                    for (int e = 0; e < VC; ++e)
                        acc[vb * VC + e] = mfma16_f32(__uint_as_float(x.v[vb][i][e]), w[i], acc[vb * VC + e]);
            }
        } else {
            // In two 16-bit parts, so that only the output is rounded.
            u32x4 hi, lo;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                hi[i] = E::pack(w[2 * i], w[2 * i + 1]);
                lo[i] = E::pack(w[2 * i] - E::lo(hi[i]), w[2 * i + 1] - E::hi(hi[i]));
                z = (z + w[2 * i]) + w[2 * i + 1];
            }
#pragma unroll
            for (int vb = 0; vb < VB; ++vb)
#pragma unroll
                for (int e = 0; e < VC; ++e) {
                    const u32x4 a = paged_column(x.v[vb], e);
                    acc[vb * VC + e] = mfma16<E>(a, lo, mfma16<E>(a, hi, acc[vb * VC + e]));
                }
        }
    };
    const int step = 32 * NW, key0 = s0 + 32 * wave;
    if constexpr (C::NBUF == 2) {
        PagedKeys<E, DP> x, y;
        if (key0 < s1) load(x, key0);
        for (int key = key0; key < s1; key += 2 * step) {
            if (key + step < s1) load(y, key + step);
            use(x, key);
            if (key + step >= s1) break;
            if (key + 2 * step < s1) load(x, key + 2 * step);
            use(y, key + step);
        }
    } else {
        PagedKeys<E, DP> x;
        for (int key = key0; key < s1; key += step) {
            load(x, key);
            use(x, key);
        }
    }
    // The wave's sums, without the fp16 factor.
    const float back = std::is_same<E, F16>::value ? 1.f / (cf * cf) : 1.f;
    z += __shfl_xor(z, 16);
    z += __shfl_xor(z, 32);
    if (j4 == 0) zred[wave][m] = z * back;
#pragma unroll
    for (int vb = 0; vb < VB; ++vb)
#pragma unroll
        for (int e = 0; e < VC; ++e)
#pragma unroll
            for (int r = 0; r < 4; ++r) red[wave][m][16 * VC * vb + VC * (4 * j4 + r) + e] = acc[vb * VC + e][r] * back;
    __syncthreads();
    for (int i = threadIdx.x; i < heads * (DP / 4); i += 64 * NW) {
        const int hh = i / (DP / 4), col = 4 * (i % (DP / 4));
        if (col >= p.D) continue;
        f32x4v x = *reinterpret_cast<const f32x4v*>(&red[0][hh][col]);
        float zz = zred[0][hh];
#pragma unroll
        for (int w = 1; w < NW; ++w) {
            x += *reinterpret_cast<const f32x4v*>(&red[w][hh][col]);
            zz += zred[w][hh];
        }
        const int h = h0 + hh;
        if (p.part != nullptr) {
            float* to = p.part + (((int64_t)b * p.H + h) * p.nsplit + split) * (p.D + 4);
            *reinterpret_cast<f32x4v*>(to + 4 + col) = x;
            if (col == 0) to[0] = zz;
        } else {
            x *= paged_inverse(p, h, zz);
            uint8_t* to = (uint8_t*)p.out + (((int64_t)b * p.H + h) * p.D + col) * IT;
            if constexpr (k32) {
                *reinterpret_cast<f32x4v*>(to) = x;
            } else {
                const u32x2 y = {E::pack(x[0], x[1]), E::pack(x[2], x[3])};
                *reinterpret_cast<u32x2*>(to) = y;
            }
        }
    }
}

// Numerators and denominators of a (sequence, head)'s splits.
struct PagedParts {
    const float* at;
    int n;
    __device__ __forceinline__ PagedParts(const PagedArgs& p, const PagedSpan& sp, int64_t bh)
        : at(p.part + bh * p.nsplit * (p.D + 4)), n(max(1, (sp.n - paged_base(sp) + p.chunk - 1) / p.chunk)) {}
};
// Splits joined in a fixed order: one workgroup per (sequence, head), `ncol`
// threads over the columns, 256 / ncol groups of them over the splits.
// WEIGH: in the same launch, for each (sequence, key head) and 256 keys, the
// sum over the group of p_j / Z, the heads in order, is added to its weights
// (a launch of their own behind the join took 4 us of 28, 16 sequences of up
// to 8192 keys).
template <class E, bool WEIGH>
__global__ __launch_bounds__(256) void born_paged_join_kernel(PagedArgs p, int ncol) {
    __shared__ f32x4v red[256];
    __shared__ float zred[256];
    if (WEIGH && (int)blockIdx.x >= p.B * p.H) {
        const int x = blockIdx.x - p.B * p.H, hk = x % p.Hkv, b = x / p.Hkv % p.B, block = x / p.Hkv / p.B;
        const PagedSpan sp = paged_span(p, b);
        const int j0 = paged_base(sp) + block * 256, j = j0 + threadIdx.x;
        if (j0 >= sp.n) return;
        const bool seen = j >= sp.first && j < sp.n && j < p.w_len;
        float sum = 0.f;
        for (int g0 = 0; g0 < p.G; g0 += 256) {
            const int h0 = hk * p.G + g0, gn = min(256, p.G - g0);
            if ((int)threadIdx.x < gn) {
                const PagedParts part(p, sp, (int64_t)b * p.H + h0 + threadIdx.x);
                float z = 0.f;
#pragma unroll 8
                for (int i = 0; i < part.n; ++i) z += part.at[(int64_t)i * (p.D + 4)];
                zred[threadIdx.x] = paged_inverse(p, h0 + threadIdx.x, z);
            }
            __syncthreads();
            if (seen) {
                const float* raw = p.raw + ((int64_t)b * p.H + h0) * p.raw_ld + (j - paged_base(sp));
#pragma unroll 4
                for (int i = 0; i < gn; ++i) sum = fmaf(raw[(int64_t)i * p.raw_ld], zred[i], sum);
            }
            __syncthreads();
        }
        if (seen) p.weights[(int64_t)b * p.w_sb + (int64_t)hk * p.w_sh + j] += sum;
        return;
    }
    const int h = blockIdx.x % p.H, b = blockIdx.x / p.H;
    const int col = threadIdx.x % ncol, group = threadIdx.x / ncol, groups = 256 / ncol;
    const PagedParts part(p, paged_span(p, b), (int64_t)b * p.H + h);
    const bool ok = 4 * col < p.D;
    f32x4v x = {0.f, 0.f, 0.f, 0.f};
    float z = 0.f;
#pragma unroll 4
    for (int i = group; i < part.n; i += groups) {
        const float* at = part.at + (int64_t)i * (p.D + 4);
        z += at[0];
        if (ok) x += *reinterpret_cast<const f32x4v*>(at + 4 + 4 * col);
    }
    red[threadIdx.x] = x;
    zred[threadIdx.x] = z;
    __syncthreads();
    if (group != 0 || !ok) return;
    for (int i = 1; i < groups; ++i) {
        x += red[i * ncol + col];
        z += zred[i * ncol + col];
    }
    x *= paged_inverse(p, h, z);
    uint8_t* to = (uint8_t*)p.out + (((int64_t)b * p.H + h) * p.D + 4 * col) * kItem<E>;
    if constexpr (std::is_same<E, F32>::value) {
        *reinterpret_cast<f32x4v*>(to) = x;
    } else {
        const u32x2 y = {E::pack(x[0], x[1]), E::pack(x[2], x[3])};
        *reinterpret_cast<u32x2*>(to) = y;
    }
}

template <class E>
hipError_t paged_fwd(const PagedArgs& a, hipStream_t st);

template <class E, bool WEIGH, bool P16>
void launch_paged_dp(const PagedArgs& a, hipStream_t st) {
    const dim3 grid((unsigned)(a.B * a.nsplit * a.Hkv * a.gblocks));
    if (a.D <= 64) hipLaunchKernelGGL((born_paged_kernel<E, 64, WEIGH, P16>), grid, dim3(256), 0, st, a);
    else if (a.D <= 128) hipLaunchKernelGGL((born_paged_kernel<E, 128, WEIGH, P16>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((born_paged_kernel<E, 256, WEIGH, P16>), grid, dim3(256), 0, st, a);
}

template <class E>
hipError_t launch_paged(const PagedArgs& a, hipStream_t st) {
    // Offsets within a page in 32 bits; a page 0 to send masked loads to.
    const bool p16 = a.page % 16 == 0 && a.cache_pages > 0 && a.page * a.kt < ((int64_t)1 << 31) && a.page * a.vt < ((int64_t)1 << 31);
    if (a.raw != nullptr) {
        if (p16) launch_paged_dp<E, true, true>(a, st);
        else launch_paged_dp<E, true, false>(a, st);
    } else if (p16) {
        launch_paged_dp<E, false, true>(a, st);
    } else {
        launch_paged_dp<E, false, false>(a, st);
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.part == nullptr) return e;
    int ncol = 2;
    while (4 * ncol < a.D) ncol *= 2;
    const unsigned join = (unsigned)(a.B * a.H);
    if (a.raw != nullptr) {
        const unsigned weigh = (unsigned)((a.raw_ld + 255) / 256 * a.B * a.Hkv);
        hipLaunchKernelGGL((born_paged_join_kernel<E, true>), dim3(join + weigh), dim3(256), 0, st, a, ncol);
    } else {
        hipLaunchKernelGGL((born_paged_join_kernel<E, false>), dim3(join), dim3(256), 0, st, a, ncol);
    }
    return hipGetLastError();
}

}  // namespace qdl
