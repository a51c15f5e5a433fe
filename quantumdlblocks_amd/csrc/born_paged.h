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
    float* part;           // (B, H, nsplit, D + 1): numerators, denominator; or nullptr (one split)
    float* weights;        // (B, Hkv, L) or nullptr: += sum over the group of p / Z
    int64_t w_sb, w_sh;    // elements
    int w_len;             // columns of weights
    float* raw;            // (B, H, raw_ld) workspace: p without s^2, where weights are kept
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

// Row of key j: page and row in it; false for keys outside [first, n) and for
// pages that are none of the cache's.
__device__ __forceinline__ bool paged_row(const PagedArgs& p, const int32_t* table, PagedSpan sp, int j, int64_t& page, int& row) {
    const bool in = j >= sp.first && j < sp.n;
    const int jj = in ? j : 0;
    const int i = p.page_shift >= 0 ? jj >> p.page_shift : jj / p.page;
    row = jj - i * p.page;
    const int32_t t = in ? table[i] : -1;
    page = t;
    return t >= 0 && t < p.cache_pages;
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

// DP: 64, 128 or 256 columns; WEIGH: the raw weights are written too.
template <class E, int DP, bool WEIGH>
__global__ __launch_bounds__(256) void born_paged_kernel(PagedArgs p) {
    constexpr bool k32 = std::is_same<E, F32>::value;
    constexpr int IT = kItem<E>, NW = 4;
    // K: 16-byte chunks of a row, four lanes of a key taking chunks 4 ks + j.
    constexpr int KS = DP * IT / 64;
    // V: columns per lane and load (VC), blocks of 16 VC columns.
    constexpr int VC = k32 ? 4 : DP == 64 ? 4 : 8, VB = DP / (16 * VC), NO = VB * VC;
    __shared__ float red[NW][16][DP + 4];
    __shared__ float zred[NW][16];

    const int gb = blockIdx.x % p.gblocks, rest = blockIdx.x / p.gblocks;
    const int hk = rest % p.Hkv, rest2 = rest / p.Hkv;
    const int split = rest2 % p.nsplit, b = rest2 / p.nsplit;
    const PagedSpan sp = paged_span(p, b);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int m = lane & 15, j4 = lane >> 4;
    const int heads = min(16, p.G - 16 * gb), h0 = hk * p.G + 16 * gb;
    const int base = sp.first & ~31;  // splits count from here
    const int s0 = base + split * p.chunk, s1 = min(sp.n, s0 + p.chunk);
    if (s0 >= s1 && split > 0) return;  // the join reads the filled splits only
    const int32_t* table = p.table + (int64_t)b * p.table_ld;
    const uint8_t* const kc = (const uint8_t*)p.k + (int64_t)hk * p.kh;
    const uint8_t* const vc = (const uint8_t*)p.v + (int64_t)hk * p.vh;

    // Query head h0 + m in the columns of S^T.
    const bool okh = m < heads;
    const float sc = arg_scale(p, okh ? h0 + m : h0);
    const uint32_t flip = packed_flip<E>(sc);
    u32x4 qr[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        const int at = 16 * (4 * ks + j4);
        u32x4 x = {0u, 0u, 0u, 0u};
        if (okh && at < IT * p.D) x = ldg16((const uint8_t*)p.q + (int64_t)b * p.q_sb + (int64_t)(h0 + m) * p.q_sh + at);
        qr[ks] = x ^ flip;
    }
    f32x4v acc[NO];
#pragma unroll
    for (int i = 0; i < NO; ++i) acc[i] = f32x4v{0.f, 0.f, 0.f, 0.f};
    float z = 0.f, cf = std::is_same<E, F16>::value ? kF16Start : 1.f;

    for (int key0 = s0 + 32 * wave; key0 < s1; key0 += 32 * NW) {
        // Keys of this lane: rows key0 + m and + 16 for K, key0 + 4 j4 + i and
        // + 16 for V.
        u32x4 kx[2][KS];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            int64_t page;
            int row;
            const bool ok = paged_row(p, table, sp, key0 + 16 * t + m, page, row);
            const uint8_t* at = kc + page * p.kp + (int64_t)row * p.kt;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const int o = 16 * (4 * ks + j4);
                u32x4 x = {0u, 0u, 0u, 0u};
                if (ok && o < IT * p.D) x = ldg16(at + o);
                kx[t][ks] = x;
            }
        }
        u32x4 vx[VB][8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            int64_t page;
            int row;
            const bool ok = paged_row(p, table, sp, key0 + 16 * (i >> 2) + 4 * j4 + (i & 3), page, row);
            const uint8_t* at = vc + page * p.vp + (int64_t)row * p.vt;
#pragma unroll
            for (int vb = 0; vb < VB; ++vb) {
                const int col = 16 * VC * vb + VC * m;
                u32x4 x = {0u, 0u, 0u, 0u};
                if (ok && col < p.D) {
                    if constexpr (VC * IT == 16) {
                        x = ldg16(at + IT * col);
                    } else {
                        const u32x2 y = *reinterpret_cast<const u32x2*>(at + IT * col);
                        x[0] = y[0];
                        x[1] = y[1];
                    }
                }
                vx[vb][i] = x;
            }
        }
        f32x4v s[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            s[t] = f32x4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                if constexpr (k32) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[t] = mfma16_f32(__uint_as_float(kx[t][ks][i]), __uint_as_float(qr[ks][i]), s[t]);
                } else {
                    s[t] = mfma16<E>(kx[t][ks], qr[ks], s[t]);
                }
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
                    const int key = key0 + 16 * t + 4 * j4;
                    float* to = p.raw + ((int64_t)b * p.H + h0 + m) * p.raw_ld + key;
                    const f32x4v x = {w[4 * t] * back, w[4 * t + 1] * back, w[4 * t + 2] * back, w[4 * t + 3] * back};
                    if (key < p.raw_ld) *reinterpret_cast<f32x4v*>(to) = x;  // raw_ld: a multiple of 32
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
                        acc[vb * VC + e] = mfma16_f32(__uint_as_float(vx[vb][i][e]), w[i], acc[vb * VC + e]);
            }
        } else {
            u32x4 pk;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                pk[i] = E::pack(w[2 * i], w[2 * i + 1]);  // the product's operand; the sum takes them as they are
                z = (z + w[2 * i]) + w[2 * i + 1];
            }
#pragma unroll
            for (int vb = 0; vb < VB; ++vb)
#pragma unroll
                for (int e = 0; e < VC; ++e) acc[vb * VC + e] = mfma16<E>(paged_column(vx[vb], e), pk, acc[vb * VC + e]);
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
            const float s = arg_scale(p, h), den = zz + (p.eps == 0.f ? 0.f : p.eps / (s * s));
            x *= den > 0.f && s != 0.f ? 1.0f / den : 0.f;
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

// Splits joined in order.  One workgroup per (sequence, head).
template <class E>
__global__ __launch_bounds__(64) void born_paged_join_kernel(PagedArgs p) {
    const int h = blockIdx.x % p.H, b = blockIdx.x / p.H;
    const PagedSpan sp = paged_span(p, b);
    const int n = max(1, (sp.n - (sp.first & ~31) + p.chunk - 1) / p.chunk);
    const float* part = p.part + ((int64_t)b * p.H + h) * p.nsplit * (p.D + 4);
    const float s = arg_scale(p, h);
    float z = 0.f;
    for (int i = 0; i < n; ++i) z += part[(int64_t)i * (p.D + 4)];
    const float den = z + (p.eps == 0.f ? 0.f : p.eps / (s * s));
    const float inv = den > 0.f && s != 0.f ? 1.0f / den : 0.f;
    for (int col = 4 * threadIdx.x; col < p.D; col += 256) {
        f32x4v x = {0.f, 0.f, 0.f, 0.f};
        for (int i = 0; i < n; ++i) x += *reinterpret_cast<const f32x4v*>(part + (int64_t)i * (p.D + 4) + 4 + col);
        x *= inv;
        uint8_t* to = (uint8_t*)p.out + (((int64_t)b * p.H + h) * p.D + col) * kItem<E>;
        if constexpr (std::is_same<E, F32>::value) {
            *reinterpret_cast<f32x4v*>(to) = x;
        } else {
            const u32x2 y = {E::pack(x[0], x[1]), E::pack(x[2], x[3])};
            *reinterpret_cast<u32x2*>(to) = y;
        }
    }
}

// weights[b][hk][j] += sum over the group of p_j / Z, the heads in order, 256
// keys per workgroup.
template <int>
__global__ __launch_bounds__(256) void born_paged_weigh_kernel(PagedArgs p) {
    __shared__ float inv[256];
    const int hk = blockIdx.x % p.Hkv, rest = blockIdx.x / p.Hkv;
    const int b = rest % p.B, block = rest / p.B;
    const PagedSpan sp = paged_span(p, b);
    const int base = sp.first & ~31;
    const int j = base + block * 256 + threadIdx.x;
    if (base + block * 256 >= sp.n) return;
    const int n = max(1, (sp.n - base + p.chunk - 1) / p.chunk);
    float sum = 0.f;
    for (int g0 = 0; g0 < p.G; g0 += 256) {
        const int gn = min(256, p.G - g0);
        if ((int)threadIdx.x < gn) {
            const int h = hk * p.G + g0 + threadIdx.x;
            const float* part = p.part + ((int64_t)b * p.H + h) * p.nsplit * (p.D + 4);
            const float s = arg_scale(p, h);
            float z = 0.f;
            for (int i = 0; i < n; ++i) z += part[(int64_t)i * (p.D + 4)];
            const float den = z + (p.eps == 0.f ? 0.f : p.eps / (s * s));
            inv[threadIdx.x] = den > 0.f && s != 0.f ? 1.0f / den : 0.f;
        }
        __syncthreads();
        if (j >= sp.first && j < sp.n && j < p.w_len) {
            const float* raw = p.raw + ((int64_t)b * p.H + hk * p.G + g0) * p.raw_ld + j;
            for (int i = 0; i < gn; ++i) sum = fmaf(raw[(int64_t)i * p.raw_ld], inv[i], sum);
        }
        __syncthreads();
    }
    if (j >= sp.first && j < sp.n && j < p.w_len) p.weights[(int64_t)b * p.w_sb + (int64_t)hk * p.w_sh + j] += sum;
}

template <class E>
hipError_t paged_fwd(const PagedArgs& a, hipStream_t st);

template <class E, bool WEIGH>
hipError_t launch_paged_dp(const PagedArgs& a, hipStream_t st) {
    const dim3 grid((unsigned)(a.B * a.nsplit * a.Hkv * a.gblocks));
    if (a.D <= 64) hipLaunchKernelGGL((born_paged_kernel<E, 64, WEIGH>), grid, dim3(256), 0, st, a);
    else if (a.D <= 128) hipLaunchKernelGGL((born_paged_kernel<E, 128, WEIGH>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((born_paged_kernel<E, 256, WEIGH>), grid, dim3(256), 0, st, a);
    return hipGetLastError();
}

template <class E>
hipError_t launch_paged(const PagedArgs& a, hipStream_t st) {
    hipError_t e = a.raw != nullptr ? launch_paged_dp<E, true>(a, st) : launch_paged_dp<E, false>(a, st);
    if (e != hipSuccess || a.part == nullptr) return e;
    hipLaunchKernelGGL((born_paged_join_kernel<E>), dim3((unsigned)(a.B * a.H)), dim3(64), 0, st, a);
    e = hipGetLastError();
    if (e != hipSuccess || a.raw == nullptr) return e;
    const int64_t span = a.window > 0 && a.window + 32 < a.raw_ld ? a.window + 32 : a.raw_ld;
    hipLaunchKernelGGL((born_paged_weigh_kernel<0>), dim3((unsigned)((span + 255) / 256 * a.B * a.Hkv)), dim3(256), 0, st, a);
    return hipGetLastError();
}

}  // namespace qdl
