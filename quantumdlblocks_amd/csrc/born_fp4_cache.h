// The 4-bit paged cache: appending a step's keys and values with the rotation
// and normalisation of its queries and keys, reading rows back, and evicting.
#pragma once

#include "born_cache.h"
#include "born_fp4.h"

namespace qdl {

// ---------------------------------------------------------------------------
// Append.  Queries as in the 16-bit cache's append: fp32, rounded once.  A key
// or value row is stored by eight columns a lane, four lanes a block:
//   e: the least with max |x| <= 7 2^e, at least -126; codes of x / 2^e to
//   nearest, halfway to even, at most 6.  e past 125 is not a number: a code of 4
//   would be infinite, as its product with a weight of 0 would not be 0.
// (Root mean square error on Gaussian rows .112; with e = floor(log2 max) - 2
// .115, without values past 6 .116, the better of two neighbours each time .112.)
//
// A key's rotation and normalisation are in 64 bits: a code is a step function
// of its value, so that its nearest value is found whatever the order of the sums.
//
// Bound by memory: 16384 tokens, 32 heads over 8, D128 bf16: 353 MB in 88 us (4.0
// TB/s); 64 single tokens, 16 heads over 4: 5.5 us.
// ---------------------------------------------------------------------------
struct Fp4AppendArgs {
    const void *q, *k, *v;
    void* q_out;
    Fp4Cache c;
    Fp4Pages t;
    const float *cos, *sin;
    const int32_t* positions;  // (N) rows of the tables, or nullptr: the slot
    const int32_t* cu;         // B + 1 starts, or nullptr: one token per sequence
    int N, B, H, Hkv, D;
    int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;  // bytes
    int table_rows, n_freq;
    int64_t freq_ld;
    int wide_tables;           // rows of whole, aligned 16-byte pieces
    double eps;
    int lpr, lpw;       // lanes of a query row, of a stored row
    int q_blocks;       // workgroups of queries; those of stored rows behind them:
    int heads, tokens;  // groups of heads, of tokens
};

// Token t's slot: its sequence and its key there; in: it belongs to one.
struct Fp4Slot {
    int s;
    int64_t slot;
    bool in;
    __device__ __forceinline__ Fp4Slot(const int32_t* cu, const int32_t* lens, int B, int t) {
        int first = t, last = t + 1;
        s = t;
        in = t < B;
        if (cu != nullptr) {
            int lo = 0, hi = B;  // the last start at or before t
            while (hi - lo > 1) {
                const int mid = (lo + hi) / 2;
                if (cu[mid] <= t) lo = mid;
                else hi = mid;
            }
            s = lo;
            in = B > 0;
            if (in) {
                first = max(cu[s], 0);
                last = cu[s + 1];
                in = t >= first && t < last;
            }
        }
        slot = in ? (int64_t)lens[s] - ((int64_t)last - t) : -1;
    }
    // Page (-1: none) and row in it.
    __device__ __forceinline__ int page(const Fp4Cache& c, const Fp4Pages& t, int& row) const {
        row = 0;
        if (slot < 0 || slot >= (int64_t)t.pages * c.page) return -1;
        const int i = fp4_page(c, (int)slot);
        row = (int)slot - i * c.page;
        const int32_t p = t.table[(int64_t)s * t.table_ld + i];
        return p >= 0 && p < c.cache_pages ? p : -1;
    }
};

// Row of the rotary tables, as an offset.
__device__ __forceinline__ int64_t fp4_angle_row(const Fp4AppendArgs& p, int t, int64_t slot) {
    const int64_t at = p.positions != nullptr ? p.positions[t] : slot;
    return min(max(at, (int64_t)0), (int64_t)p.table_rows - 1) * p.freq_ld;  // rows past the tables: their last
}

template <class E>
__device__ __forceinline__ float fp4_element(const uint8_t* row, int col) {
    if constexpr (std::is_same<E, F32>::value) {
        return *reinterpret_cast<const float*>(row + 4 * col);
    } else {
        return E::lo(*reinterpret_cast<const uint16_t*>(row + 2 * col));
    }
}
// Columns at .. at + 7 of a row as they are, zeros past D or before 0.  WHOLE: D
// is a multiple of 16, so that eight columns from a multiple of eight are one
// aligned piece, in one half of the row, or past it.
template <class E, bool WHOLE>
struct Fp4Eight {
    static constexpr int W = kItem<E> / 2;
    u32x4 u[W];
    __device__ __forceinline__ void load(const uint8_t* row, int at, int D) {
        if constexpr (WHOLE) {
#pragma unroll
            for (int i = 0; i < W; ++i) u[i] = at < D ? ldg16(row + kItem<E> * at + 16 * i) : u32x4{0u, 0u, 0u, 0u};
        } else {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = at + i >= 0 && at + i < D ? fp4_element<E>(row, at + i) : 0.f;
#pragma unroll
            for (int i = 0; i < 4 * W; ++i) {
                if constexpr (std::is_same<E, F32>::value) u[i >> 2][i & 3] = __float_as_uint(x[i]);
                else u[0][i] = E::pack(x[2 * i], x[2 * i + 1]);  // exact: they are E's
            }
        }
    }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (std::is_same<E, F32>::value) return __uint_as_float(u[i >> 2][i & 3]);
        else return (i & 1) ? E::hi(u[0][i >> 1]) : E::lo(u[0][i >> 1]);
    }
};

// The block's scale byte from its largest magnitude, kept as the upper 31 bits
// of a double's magnitude with the lower ones as a sticky bit, and the exponent
// that brings values to their codes'.
__device__ __forceinline__ int fp4_exponent(uint32_t top) {
    const int e = (int)(top >> 20) - 1023 - 2 + ((top & 0xfffffu) > 0xc0000u ? 1 : 0);
    return e > 125 ? (int)kFp4Bad - 127 : max(e, -126);
}
__device__ __forceinline__ uint32_t fp4_sticky(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    return ((uint32_t)(u >> 32) & 0x7fffffffu) | ((uint32_t)u != 0 ? 1u : 0u);
}
// x / 2^e as fp32 from its magnitude's form, sticky bit and all: halfway cases stay apart.
__device__ __forceinline__ float fp4_scaled(uint32_t h, int e, double x) {
    const int u = max((int)(h - ((uint32_t)(e + 896) << 20)), 0);
    return __uint_as_float(((uint32_t)u << 3) | ((uint32_t)(__builtin_bit_cast(uint64_t, x) >> 32) & 0x80000000u));
}

// Eight columns of a stored row: codes and, from a block's first lane, its scale.
__device__ __forceinline__ void fp4_store_row(const double (&y)[8], uint8_t* to, uint8_t* scale, int lane, bool in) {
    uint32_t u[8], top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        u[i] = fp4_sticky(y[i]);
        top = max(top, u[i]);
    }
    top = max(top, (uint32_t)__shfl_xor((int)top, 1));
    top = max(top, (uint32_t)__shfl_xor((int)top, 2));
    const int e = fp4_exponent(top);
    uint32_t codes = 0;
    if (e != (int)kFp4Bad - 127) {
#define QDL_FP4_PACK(I)                                                                                            \
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, fp4_scaled(u[2 * I], e, y[2 * I]),                       \
                                                     fp4_scaled(u[2 * I + 1], e, y[2 * I + 1]), 1.0f, I)
        QDL_FP4_PACK(0);
        QDL_FP4_PACK(1);
        QDL_FP4_PACK(2);
        QDL_FP4_PACK(3);
#undef QDL_FP4_PACK
    }
    if (!in) return;
    *reinterpret_cast<uint32_t*>(to + 4 * lane) = codes;
    if ((lane & 3) == 0) scale[lane >> 2] = (uint8_t)(e + 127);
}

// Heads of stored rows that a token's lanes go through, ROWS at a time: its slot
// and angles once for them (the 16384 tokens read back too, 8 key heads: 99 us with
// 8, 101 with 4, 115 with 2).
template <int ROWS>
constexpr int kFp4AppendHeads = ROWS > 1 ? 8 : 1;

// Angles f0 .. f0 + VEC - 1 of a row of the tables; 1 and 0 past their columns.
template <int VEC>
__device__ __forceinline__ void fp4_angles(const Fp4AppendArgs& p, int64_t row, int f0, float (&c)[VEC], float (&s)[VEC]) {
    if (p.wide_tables && f0 + VEC <= p.n_freq) {  // f0: a multiple of 4
#pragma unroll
        for (int i = 0; i < VEC; i += 4) {
            const f32x4v x = *reinterpret_cast<const f32x4v*>(p.cos + row + f0 + i), y = *reinterpret_cast<const f32x4v*>(p.sin + row + f0 + i);
#pragma unroll
            for (int e = 0; e < 4; ++e) c[i + e] = x[e], s[i + e] = y[e];
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        const bool in = p.cos != nullptr && f0 + i < p.n_freq;
        c[i] = in ? p.cos[row + f0 + i] : 1.f;
        s[i] = in ? p.sin[row + f0 + i] : 0.f;
    }
}

// Keys or values of a token: `lpw` lanes, heads from h0 on, HEADS at a time, the
// token's slot and angles found once.
template <class E, int HEADS, bool WHOLE>
__device__ __forceinline__ void fp4_append_rows(const Fp4AppendArgs& p, bool value, int t, int h0, int lane) {
    const Fp4Slot slot(p.cu, p.t.lens, p.B, t);
    int row;
    const int page = slot.page(p.c, p.t, row);
    if (page < 0) return;  // uniform in the token's lanes
    const int c0 = 8 * lane, half = p.D >> 1;
    const bool in = lane < 4 * p.c.nb;
    const Fp4Cache& c = p.c;
    const int h1 = min(h0 + kFp4AppendHeads<HEADS>, p.Hkv);
    uint8_t* const to = value ? c.v + fp4_at(page, c.vp, row, c.vt, 0, 0) : c.k + fp4_at(page, c.kp, row, c.kt, 0, 0);
    uint8_t* const scale = value ? c.vs + fp4_at(page, c.vsp, row, c.vst, 0, 0) : c.ks + fp4_at(page, c.ksp, row, c.kst, 0, 0);
    const uint32_t th = value ? c.vh : c.kh, sh = value ? c.vsh : c.ksh;
    const uint8_t* const src = value ? (const uint8_t*)p.v + (int64_t)t * p.v_st : (const uint8_t*)p.k + (int64_t)t * p.k_st;
    const int64_t hs = value ? p.v_sh : p.k_sh;
    if (value) {
        for (int h = h0; h < h1; h += HEADS) {
            Fp4Eight<E, WHOLE> x[HEADS];
#pragma unroll
            for (int i = 0; i < HEADS; ++i)
                if (h + i < h1) x[i].load(src + (h + i) * hs, c0, p.D);
#pragma unroll
            for (int i = 0; i < HEADS; ++i) {
                if (h + i >= h1) break;
                double y[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = x[i].get(e);
                fp4_store_row(y, to + (uint64_t)(h + i) * th, scale + (uint64_t)(h + i) * sh, lane, in);
            }
        }
        return;
    }
    // Columns c and c + D / 2 are a pair; where eight are of both halves, `down`
    // holds the partners of the upper half's.
    const bool both = !WHOLE && c0 < half && c0 + 8 > half;
    float cs[8], sn[8];
    const int64_t at = p.cos != nullptr ? fp4_angle_row(p, t, slot.slot) : 0;
    if (both) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int f = c0 + e < half ? c0 + e : c0 + e - half;
            const bool there = p.cos != nullptr && f < p.n_freq;
            cs[e] = there ? p.cos[at + f] : 1.f;
            sn[e] = there ? p.sin[at + f] : 0.f;
        }
    } else if (c0 < p.D) {
        fp4_angles(p, at, c0 < half ? c0 : c0 - half, cs, sn);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) cs[e] = 1.f, sn[e] = 0.f;
    }
    for (int h = h0; h < h1; h += HEADS) {
        Fp4Eight<E, WHOLE> x[HEADS], up[HEADS], down[WHOLE ? 1 : HEADS];
#pragma unroll
        for (int i = 0; i < HEADS; ++i) {
            if (h + i >= h1) break;
            const uint8_t* from = src + (h + i) * hs;
            x[i].load(from, c0, p.D);
            up[i].load(from, c0 < half ? c0 + half : c0 < p.D ? c0 - half : p.D, p.D);
            if constexpr (!WHOLE) down[i].load(from, both ? c0 - half : p.D, p.D);
        }
#pragma unroll
        for (int i = 0; i < HEADS; ++i) {
            if (h + i >= h1) break;
            double y[8], ss = 0.0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const bool low = (WHOLE ? c0 : c0 + e) < half;
                float other = up[i].get(e);
                if constexpr (!WHOLE) other = both && !low ? down[i].get(e) : other;
                y[e] = low ? (double)x[i].get(e) * cs[e] - (double)other * sn[e] : (double)other * sn[e] + (double)x[i].get(e) * cs[e];
                ss += y[e] * y[e];
            }
            if (c0 >= p.D) ss = 0.0;
            for (int o = 1; o < p.lpw; o <<= 1) ss += __shfl_xor(ss, o);
            // Quotients rounded once, as ties between codes have it: the product with
            // the reciprocal, and what it leaves of y, again, if anything (a zero keeps
            // its sign).  Denominators of 0, an infinity or NaN take the product alone.
            const double den = sqrt(ss + p.eps), f = 1.0 / den;
            const bool exact = f > 0.0 && f < HUGE_VAL;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const double g = y[e] * f, left = fma(-g, den, y[e]);
                y[e] = c0 >= p.D ? 0.0 : exact && left != 0.0 ? fma(left, f, g) : g;  // zeros: the padding of the last block, whatever the row
            }
            fp4_store_row(y, to + (uint64_t)(h + i) * th, scale + (uint64_t)(h + i) * sh, lane, in);
        }
    }
}

// Query rows: a group of `lpr` lanes each, lane i with VEC columns of the first
// half and the matching ones of the second; ROWS heads of a token a group.
template <class E, int VEC, int ROWS>
__device__ __forceinline__ void fp4_append_queries(const Fp4AppendArgs& p, int64_t item, int lane) {
    const int groups = (p.H + ROWS - 1) / ROWS;
    if (item >= (int64_t)p.N * groups) return;
    const int t = (int)(item / groups), r0 = (int)(item % groups) * ROWS, half = p.D >> 1;
    const bool own = lane * VEC < half;  // lanes of a group past the row's chunks
    const int o1 = lane * VEC * kItem<E>, o2 = o1 + half * kItem<E>;
    const Fp4Slot slot(p.cu, p.t.lens, p.B, t);
    float c[VEC], sn[VEC];
    fp4_angles(p, p.cos != nullptr ? fp4_angle_row(p, t, slot.slot) : 0, own ? lane * VEC : 0, c, sn);
    RowVec<E, VEC> x1[ROWS], x2[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        if (r0 + i >= p.H || !own) continue;
        const uint8_t* src = (const uint8_t*)p.q + (int64_t)t * p.q_st + (int64_t)(r0 + i) * p.q_sh;
        x1[i].load(src + o1);
        x2[i].load(src + o2);
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        if (r0 + i >= p.H) continue;  // uniform in the group
        float y1[VEC], y2[VEC], ss = 0.f;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float a = own ? x1[i].get(e) : 0.f, b = own ? x2[i].get(e) : 0.f;
            y1[e] = a * c[e] - b * sn[e];
            y2[e] = a * sn[e] + b * c[e];
            ss = fmaf(y1[e], y1[e], fmaf(y2[e], y2[e], ss));
        }
        for (int o = 1; o < p.lpr; o <<= 1) ss += __shfl_xor(ss, o);
        const float f = 1.0f / sqrtf(ss + (float)p.eps);
        if (!own) continue;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            // A token of no sequence has a zero query.
            y1[e] = slot.in ? y1[e] * f : 0.f;
            y2[e] = slot.in ? y2[e] * f : 0.f;
        }
        x1[i].set(y1);
        x2[i].set(y2);
        uint8_t* to = (uint8_t*)p.q_out + ((int64_t)t * p.H + r0 + i) * p.D * kItem<E>;
        x1[i].store(to + o1);
        x2[i].store(to + o2);
    }
}

template <class E, int VEC, int ROWS, bool WHOLE>
__global__ __launch_bounds__(256) void born_fp4_append_kernel(Fp4AppendArgs p) {
    if ((int)blockIdx.x < p.q_blocks) {
        fp4_append_queries<E, VEC, ROWS>(p, (int64_t)blockIdx.x * (256 / p.lpr) + threadIdx.x / p.lpr, threadIdx.x & (p.lpr - 1));
        return;
    }
    const int x = blockIdx.x - p.q_blocks;
    const int which = x / p.tokens, per = 256 / p.lpw;  // keys' groups of heads, then values'
    const int t = (x - which * p.tokens) * per + threadIdx.x / p.lpw;
    const bool value = which >= p.heads;
    if (t < p.N) fp4_append_rows<E, ROWS, WHOLE>(p, value, t, kFp4AppendHeads<ROWS> * (value ? which - p.heads : which), threadIdx.x & (p.lpw - 1));
}

// ---------------------------------------------------------------------------
// Read.  Rows (token, head) of a packed batch, each sequence's last keys, as
// values: eight columns of K and of V a lane, `lpr` lanes a token, its slot found
// once for four heads; the lanes' tokens follow each other, as a head's rows do in
// the cache.  Bound by memory: 63 thousand keys of 8 heads D128 to bf16, 326 MB in
// 66 us (4.9 TB/s); 1531 keys 4.2 us.
// ---------------------------------------------------------------------------
constexpr int kFp4ReadHeads = 4;
struct Fp4ReadArgs {
    Fp4Cache c;
    Fp4Pages t;
    const int32_t* cu;
    void *k, *v;     // (N, Hkv, D)
    int N, B, Hkv, D;
    int lpr, heads;  // lanes of a row, groups of heads
};

template <class E>
__device__ __forceinline__ void fp4_put8(uint8_t* to, uint32_t codes, float scale) {
    const u32x4 y = fp4_eight(codes, scale);  // exact in bf16
    if constexpr (std::is_same<E, BF16>::value) {
        *reinterpret_cast<u32x4*>(to) = y;
    } else if constexpr (std::is_same<E, F16>::value) {
        u32x4 z;
#pragma unroll
        for (int i = 0; i < 4; ++i) z[i] = F16::pack(BF16::lo(y[i]), BF16::hi(y[i]));
        *reinterpret_cast<u32x4*>(to) = z;
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            *reinterpret_cast<u32x4*>(to + 16 * i) = u32x4{y[2 * i] << 16, y[2 * i] & 0xffff0000u, y[2 * i + 1] << 16, y[2 * i + 1] & 0xffff0000u};
    }
}

template <class E>
__global__ __launch_bounds__(256) void born_fp4_read_kernel(Fp4ReadArgs p) {
    const int group = blockIdx.x % p.heads, h0 = kFp4ReadHeads * group, piece = threadIdx.x & (p.lpr - 1);
    const int t = blockIdx.x / p.heads * (256 / p.lpr) + threadIdx.x / p.lpr;
    if (t >= p.N || 8 * piece >= p.D) return;
    const Fp4Slot slot(p.cu, p.t.lens, p.B, t);
    int row;
    const int page = slot.page(p.c, p.t, row);
    const Fp4Cache& c = p.c;
    uint32_t k[kFp4ReadHeads], v[kFp4ReadHeads], ks[kFp4ReadHeads], vs[kFp4ReadHeads];
#pragma unroll
    for (int i = 0; i < kFp4ReadHeads; ++i) {
        k[i] = v[i] = ks[i] = vs[i] = 0;
        if (page < 0 || h0 + i >= p.Hkv) continue;
        k[i] = *reinterpret_cast<const uint32_t*>(c.k + fp4_at(page, c.kp, row, c.kt, h0 + i, c.kh) + 4 * piece);
        v[i] = *reinterpret_cast<const uint32_t*>(c.v + fp4_at(page, c.vp, row, c.vt, h0 + i, c.vh) + 4 * piece);
        ks[i] = c.ks[fp4_at(page, c.ksp, row, c.kst, h0 + i, c.ksh) + (piece >> 2)];
        vs[i] = c.vs[fp4_at(page, c.vsp, row, c.vst, h0 + i, c.vsh) + (piece >> 2)];
    }
    const int64_t at = (((int64_t)t * p.Hkv + h0) * p.D + 8 * piece) * kItem<E>;
#pragma unroll
    for (int i = 0; i < kFp4ReadHeads; ++i) {
        if (h0 + i >= p.Hkv) break;
        fp4_put8<E>((uint8_t*)p.k + at + (int64_t)i * p.D * kItem<E>, k[i], fp4_scale(ks[i]));
        fp4_put8<E>((uint8_t*)p.v + at + (int64_t)i * p.D * kItem<E>, v[i], fp4_scale(vs[i]));
    }
}

// ---------------------------------------------------------------------------
// Evict: the 16-bit cache's selection, then the move of the kept rows: a lane
// has a block of K and of V, 16 bytes of codes and a scale byte each.  16 caches cut
// from 97 thousand tokens to 4096 each, 8 key heads D128: selection 19 us, move 49
// for 140 MB of scattered rows of 64 and 4 bytes.
// ---------------------------------------------------------------------------
struct Fp4EvictArgs {
    EvictArgs s;  // the selection's, and the tables
    Fp4Cache c;
};

struct Fp4Row {
    u32x4 k, v;
    uint8_t ks, vs;
    __device__ __forceinline__ void load(const Fp4Cache& c, int page, int row, int hk, int piece, bool ok) {
        k = v = u32x4{0u, 0u, 0u, 0u};  // a missing page's rows are zeros
        ks = vs = 0;
        if (!ok) return;
        k = ldg16(c.k + fp4_at(page, c.kp, row, c.kt, hk, c.kh) + 16 * piece);
        v = ldg16(c.v + fp4_at(page, c.vp, row, c.vt, hk, c.vh) + 16 * piece);
        ks = c.ks[fp4_at(page, c.ksp, row, c.kst, hk, c.ksh) + piece];
        vs = c.vs[fp4_at(page, c.vsp, row, c.vst, hk, c.vsh) + piece];
    }
    __device__ __forceinline__ void store(const Fp4Cache& c, int page, int row, int hk, int piece) const {
        *reinterpret_cast<u32x4*>(c.k + fp4_at(page, c.kp, row, c.kt, hk, c.kh) + 16 * piece) = k;
        *reinterpret_cast<u32x4*>(c.v + fp4_at(page, c.vp, row, c.vt, hk, c.vh) + 16 * piece) = v;
        c.ks[fp4_at(page, c.ksp, row, c.kst, hk, c.ksh) + piece] = ks;
        c.vs[fp4_at(page, c.vsp, row, c.vst, hk, c.vsh) + piece] = vs;
    }
};

// Page (-1: none) and row of slot j in a table.
__device__ __forceinline__ int fp4_slot(const Fp4Cache& c, const int32_t* table, int pages, int j, int& row) {
    const int i = fp4_page(c, j);
    row = j - i * c.page;
    const int32_t p = i < pages ? table[i] : -1;
    return p >= 0 && p < c.cache_pages ? p : -1;
}

constexpr int kFp4EvictUnroll = 4;
inline __host__ __device__ int fp4_evict_rows(int nb) { return 256 / nb * kFp4EvictUnroll; }  // per workgroup

// To other pages.
template <int>
__global__ __launch_bounds__(256) void born_fp4_evict_move_kernel(Fp4EvictArgs a) {
    const EvictArgs& p = a.s;
    const int hk = blockIdx.x % p.Hkv, rest = blockIdx.x / p.Hkv, b = rest % p.B, tile = rest / p.B;
    const int m = min(evict_len(p, b), p.budget), rows = 256 / a.c.nb;
    const int mine = threadIdx.x / a.c.nb, piece = threadIdx.x % a.c.nb;
    const int i0 = tile * fp4_evict_rows(a.c.nb) + mine;
    if (mine >= rows || i0 >= m) return;
    const int32_t* kept = p.kept + ((int64_t)b * p.Hkv + hk) * p.budget;
    const int32_t *from = p.table + (int64_t)b * p.table_ld, *to = p.to + (int64_t)b * p.to_ld;
    Fp4Row x[kFp4EvictUnroll];
#pragma unroll
    for (int u = 0; u < kFp4EvictUnroll; ++u) {
        const int i = i0 + u * rows;
        int row = 0;
        const int page = i < m ? fp4_slot(a.c, from, p.pages, kept[i], row) : -1;
        x[u].load(a.c, page, row, hk, piece, page >= 0);
    }
#pragma unroll
    for (int u = 0; u < kFp4EvictUnroll; ++u) {
        const int i = i0 + u * rows;
        int row = 0;
        const int page = i < m ? fp4_slot(a.c, to, p.to_pages, i, row) : -1;
        if (page >= 0) x[u].store(a.c, page, row, hk, piece);
    }
}

// To the front of their own pages: rows only move down and keep their order, so
// one workgroup per (sequence, key head) walks them upwards: a batch is read
// whole before any of it is written, and what it writes lies below every row
// still to be read.
template <int>
__global__ __launch_bounds__(1024) void born_fp4_evict_compact_kernel(Fp4EvictArgs a) {
    constexpr int U = 4;
    const EvictArgs& p = a.s;
    const int hk = blockIdx.x % p.Hkv, b = blockIdx.x / p.Hkv;
    const int m = min(evict_len(p, b), p.budget), rows = 1024 / a.c.nb;
    const int mine = threadIdx.x / a.c.nb, piece = threadIdx.x % a.c.nb;
    const int32_t* kept = p.kept + ((int64_t)b * p.Hkv + hk) * p.budget;
    const int32_t* table = p.table + (int64_t)b * p.table_ld;
    for (int i0 = 0; i0 < m; i0 += U * rows) {
        Fp4Row x[U];
        int page[U], row[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * rows + mine;
            page[u] = -1;
            row[u] = 0;
            if (mine < rows && i < m && kept[i] != i) {
                page[u] = fp4_slot(a.c, table, p.pages, i, row[u]);
                int r;
                const int src = fp4_slot(a.c, table, p.pages, kept[i], r);
                x[u].load(a.c, src, r, hk, piece, src >= 0);
            }
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (page[u] >= 0) x[u].store(a.c, page[u], row[u], hk, piece);
        __syncthreads();
    }
}

}  // namespace qdl
