// Born attention over packed sequences with grouped heads: forward, dQ and
// dK/dV for rows of tokens (N, H, D) that several sequences of different
// lengths share, G = H / Hkv query heads reading one key head.
//
//   r_ij = q_i . k_j,  p_ij = (s relu(sign(s) r_ij))^2 M_ij,
//   Z_i = sum_j p_ij + eps,  O_i = sum_j p_ij v_j / Z_i,
//   M_ij = [lower <= (i + len_k - len_q) - j < upper]
// with i, j counted from the sequence's own starts (causal: lower = 0; a
// window: upper = window).  The scale is folded out of the tile loop: p' =
// relu(r)^2 and s^2 once per row.  Backward, with zs = s^2 / Z and delta_i =
// dO_i . O_i:
//   u_ij = relu(r_ij) zs_i (dO_i . v_j - delta_i),  dQ_i = 2 sign(s) sum_j u_ij k_j,
//   dK_j = 2 sign(s) sum_i u_ij q_i,  dV_j = sum_i relu(r_ij)^2 zs_i dO_i,
// the last two over the queries of all G heads of the group, in a fixed order.
//
// What bounds them: the matrix pipe.  A workgroup's four waves own 32
// stationary rows each (queries in the forward and dQ, keys in dK/dV) and
// share the tiles of the streamed operands, which LDS-DMA loads bring into a
// ring of stages, one barrier per tile.  The weights of a row have no running
// maximum, so nothing but the sums passes from tile to tile.
//
// Blocks: sequence s takes the block slots from cu[s] / BM + s on.  Since
// ceil(len / BM) <= cu[s+1] / BM - cu[s] / BM + 1 they never overlap, so the
// grid follows from N and S alone (no copy of the lengths to the host, no list
// made by another launch), and a block finds its sequence by a 64-way search.
// Slots without rows end at once.  The rows behind the last sequence belong to
// a sequence of their own without keys: zero outputs and gradients.
#pragma once

#include <type_traits>

#include "born_common.h"
#include "born_fwd_fast.h"

namespace qdl {

struct F32 {
    static constexpr int kDtype = 0;
};

template <class E>
constexpr int kItem = std::is_same<E, F32>::value ? 4 : 2;

// Argument block of the packed kernels.  Strides are in bytes.
struct PackedArgs {
    const void *q, *k, *v, *o, *dout;
    void *out, *dq, *dk, *dv;
    float* z;       // (H, Nq), or nullptr: no backward follows
    float* ndelta;  // (H, Nq) workspace: -(dO . O)
    float* zs;      // (H, Nq) workspace: s^2 / Z
    const float* scale;  // 1 or H values, or nullptr: scale_value
    float scale_value;
    int per_head_scale;
    const int32_t *cu_q, *cu_k;  // S + 1 starts
    int S, Nq, Nk, H, Hkv, G, D;
    int lower, upper;  // visible: lower <= query position - key < upper
    float eps;
    int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh, do_st, do_sh;
};

constexpr int kPackedWaves = 4;
constexpr int kPackedRows = 32 * kPackedWaves;  // stationary rows per workgroup

// A sequence's rows: queries q0 .. q0 + nq - 1, keys k0 .. k0 + nk - 1.
struct PackedSeq {
    int q0, nq, k0, nk;
    int tile;  // this block's tile within it
};

__device__ __forceinline__ int packed_start(const int32_t* cu, int s, int N) {
    return s == 0 ? 0 : min(max(cu[s], 0), N);
}

// The sequence and tile of block slot x, slots counted along `cu` (N rows).
__device__ __forceinline__ int packed_find(const int32_t* cu, int S, int N, int x) {
    const int lane = threadIdx.x & 63;
    int lo = 0, hi = S + 1;
    while (hi - lo > 1) {
        const int step = (hi - lo + 63) / 64;
        const int s = lo + (lane + 1) * step;
        const bool below = s < hi && packed_start(cu, s, N) / kPackedRows + s <= x;
        lo += (int)__popcll(__ballot(below)) * step;
        hi = min(hi, lo + step);
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

template <bool KEYS>
__device__ __forceinline__ PackedSeq packed_seq(const PackedArgs& p, int x) {
    const int32_t* cu = KEYS ? p.cu_k : p.cu_q;
    const int N = KEYS ? p.Nk : p.Nq;
    const int s = packed_find(cu, p.S, N, x);
    PackedSeq r;
    r.q0 = r.k0 = r.nq = r.nk = 0;
    if (s < p.S) {
        r.q0 = packed_start(p.cu_q, s, p.Nq);
        r.nq = max(packed_start(p.cu_q, s + 1, p.Nq) - r.q0, 0);
        r.k0 = packed_start(p.cu_k, s, p.Nk);
        r.nk = max(packed_start(p.cu_k, s + 1, p.Nk) - r.k0, 0);
    } else if (KEYS) {  // behind the last sequence
        r.k0 = packed_start(cu, s, N);
        r.nk = N - r.k0;
    } else {
        r.q0 = packed_start(cu, s, N);
        r.nq = N - r.q0;
    }
    r.tile = x - (packed_start(cu, s, N) / kPackedRows + s);
    return r;
}

// ROWS rows of one streamed operand in LDS: 16-byte chunks XOR-swizzled per
// row so that neither a row read (16 rows, one chunk) nor a transposed read (4
// consecutive rows, 64 bytes each) meets a bank twice: rows that all start on
// bank 0 by all four bits of the row, rows of alternating halves by lds_swz,
// rows on four starts by the row's upper bits.
template <class E, int DP, int ROWS>
struct PackedTile {
    static constexpr int IT = kItem<E>, RB = IT * DP, CPR = RB / 16, BYTES = ROWS * RB;
    static constexpr int LPW = BYTES / (1024 * kPackedWaves);  // 1-KiB loads per wave
    static constexpr int KS = RB / 32, DB = DP / 32;
    static_assert(BYTES % (1024 * kPackedWaves) == 0, "whole loads per wave");
    uint8_t* lds;
    __device__ __forceinline__ static int swz(int row) {
        if constexpr (RB % 256 == 0) return ((row & 3) << 2) | ((row >> 2) & 3);
        else if constexpr (RB % 256 == 128) return lds_swz(row);
        else return (row >> 2) & 3;
    }
    // Byte offsets of this lane's loads within ROWS rows of `stride` bytes;
    // columns past D read out of range (zeros).
    __device__ __forceinline__ static void offsets(int (&off)[LPW], int stride, int D, int wave, int lane) {
#pragma unroll
        for (int i = 0; i < LPW; ++i) {
            const int slot = (wave * LPW + i) * 64 + lane, row = slot / CPR, chunk = (slot % CPR) ^ swz(row);
            off[i] = 16 * chunk < IT * D ? row * stride + 16 * chunk : kBufOOB;
        }
    }
    // `left` rows from `at` on; rows past them are zeros.
    __device__ __forceinline__ void issue(const uint8_t* at, int left, int stride, int D, const int (&off)[LPW], int wave) const {
        const int rows = min(left, ROWS);
        i32x4 rs = buffer_rsrc(at, rows > 0 ? (uint32_t)(rows - 1) * (uint32_t)stride + (uint32_t)(IT * D) : 0u);
#pragma unroll
        for (int i = 0; i < 4; ++i) rs[i] = __builtin_amdgcn_readfirstlane(rs[i]);
#pragma unroll
        for (int i = 0; i < LPW; ++i) dma_load16(rs, lds_addr(lds + (wave * LPW + i) * 1024), off[i]);
    }
    // A operand of a contraction over the head dim: row, chunk 2 ks + g.
    __device__ __forceinline__ u32x4 row(int r, int ks, int g) const {
        return *reinterpret_cast<const u32x4*>(lds + r * RB + (((2 * ks + g) ^ swz(r)) << 4));
    }
    // A operand of a contraction over the rows r0 .. r0 + 15 in the
    // accumulators' row order (16-bit): columns 32 db .. + 31 across the lanes.
    __device__ __forceinline__ u32x4 transposed(int r0, int db, int lane) const {
        const int r = r0 + 4 * (lane >> 5) + ((lane & 15) >> 2);
        const int col = 32 * db + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
        auto at = [&](int row) {
            return reinterpret_cast<const uint16_t*>(lds + row * RB + (((col >> 3) ^ swz(row)) << 4) + (col & 7) * 2);
        };
        const u32x2 x = lds_read_tr16(at(r)), y = lds_read_tr16(at(r + 8));
        const u32x4 a = {x[0], x[1], y[0], y[1]};
        return a;
    }
    // fp32: row r, columns 32 db + c.
    __device__ __forceinline__ float scalar(int r, int db, int c) const {
        const int col = 32 * db + c;
        return *reinterpret_cast<const float*>(lds + r * RB + (((col >> 2) ^ swz(r)) << 4) + 4 * (col & 3));
    }
};

// The 16 values that a lane holds of a 32 x 32 product, as the B operand of the
// next one: packed to 16 bits, or as they are.
template <class E>
struct PackedWeights {
    uint32_t w[8];
    __device__ __forceinline__ void set(int j, float x, float y) { w[j] = E::pack(x, y); }
};
template <>
struct PackedWeights<F32> {
    float w[16];
    __device__ __forceinline__ void set(int j, float x, float y) { w[2 * j] = x, w[2 * j + 1] = y; }
};

// acc += a . b over one 32-byte step of the head dim.
template <class E>
__device__ __forceinline__ f32x16 packed_step(u32x4 a, u32x4 b, f32x16 acc) {
    if constexpr (std::is_same<E, F32>::value) {
#pragma unroll
        for (int i = 0; i < 4; ++i) acc = mfma_f32(__uint_as_float(a[i]), __uint_as_float(b[i]), acc);
        return acc;
    } else {
        return E::mfma(a, b, acc);
    }
}

// acc[db] += (rows r0 .. r0 + 31 of the tile)^T . w.
template <class E, class Tile, int DB>
__device__ __forceinline__ void packed_columns(const Tile& t, int r0, const PackedWeights<E>& w, f32x16 (&acc)[DB], int lane) {
    if constexpr (std::is_same<E, F32>::value) {
        const int c = lane & 31, g = lane >> 5;
#pragma unroll
        for (int r = 0; r < 16; ++r)
#pragma unroll
            for (int db = 0; db < DB; ++db) acc[db] = mfma_f32(t.scalar(r0 + acc_row(r, g), db, c), w.w[r], acc[db]);
    } else {
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
            const u32x4 b = {w.w[4 * hh], w.w[4 * hh + 1], w.w[4 * hh + 2], w.w[4 * hh + 3]};
#pragma unroll
            for (int db = 0; db < DB; ++db) acc[db] = E::mfma(t.transposed(r0 + 16 * hh, db, lane), b, acc[db]);
        }
    }
}

// A stationary row as B operands: lane (c, g) holds its row's chunks 2 ks + g,
// zeros past the rows and past D.
template <class E, int KS>
__device__ __forceinline__ void packed_load_row(u32x4 (&x)[KS], const uint8_t* row, bool ok, int D, int g) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        const int at = 32 * ks + 16 * g;
        u32x4 y = {0u, 0u, 0u, 0u};
        if (ok && at < kItem<E> * D) y = ldg16(row + at);
        x[ks] = y;
    }
}

// 0 or the sign bits of one 32-bit word of E.
template <class E>
__device__ __forceinline__ uint32_t packed_flip(float s) {
    return s < 0.f ? (std::is_same<E, F32>::value ? 0x80000000u : 0x80008000u) : 0u;
}

// One row of 32 db + 8 j + 4 g + e columns from the accumulators.
template <class E, int DB>
__device__ __forceinline__ void packed_store_row(uint8_t* row, const f32x16 (&acc)[DB], float f, int D, int g) {
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int col = 32 * db + 8 * j + 4 * g;
            if (col >= D) continue;
            const f32x16& a = acc[db];
            const f32x4 w = {a[4 * j] * f, a[4 * j + 1] * f, a[4 * j + 2] * f, a[4 * j + 3] * f};
            if constexpr (std::is_same<E, F32>::value) {
                *reinterpret_cast<f32x4*>(row + 4 * col) = w;
            } else {
                const u32x2 x = {E::pack(w[0], w[1]), E::pack(w[2], w[3])};
                *reinterpret_cast<u32x2*>(row + 2 * col) = x;
            }
        }
}

// fp16 weights: relu(r)^2 leaves fp16's range where |r| passes 255 and its
// normal range below 2^-7, so a row's overlaps are scaled by a power of two c
// that keeps the largest so far under 255.  c starts far up; where a tile's
// largest overlap would pass the bound, c drops to bring it to [64, 128) and
// what the row has summed is scaled by the square of the change, exactly.
constexpr float kF16Start = 0x1p60f;
__device__ __forceinline__ float f16_factor(float largest) {
    const int e = (int)((__float_as_uint(largest) >> 23) & 255u) - 127;
    return __uint_as_float((uint32_t)(min(max(6 - e, -126), 127) + 127) << 23);
}

// fp16 gradients' operands: p / Z is at most 1 and the factor of dS has no
// bound; these powers of two keep small ones in fp16's normal range.
template <class E>
constexpr float kUpW = std::is_same<E, F16>::value ? 1024.f : 1.f;
template <class E>
constexpr float kUpU = std::is_same<E, F16>::value ? 64.f : 1.f;

template <class E, int DP>
struct PackedCfg {
    static constexpr bool k16 = kItem<E> == 2;
    static constexpr int BN = k16 && DP <= 128 ? 64 : 32;  // streamed rows per tile
    static constexpr int RB = kItem<E> * DP;
    static constexpr int STAGE = 2 * BN * RB;              // two operands
    // 16-bit up to head dim 128: two workgroups per CU; above and fp32, one.
    static constexpr int NST = 2;
    static constexpr int WPE = RB <= 256 ? 2 : 1;
};

// ---------------------------------------------------------------------------
// Forward: S^T = K Q^T per 32 keys, the weights in place, O^T += V^T P^T.
// ---------------------------------------------------------------------------
template <class E, int DP>
__global__ __launch_bounds__(64 * kPackedWaves) __attribute__((amdgpu_waves_per_eu(PackedCfg<E, DP>::WPE, PackedCfg<E, DP>::WPE)))
void born_packed_fwd_kernel(PackedArgs p) {
    using C = PackedCfg<E, DP>;
    using Tile = PackedTile<E, DP, C::BN>;
    constexpr int KS = Tile::KS, DB = Tile::DB, BN = C::BN, NST = C::NST, BM = kPackedRows;
    __shared__ __attribute__((aligned(1024))) uint8_t ring[NST * C::STAGE];

    const int slots = p.Nq / BM + p.S + 1;
    const int hk = blockIdx.x % p.Hkv, rest = blockIdx.x / p.Hkv;
    const int h = hk * p.G + rest % p.G;
    const PackedSeq sq = packed_seq<false>(p, slots - 1 - rest / p.G);
    const int m0 = sq.tile * BM;
    if (m0 >= sq.nq) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 31, g = lane >> 5;
    const int D = p.D, off = sq.nk - sq.nq;
    const float sc = arg_scale(p, h);

    // Keys that the block's rows see, as tiles of BN.
    const int m1 = min(sq.nq, m0 + BM);
    const int jlo = max(0, m0 + off - p.upper + 1), jhi = min(sq.nk - 1, m1 - 1 + off - p.lower);
    const int t0 = jlo / BN, n = jhi >= jlo ? jhi / BN - t0 + 1 : 0;

    const uint8_t* const kb = (const uint8_t*)p.k + (int64_t)sq.k0 * p.k_st + (int64_t)hk * p.k_sh;
    const uint8_t* const vb = (const uint8_t*)p.v + (int64_t)sq.k0 * p.v_st + (int64_t)hk * p.v_sh;
    int koff[Tile::LPW], voff[Tile::LPW];
    Tile::offsets(koff, (int)p.k_st, D, wave, lane);
    Tile::offsets(voff, (int)p.v_st, D, wave, lane);
    auto kt = [&](int st) { return Tile{ring + st * C::STAGE}; };
    auto vt = [&](int st) { return Tile{ring + st * C::STAGE + Tile::BYTES}; };
    auto issue = [&](int u, int st) __attribute__((always_inline)) {
        const int key0 = (t0 + u) * BN;
        kt(st).issue(kb + (int64_t)key0 * p.k_st, sq.nk - key0, (int)p.k_st, D, koff, wave);
        vt(st).issue(vb + (int64_t)key0 * p.v_st, sq.nk - key0, (int)p.v_st, D, voff, wave);
    };

    const int rw = m0 + 32 * wave, row = rw + c;
    const bool ok = row < sq.nq;
    u32x4 qr[KS];
    packed_load_row<E>(qr, (const uint8_t*)p.q + (int64_t)(sq.q0 + row) * p.q_st + (int64_t)h * p.q_sh, ok, D, g);
    const uint32_t flip = packed_flip<E>(sc);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        qr[ks] ^= flip;
        asm volatile("" : "+v"(qr[ks]));  // landed before the ring's loads are counted
    }
    f32x16 acc[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db) acc[db] = zero16();
    float z = 0.f, cf = kF16Start;
    const int pos = row + off, span = p.upper - p.lower;

    if (n > 0) issue(0, 0);
    for (int u = 0; u < n; ++u) {
        const int st = u % NST, key0 = (t0 + u) * BN;
        wait_vmcnt<0>();
        __syncthreads();
        if (u + 1 < n) issue(u + 1, (u + 1) % NST);
        const bool none = key0 > rw + 31 + off - p.lower || key0 + BN <= rw + off - p.upper + 1;
        if (none) continue;
        const bool cut = key0 + BN - 1 > rw + off - p.lower || key0 < rw + 31 + off - p.upper + 1;
#pragma unroll
        for (int nb = 0; nb < BN / 32; ++nb) {
            f32x16 s = zero16();
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) s = packed_step<E>(kt(st).row(32 * nb + c, ks, g), qr[ks], s);
            if (cut) {
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if ((uint32_t)(pos - (key0 + 32 * nb + acc_row(r, g)) - p.lower) >= (uint32_t)span) s[r] = 0.f;
            }
            PackedWeights<E> w;
            if constexpr (std::is_same<E, F32>::value) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float a = relu_f32(s[r]);
                    w.w[r] = a * a;
                    z += w.w[r];
                }
            } else if constexpr (std::is_same<E, F16>::value) {
                float m = 0.f;
#pragma unroll
                for (int r = 0; r < 16; ++r) m = fmaxf(m, s[r]);
                m = fmaxf(m, __shfl_xor(m, 32));
                if (__ballot(m * cf > 255.f) != 0) {
                    const float to = m * cf > 255.f ? f16_factor(m) : cf;
                    const float by = (to / cf) * (to / cf);
                    cf = to;
                    z *= by;
#pragma unroll
                    for (int db = 0; db < DB; ++db) acc[db] *= by;
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) w.w[j] = born_weight_pair<F16>(s[2 * j], s[2 * j + 1], cf, z);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) w.w[j] = born_weight_pair<BF16>(s[2 * j], s[2 * j + 1], 1.f, z);
            }
            packed_columns<E>(vt(st), 32 * nb, w, acc, lane);
        }
    }

    z += __shfl_xor(z, 32);
    const float s1 = std::is_same<E, F16>::value ? sc / cf : sc, s2 = s1 * s1;
    const float den = z + (p.eps == 0.f ? 0.f : p.eps / s2);
    const float inv = den > 0.f && sc != 0.f ? 1.0f / den : 0.f;
    if (!ok) return;
    packed_store_row<E>((uint8_t*)p.out + ((size_t)(sq.q0 + row) * p.H + h) * D * kItem<E>, acc, inv, D, g);
    if (g == 0 && p.z != nullptr) p.z[(size_t)h * p.Nq + sq.q0 + row] = s2 * z + p.eps;
}

// ---------------------------------------------------------------------------
// dQ; also -delta and s^2 / Z per row for the dK/dV kernel.
// ---------------------------------------------------------------------------
template <class E, int DP>
__global__ __launch_bounds__(64 * kPackedWaves) __attribute__((amdgpu_waves_per_eu(PackedCfg<E, DP>::WPE, PackedCfg<E, DP>::WPE)))
void born_packed_dq_kernel(PackedArgs p) {
    using C = PackedCfg<E, DP>;
    using Tile = PackedTile<E, DP, C::BN>;
    constexpr int KS = Tile::KS, DB = Tile::DB, BN = C::BN, NST = C::NST, BM = kPackedRows, IT = kItem<E>;
    __shared__ __attribute__((aligned(1024))) uint8_t ring[NST * C::STAGE];

    const int slots = p.Nq / BM + p.S + 1;
    const int hk = blockIdx.x % p.Hkv, rest = blockIdx.x / p.Hkv;
    const int h = hk * p.G + rest % p.G;
    const PackedSeq sq = packed_seq<false>(p, slots - 1 - rest / p.G);
    const int m0 = sq.tile * BM;
    if (m0 >= sq.nq) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 31, g = lane >> 5;
    const int D = p.D, off = sq.nk - sq.nq;
    const float sc = arg_scale(p, h);

    const int m1 = min(sq.nq, m0 + BM);
    const int jlo = max(0, m0 + off - p.upper + 1), jhi = min(sq.nk - 1, m1 - 1 + off - p.lower);
    const int t0 = jlo / BN, n = jhi >= jlo ? jhi / BN - t0 + 1 : 0;

    const uint8_t* const kb = (const uint8_t*)p.k + (int64_t)sq.k0 * p.k_st + (int64_t)hk * p.k_sh;
    const uint8_t* const vb = (const uint8_t*)p.v + (int64_t)sq.k0 * p.v_st + (int64_t)hk * p.v_sh;
    int koff[Tile::LPW], voff[Tile::LPW];
    Tile::offsets(koff, (int)p.k_st, D, wave, lane);
    Tile::offsets(voff, (int)p.v_st, D, wave, lane);
    auto kt = [&](int st) { return Tile{ring + st * C::STAGE}; };
    auto vt = [&](int st) { return Tile{ring + st * C::STAGE + Tile::BYTES}; };
    auto issue = [&](int u, int st) __attribute__((always_inline)) {
        const int key0 = (t0 + u) * BN;
        kt(st).issue(kb + (int64_t)key0 * p.k_st, sq.nk - key0, (int)p.k_st, D, koff, wave);
        vt(st).issue(vb + (int64_t)key0 * p.v_st, sq.nk - key0, (int)p.v_st, D, voff, wave);
    };

    const int rw = m0 + 32 * wave, row = rw + c;
    const bool ok = row < sq.nq;
    u32x4 qr[KS], dr[KS];
    packed_load_row<E>(qr, (const uint8_t*)p.q + (int64_t)(sq.q0 + row) * p.q_st + (int64_t)h * p.q_sh, ok, D, g);
    packed_load_row<E>(dr, (const uint8_t*)p.dout + (int64_t)(sq.q0 + row) * p.do_st + (int64_t)h * p.do_sh, ok, D, g);
    const size_t at = ((size_t)(sq.q0 + row) * p.H + h) * D * IT;  // contiguous (Nq, H, D)
    float delta = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        const int b = 32 * ks + 16 * g;
        if (!ok || b >= IT * D) continue;
        const u32x4 o = ldg16((const uint8_t*)p.o + at + b);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (std::is_same<E, F32>::value) delta = fmaf(__uint_as_float(o[j]), __uint_as_float(dr[ks][j]), delta);
            else delta += E::lo(o[j]) * E::lo(dr[ks][j]) + E::hi(o[j]) * E::hi(dr[ks][j]);
        }
    }
    delta += __shfl_xor(delta, 32);
    const size_t stat = (size_t)h * p.Nq + sq.q0 + row;
    const float zr = ok ? p.z[stat] : 1.f;
    const float zs = zr > 0.f ? sc * sc / zr : 0.f;
    if (ok && g == 0) {
        p.ndelta[stat] = -delta;
        p.zs[stat] = zs;
    }
    const uint32_t flip = packed_flip<E>(sc);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        qr[ks] ^= flip;
        asm volatile("" : "+v"(qr[ks]), "+v"(dr[ks]));
    }
    f32x16 acc[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db) acc[db] = zero16();
    // fp16 scales each operand into its range; otherwise zs is a row's factor.
    const float pre = std::is_same<E, F16>::value ? kUpU<E> * zs : 1.f;
    const int pos = row + off, span = p.upper - p.lower;
    asm volatile("" : "+v"(delta));

    if (n > 0) issue(0, 0);
    for (int u = 0; u < n; ++u) {
        const int st = u % NST, key0 = (t0 + u) * BN;
        wait_vmcnt<0>();
        __syncthreads();
        if (u + 1 < n) issue(u + 1, (u + 1) % NST);
        const bool none = key0 > rw + 31 + off - p.lower || key0 + BN <= rw + off - p.upper + 1;
        if (none) continue;
        const bool cut = key0 + BN - 1 > rw + off - p.lower || key0 < rw + 31 + off - p.upper + 1;
#pragma unroll
        for (int nb = 0; nb < BN / 32; ++nb) {
            f32x16 s = zero16(), t;
#pragma unroll
            for (int r = 0; r < 16; ++r) t[r] = -delta;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                s = packed_step<E>(kt(st).row(32 * nb + c, ks, g), qr[ks], s);
                t = packed_step<E>(vt(st).row(32 * nb + c, ks, g), dr[ks], t);
            }
            if (cut) {
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if ((uint32_t)(pos - (key0 + 32 * nb + acc_row(r, g)) - p.lower) >= (uint32_t)span) s[r] = 0.f;
            }
            PackedWeights<E> w;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float x[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float a = relu_f32(s[2 * j + e]);
                    x[e] = (std::is_same<E, F16>::value ? a * pre : a) * t[2 * j + e];
                }
                w.set(j, x[0], x[1]);
            }
            packed_columns<E>(kt(st), 32 * nb, w, acc, lane);
        }
    }
    if (!ok) return;
    const float f = (sc < 0.f ? -2.f : 2.f) * (std::is_same<E, F16>::value ? 1.f / kUpU<E> : zs);
    packed_store_row<E>((uint8_t*)p.dq + at, acc, f, D, g);
}

// ---------------------------------------------------------------------------
// dK / dV: 32 keys per wave, the queries of all heads of the group streamed.
// fp32 above head dim 128 takes one launch for each (the registers hold the
// operands of both or the accumulators of both).
// ---------------------------------------------------------------------------
template <class E, int DP, bool DK, bool DV>
__global__ __launch_bounds__(64 * kPackedWaves) __attribute__((amdgpu_waves_per_eu(1, 1)))
void born_packed_dkdv_kernel(PackedArgs p) {
    using C = PackedCfg<E, DP>;
    using Tile = PackedTile<E, DP, C::BN>;
    constexpr int KS = Tile::KS, DB = Tile::DB, BN = C::BN, NST = C::NST, BM = kPackedRows, IT = kItem<E>;
    __shared__ __attribute__((aligned(1024))) uint8_t ring[NST * C::STAGE];
    __shared__ __attribute__((aligned(16))) float stats[NST][2][BN];  // -delta, zs

    const int hk = blockIdx.x % p.Hkv;
    const PackedSeq sq = packed_seq<true>(p, blockIdx.x / p.Hkv);
    const int k0 = sq.tile * BM;
    if (k0 >= sq.nk) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 31, g = lane >> 5;
    const int D = p.D, off = sq.nk - sq.nq;

    // Queries that see the block's keys, as tiles of BN, for each head.
    const int k1 = min(sq.nk, k0 + BM);
    const int ilo = max(0, k0 - off + p.lower), ihi = min(sq.nq - 1, k1 - 1 - off + p.upper - 1);
    const int t0 = ilo / BN, nt = ihi >= ilo ? ihi / BN - t0 + 1 : 0, n = nt * p.G;

    int qoff[Tile::LPW], doff[Tile::LPW];
    Tile::offsets(qoff, (int)p.q_st, D, wave, lane);
    Tile::offsets(doff, (int)p.do_st, D, wave, lane);
    auto qt = [&](int st) { return Tile{ring + st * C::STAGE}; };
    auto dt = [&](int st) { return Tile{ring + st * C::STAGE + Tile::BYTES}; };
    auto issue = [&](int h, int t, int st) __attribute__((always_inline)) {
        const int i0 = (t0 + t) * BN, left = sq.nq - i0;
        const int64_t r = sq.q0 + i0;
        qt(st).issue((const uint8_t*)p.q + r * p.q_st + (int64_t)h * p.q_sh, left, (int)p.q_st, D, qoff, wave);
        dt(st).issue((const uint8_t*)p.dout + r * p.do_st + (int64_t)h * p.do_sh, left, (int)p.do_st, D, doff, wave);
        if (wave < 2) {
            const float* v = (wave == 0 ? p.ndelta : p.zs) + (size_t)h * p.Nq + r;
            i32x4 rs = buffer_rsrc(v, (uint32_t)(4 * max(0, min(left, BN))));
#pragma unroll
            for (int i = 0; i < 4; ++i) rs[i] = __builtin_amdgcn_readfirstlane(rs[i]);
            if (lane < BN / 4) dma_load16(rs, lds_addr(stats[st][wave]), 16 * lane);
        }
    };

    const int kw = k0 + 32 * wave, key = kw + c;
    const bool ok = key < sq.nk;
    u32x4 kr[KS], vr[DK ? KS : 1];
    packed_load_row<E>(kr, (const uint8_t*)p.k + (int64_t)(sq.k0 + key) * p.k_st + (int64_t)hk * p.k_sh, ok, D, g);
    if constexpr (DK)
        packed_load_row<E>(vr, (const uint8_t*)p.v + (int64_t)(sq.k0 + key) * p.v_st + (int64_t)hk * p.v_sh, ok, D, g);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        asm volatile("" : "+v"(kr[ks]));
        if constexpr (DK) asm volatile("" : "+v"(vr[ks]));
    }
    f32x16 dk[DK ? DB : 1], dv[DV ? DB : 1];
#pragma unroll
    for (int db = 0; db < DB; ++db) {
        if constexpr (DK) dk[db] = zero16();
        if constexpr (DV) dv[db] = zero16();
    }
    const int span = p.upper - p.lower;

    int gi = 0, t = 0, ni = 0, nx = 0;  // this tile's and the next one's head of the group and tile
    if (n > 0) issue(hk * p.G, 0, 0);
    for (int u = 0; u < n; ++u) {
        const int st = u % NST, i0 = (t0 + t) * BN;
        const float sc = arg_scale(p, hk * p.G + gi);
        nx = t + 1, ni = gi;
        if (nx == nt) nx = 0, ++ni;
        wait_vmcnt<0>();
        __syncthreads();
        if (u + 1 < n) issue(hk * p.G + ni, nx, (u + 1) % NST);
        t = nx, gi = ni;
        const bool none = i0 + BN - 1 + off - kw < p.lower || i0 + off - (kw + 31) >= p.upper;
        if (none) continue;
        const bool cut = i0 + off - (kw + 31) < p.lower || i0 + BN - 1 + off - kw >= p.upper;
        const float sign = sc < 0.f ? -1.f : 1.f;
#pragma unroll
        for (int nb = 0; nb < BN / 32; ++nb) {
            f32x16 s = zero16(), dp, zi;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const f32x4 a = *reinterpret_cast<const f32x4*>(&stats[st][0][32 * nb + 8 * j + 4 * g]);
                const f32x4 b = *reinterpret_cast<const f32x4*>(&stats[st][1][32 * nb + 8 * j + 4 * g]);
#pragma unroll
                for (int e = 0; e < 4; ++e) dp[4 * j + e] = a[e], zi[4 * j + e] = b[e];
            }
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                s = packed_step<E>(qt(st).row(32 * nb + c, ks, g), kr[ks], s);
                if constexpr (DK) dp = packed_step<E>(dt(st).row(32 * nb + c, ks, g), vr[ks], dp);
            }
            if (cut) {
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if ((uint32_t)(i0 + 32 * nb + acc_row(r, g) + off - key - p.lower) >= (uint32_t)span) s[r] = 0.f;
            }
            PackedWeights<E> w, x;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float ww[2], uu[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int r = 2 * j + e;
                    const float a = relu_f32(s[r] * sign), tz = a * zi[r];
                    ww[e] = kUpW<E> * tz * a;
                    uu[e] = kUpU<E> * sign * tz * dp[r];
                }
                w.set(j, ww[0], ww[1]);
                x.set(j, uu[0], uu[1]);
            }
            if constexpr (DV) packed_columns<E>(dt(st), 32 * nb, w, dv, lane);
            if constexpr (DK) packed_columns<E>(qt(st), 32 * nb, x, dk, lane);
        }
    }
    if (!ok) return;
    const size_t at = ((size_t)(sq.k0 + key) * p.Hkv + hk) * D * IT;  // contiguous (Nk, Hkv, D)
    if constexpr (DK) packed_store_row<E>((uint8_t*)p.dk + at, dk, 2.f / kUpU<E>, D, g);
    if constexpr (DV) packed_store_row<E>((uint8_t*)p.dv + at, dv, 1.f / kUpW<E>, D, g);
}

// ---------------------------------------------------------------------------
// dscale_h = (2 / s) sum_i delta_i eps / Z_i = (2 eps / s^3) sum_i delta_i zs_i:
// 32 partial sums per head in 64 bits, then their sums in order.
// ---------------------------------------------------------------------------
constexpr int kPackedParts = 32;

template <int>
__global__ __launch_bounds__(256) void born_packed_dscale_part_kernel(PackedArgs p, double* part) {
    __shared__ double red[4];
    const int h = blockIdx.x;
    double x = 0.0;
    for (int64_t i = blockIdx.y * 256 + threadIdx.x; i < p.Nq; i += kPackedParts * 256) {
        const size_t at = (size_t)h * p.Nq + i;
        x -= (double)p.ndelta[at] * (double)p.zs[at];
    }
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
    __syncthreads();
    if (threadIdx.x == 0) part[(size_t)h * kPackedParts + blockIdx.y] = ((red[0] + red[1]) + red[2]) + red[3];
}

template <int>
__global__ __launch_bounds__(64) void born_packed_dscale_kernel(PackedArgs p, const double* part, float* dscale, int n_scale) {
    double total = 0.0;
    for (int h = threadIdx.x; h < p.H; h += 64) {
        double x = 0.0;
        for (int i = 0; i < kPackedParts; ++i) x += part[(size_t)h * kPackedParts + i];
        const double s = (double)arg_scale(p, h);
        x = s != 0.0 ? 2.0 * (double)p.eps / (s * s * s) * x : 0.0;
        if (n_scale > 1) dscale[h] = (float)x;
        total += x;
    }
    if (n_scale > 1) return;
    for (int o = 32; o > 0; o >>= 1) total += __shfl_xor(total, o);
    if (threadIdx.x == 0) dscale[0] = (float)total;
}

// ---------------------------------------------------------------------------
// Launches.
// ---------------------------------------------------------------------------
inline unsigned packed_blocks(int N, int S) { return (unsigned)(N / kPackedRows + S + 1); }

#define QDL_PACKED_DP(D, BODY)                            \
    if ((D) <= 64) {                                      \
        constexpr int DPV = 64;                           \
        BODY                                              \
    } else if ((D) <= 96) {                               \
        constexpr int DPV = 96;                           \
        BODY                                              \
    } else if ((D) <= 128) {                              \
        constexpr int DPV = 128;                          \
        BODY                                              \
    } else {                                              \
        constexpr int DPV = 256;                          \
        BODY                                              \
    }

template <class E>
hipError_t launch_packed_fwd(const PackedArgs& a, hipStream_t st) {
    const dim3 grid(packed_blocks(a.Nq, a.S) * (unsigned)a.H), block(64 * kPackedWaves);
    QDL_PACKED_DP(a.D, { hipLaunchKernelGGL((born_packed_fwd_kernel<E, DPV>), grid, block, 0, st, a); })
    return hipGetLastError();
}

// dQ first: it forms the rows' -delta and s^2 / Z.
template <class E>
hipError_t launch_packed_bwd(const PackedArgs& a, hipStream_t st) {
    const dim3 grid(packed_blocks(a.Nq, a.S) * (unsigned)a.H), block(64 * kPackedWaves);
    const dim3 kgrid(packed_blocks(a.Nk, a.S) * (unsigned)a.Hkv);
    QDL_PACKED_DP(a.D, {
        if (a.Nq > 0) {
            hipLaunchKernelGGL((born_packed_dq_kernel<E, DPV>), grid, block, 0, st, a);
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
        }
        if (a.Nk > 0) {
            if constexpr (kItem<E> * DPV > 512) {
                hipLaunchKernelGGL((born_packed_dkdv_kernel<E, DPV, true, false>), kgrid, block, 0, st, a);
                const hipError_t e = hipGetLastError();
                if (e != hipSuccess) return e;
                hipLaunchKernelGGL((born_packed_dkdv_kernel<E, DPV, false, true>), kgrid, block, 0, st, a);
            } else {
                hipLaunchKernelGGL((born_packed_dkdv_kernel<E, DPV, true, true>), kgrid, block, 0, st, a);
            }
        }
    })
    return hipGetLastError();
}

// Entry points of the per-dtype translation units.
template <class E>
hipError_t packed_fwd(const PackedArgs& a, hipStream_t st);
template <class E>
hipError_t packed_bwd(const PackedArgs& a, hipStream_t st);

}  // namespace qdl
