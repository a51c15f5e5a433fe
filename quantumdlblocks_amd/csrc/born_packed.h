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
// Roundings.  Scores, sums, statistics and accumulators are fp32.  The 16-bit
// matrix instructions take 16-bit operands, so the factor that a kernel forms
// itself is rounded once before each second product: p (forward), p / Z (dV)
// and u (dQ, dK), half a step each.  Z adds the rounded p, so numerator and
// denominator carry the same error: a row that one key takes whole is that key's
// v, and its delta that key's dP.  (With fp16's p added unrounded such rows'
// gradients were off by p's rounding over a small a: dQ of a batch of 6, 20 and 7
// tokens 14 times as far off as its output's rounding, now 5.)  delta comes from
// the output as it was rounded: an unrounded O would cost 2 N H D bytes more to
// write and to read.  Against 64 bits the 16-bit dQ and dK are 1.9 and 1.5 times
// as far off as gradients whose only rounding is the output's (in norm, medians
// of 1228 drawn batches; bf16 3.2e-3 and 2.5e-3 for 1.7e-3), 2.1 and 1.8 times in
// one of twenty, 5.8 and 4.4 times in the worst: short sequences, where a row
// that one key takes nearly whole has dO . v - delta next to nothing there, and
// delta's rounding is divided by a.  A simulation in 64 bits, bf16, with
// everything, with delta from an unrounded O, with u in two parts, with both:
// dQ of 1500 tokens D128 1.9, 1.7, 1.5, 1.2 times, of a batch of 33, 26, 8, 2 and
// 4 tokens D32 2.3, 1.8, 2.0, 1.4; u in two parts would take a second product in
// kernels that the matrix pipe bounds.
// fp32 rounds nothing on the way (3.3e-7, plain fp32 4.8e-7).
//
// What bounds them: the matrix pipe.  A workgroup's four waves share the tiles
// of the streamed operands, which LDS-DMA loads bring into a ring of two stages,
// one barrier per tile.  Each wave owns 32 stationary rows (queries in the
// forward and dQ, keys in dK/dV); the weights of a row have no running maximum,
// so waves may also share stationary rows and take different rows of each tile
// (SPLIT of them), their sums meeting in LDS once, at the end: fewer rows per
// block, so more and shorter blocks.
//
// Blocks of BM rows: sequence s takes the block slots from cu[s] / BM + s on.  Since
// ceil(len / BM) <= cu[s+1] / BM - cu[s] / BM + 1 they never overlap, so the
// grid follows from N and S alone (no copy of the lengths to the host, no list
// made by another launch), and a block finds its sequence by a 64-way search.
// Slots without rows end at once.  The rows behind the last sequence belong to
// a sequence of their own without keys: zero outputs and gradients.
#pragma once

#include <type_traits>

#include "born_common.h"
#include "born_fwd_fast.h"
#include "packed_mask.h"

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
    float* zs;      // (H, Nq) workspace: sign(s) s^2 / Z (fp16: times kUp)
    const float* scale;  // 1 or H values, or nullptr: scale_value
    float scale_value;
    int per_head_scale;
    const int32_t *cu_q, *cu_k;  // S + 1 starts
    int S, Nq, Nk, H, Hkv, G, D;
    int lower, upper;  // visible: lower <= query position - key < upper
    int head_splits;   // dK/dV: workgroups that share a group's heads
    float* part;       // their fp32 sums, (2, head_splits, Nk, Hkv, D), where there are several
    float eps;
    int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh, do_st, do_sh;
};

constexpr int kPackedWaves = 4;
constexpr int packed_rows(int split) { return 32 * kPackedWaves / split; }  // stationary rows per workgroup

// A sequence's rows: queries q0 .. q0 + nq - 1, keys k0 .. k0 + nk - 1.
struct PackedSeq {
    int q0, nq, k0, nk;
    int tile;  // this block's tile within it
};

__device__ __forceinline__ int packed_start(const int32_t* cu, int s, int N) {
    return s == 0 ? 0 : min(max(cu[s], 0), N);
}

// Block x of the launch: a tile of BM query rows or (KEYS) key rows.  Slots are
// counted along `cu`; the sequence is found by a 64-way search.  Under plain
// causality, with few enough sequences for a lane each, the blocks go in the
// order of their work instead, over all sequences (a block's tiles are those
// before its queries or behind its keys): a launch ends with short blocks
// (8 ragged sequences, 16384 tokens, D128: dK/dV 541 us, in the slots' order
// 554 to 571).
template <bool KEYS, int BM>
__device__ __forceinline__ PackedSeq packed_seq(const PackedArgs& p, int x) {
    const int32_t* cu = KEYS ? p.cu_k : p.cu_q;
    const int N = KEYS ? p.Nk : p.Nq, lane = threadIdx.x & 63;
    PackedSeq r;
    int s;
    if (p.S < 64 && p.lower == 0 && p.upper == kPackedFar) {
        const int a = lane <= p.S ? packed_start(cu, lane, N) : 0;
        const int e = lane < p.S ? max(packed_start(cu, lane + 1, N), a) : lane == p.S ? N : 0;
        const int tiles = (e - a + BM - 1) / BM;
        int left = tiles;  // the most work of any block, then one less
        for (int o = 1; o < 64; o <<= 1) left = max(left, __shfl_xor(left, o));
        left = __builtin_amdgcn_readfirstlane(left);
        uint64_t have = 0;
        for (; left > 0; --left) {
            have = __ballot(tiles >= left);
            const int n = (int)__popcll(have);
            if (x < n) break;
            x -= n;
        }
        // The x-th of them.
        const bool mine = ((have >> lane) & 1) != 0 && (int)__popcll(have & ((1ull << lane) - 1)) == x;
        const uint64_t at = __ballot(left > 0 && mine);
        s = at != 0 ? __ffsll((long long)at) - 1 : p.S;
        r.tile = at != 0 ? (KEYS ? __builtin_amdgcn_readlane(tiles, s) - left : left - 1) : (1 << 22);
    } else {
        if (!KEYS) x = N / BM + p.S - x;  // a sequence's last queries first
        int lo = 0, hi = p.S + 1;
        while (hi - lo > 1) {
            const int step = (hi - lo + 63) / 64;
            const int i = lo + (lane + 1) * step;
            const bool below = i < hi && packed_start(cu, i, N) / BM + i <= x;
            lo += (int)__popcll(__ballot(below)) * step;
            hi = min(hi, lo + step);
        }
        s = __builtin_amdgcn_readfirstlane(lo);
        r.tile = x - (packed_start(cu, s, N) / BM + s);
    }
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
    return r;
}

// ROWS rows of one streamed operand in LDS: 16-byte chunks XOR-swizzled per
// row so that neither a row read (16 rows, one chunk) nor a transposed read (4
// consecutive rows, 64 bytes each) meets a bank twice: rows that all start on
// bank 0 by all four bits of the row, rows of alternating halves by lds_swz,
// rows on four starts by the row's upper bits.
template <class E, int DP, int ROWS, int NW = kPackedWaves>
struct PackedTile {
    static constexpr int IT = kItem<E>, RB = IT * DP, CPR = RB / 16, BYTES = ROWS * RB;
    static constexpr int LOADS = BYTES / 1024, LPW = (LOADS + NW - 1) / NW;  // 1-KiB loads, dealt to the waves
    static constexpr int KS = RB / 32, DB = DP / 32;
    static_assert(BYTES % 1024 == 0, "whole loads");
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
            const int slot = (i * NW + wave) * 64 + lane, row = slot / CPR, chunk = (slot % CPR) ^ swz(row);
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
        for (int i = 0; i < LPW; ++i)
            if (LOADS % NW == 0 || i * NW + wave < LOADS) dma_load16(rs, lds_addr(lds + (i * NW + wave) * 1024), off[i]);
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

// 1 / den; 0 for rows without weight, and for sums below fp32's normal range,
// whose reciprocals may be infinite: a row of zeros times that is not a number.
// The backward's zs = 1 / den is cut at the same sum, its bound divided by the
// factor that it is stored with.
__device__ __forceinline__ float packed_inverse(float den) { return den >= 0x1p-126f ? 1.0f / den : 0.f; }

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
    return __uint_as_float((uint32_t)(min(max(6 - e, -126), 60) + 127) << 23);
}

// fp16 gradients' operands.  p / Z is at most 1: times 16, what rounding takes
// from a small one lies below the step of a small fp16 output.  The factor u of
// dS has no bound (a row whose overlaps are all small divides by their sum), so
// it is kept in fp16's range like the weights: by a power of two per column of
// its product, which drops where a part would pass the bound, with what that
// column has summed.
template <class E>
constexpr float kUp = std::is_same<E, F16>::value ? 16.f : 1.f;
template <class E, int DB>
__device__ __forceinline__ void packed_fit(float (&u)[16], float& f, f32x16 (&acc)[DB]) {
    if constexpr (std::is_same<E, F16>::value) {
        float m = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) m = fmaxf(m, fabsf(u[r]));
        m = fmaxf(m, __shfl_xor(m, 32));
        if (__ballot(m * f > 61440.f) != 0) {
            const float to = m * f > 61440.f ? f16_factor(m) * 256.f : f, by = to / f;  // to [2^14, 2^15)
            f = to;
#pragma unroll
            for (int db = 0; db < DB; ++db) acc[db] *= by;
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) u[r] *= f;
    }
}
template <class E, int DB>
__device__ __forceinline__ void packed_unfit(float& f, f32x16 (&acc)[DB]) {
    if constexpr (std::is_same<E, F16>::value) {
        const float by = 1.f / f;
        f = 1.f;
#pragma unroll
        for (int db = 0; db < DB; ++db) acc[db] *= by;
    }
}

// 32 rows of a wave's accumulators to its share of the reduction buffer, rows of
// DP + 4 floats, and another wave's share added to a wave's own.
template <int DB>
__device__ __forceinline__ void packed_put(float* red, const f32x16 (&acc)[DB], int c, int g) {
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const f32x4 w = {acc[db][4 * j], acc[db][4 * j + 1], acc[db][4 * j + 2], acc[db][4 * j + 3]};
            *reinterpret_cast<f32x4*>(red + c * (32 * DB + 4) + 32 * db + 8 * j + 4 * g) = w;
        }
}
template <int DB>
__device__ __forceinline__ void packed_add(f32x16 (&acc)[DB], const float* red, int c, int g) {
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const f32x4 w = *reinterpret_cast<const f32x4*>(red + c * (32 * DB + 4) + 32 * db + 8 * j + 4 * g);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[db][4 * j + e] += w[e];
        }
}

// A wave's tiles 0 .. n - 1, whose rows start at first + u step and number w,
// against the positions that it sees: those from a0 to a1 by some of its rows,
// from b0 to b1 by all.  [0, ta): none visible; [ta, tf) and [tg, tv): some
// pairs masked; [tf, tg): none masked; [tv, n): none visible.  Each run has a
// loop of its own: a masked and an unmasked body behind one branch would move
// the accumulators on every tile, or spill.
struct PackedRuns {
    int ta, tf, tg, tv;
    __device__ __forceinline__ PackedRuns(int n, int first, int step, int w, int a0, int a1, int b0, int b1) {
        auto from = [&](int x) {  // the first tile that starts at x or behind
            const int d = x - first;
            return __builtin_amdgcn_readfirstlane(d <= 0 ? 0 : min((d + step - 1) / step, n));
        };
        ta = from(a0 - w + 1);
        tv = max(from(a1 + 1), ta);
        tf = min(max(from(b0), ta), tv);
        tg = min(max(from(b1 - w + 2), tf), tv);
    }
};
typedef std::integral_constant<int, 0> PackedIdle;
typedef std::integral_constant<int, 1> PackedFull;
typedef std::integral_constant<int, 2> PackedCut;

// A block's shape.  SPLIT waves share 32 stationary rows and take SUB 32-row
// parts of each tile in turn.
template <class E, int DP, int SPLIT>
struct PackedCfg {
    static constexpr int RB = kItem<E> * DP;
    static constexpr int SUB = SPLIT == 1 ? (kItem<E> == 2 && DP <= 128 ? 2 : 1) : SPLIT == 2 && RB <= 256 ? 2 : 1;
    static constexpr int BN = 32 * SUB * SPLIT;  // streamed rows per tile
    static constexpr int BM = packed_rows(SPLIT), GROUPS = kPackedWaves / SPLIT;
    static constexpr int STAGE = 2 * BN * RB, NST = 2;  // two operands
    static constexpr int RING = NST * STAGE, REDUCE = (SPLIT - 1) * GROUPS * 32 * (DP + 4) * 4;
    static constexpr int SMEM = RING > REDUCE ? RING : REDUCE;
    static_assert(SMEM <= 160 * 1024 - 4096, "LDS");
    // Forward and dQ: two workgroups per CU where the ring and the registers
    // let them; above, one.  The 16-bit forward up to head dim 64, whose
    // products are short beside its weights, has room for four (8 prompts of
    // 2048 tokens, 16 heads: 95 us with two, 88 with three, 86 with four).
    static constexpr int WPE = RB <= 256 && SMEM <= 78 * 1024 ? 2 : 1;
    static constexpr int FWD_WPE = RB == 128 && SPLIT == 1 ? 4 : WPE;
};

// A block of the forward or dQ: its rows, the keys that they see, their loads.
template <class E, int DP, int SPLIT>
struct PackedQueries {
    using C = PackedCfg<E, DP, SPLIT>;
    using Tile = PackedTile<E, DP, C::BN>;
    PackedSeq sq;
    int hk, h, m0, off, t0, n;
    int lane, wave, c, g, group, part;  // the wave's rows among the block's, its part of each tile
    int rw, row;                        // its first row, the lane's
    bool ok;
    const uint8_t *kb, *vb;
    int koff[Tile::LPW], voff[Tile::LPW];

    __device__ __forceinline__ bool init(const PackedArgs& p) {
        hk = blockIdx.x % p.Hkv;
        const int rest = blockIdx.x / p.Hkv;
        h = hk * p.G + rest % p.G;
        sq = packed_seq<false, C::BM>(p, rest / p.G);
        m0 = sq.tile * C::BM;
        if (m0 >= sq.nq) return false;
        lane = threadIdx.x & 63;
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        c = lane & 31;
        g = lane >> 5;
        group = wave % C::GROUPS;
        part = wave / C::GROUPS;
        off = sq.nk - sq.nq;
        const int m1 = min(sq.nq, m0 + C::BM);
        const int jlo = max(0, m0 + off - p.upper + 1), jhi = min(sq.nk - 1, m1 - 1 + off - p.lower);
        t0 = jlo / C::BN;
        n = jhi >= jlo ? jhi / C::BN - t0 + 1 : 0;
        kb = (const uint8_t*)p.k + (int64_t)sq.k0 * p.k_st + (int64_t)hk * p.k_sh;
        vb = (const uint8_t*)p.v + (int64_t)sq.k0 * p.v_st + (int64_t)hk * p.v_sh;
        Tile::offsets(koff, (int)p.k_st, p.D, wave, lane);
        Tile::offsets(voff, (int)p.v_st, p.D, wave, lane);
        rw = m0 + 32 * group;
        row = rw + c;
        ok = row < sq.nq;
        return true;
    }
    __device__ __forceinline__ static Tile kt(uint8_t* ring, int st) { return Tile{ring + st * C::STAGE}; }
    __device__ __forceinline__ static Tile vt(uint8_t* ring, int st) { return Tile{ring + st * C::STAGE + Tile::BYTES}; }
    __device__ __forceinline__ void issue(const PackedArgs& p, uint8_t* ring, int u, int st) const {
        const int key0 = (t0 + u) * C::BN;
        kt(ring, st).issue(kb + (int64_t)key0 * p.k_st, sq.nk - key0, (int)p.k_st, p.D, koff, wave);
        vt(ring, st).issue(vb + (int64_t)key0 * p.v_st, sq.nk - key0, (int)p.v_st, p.D, voff, wave);
    }
    // The wave's tiles: u's keys from key0(u) on.
    __device__ __forceinline__ int key0(int u) const { return (t0 + u) * C::BN + 32 * C::SUB * part; }
    __device__ __forceinline__ PackedRuns runs(const PackedArgs& p) const {
        return PackedRuns(n, key0(0), C::BN, 32 * C::SUB, rw + off - p.upper + 1, rw + 31 + off - p.lower,
                          rw + 31 + off - p.upper + 1, rw + off - p.lower);
    }
    // Every tile in turn: tile(u, stage, kind) where the wave sees any of it.
    template <class F>
    __device__ __forceinline__ void tiles(const PackedArgs& p, uint8_t* ring, F&& tile) const {
        const PackedRuns r = runs(p);
        if (n > 0) issue(p, ring, 0, 0);
        int u = 0;
        auto run = [&](int end, auto kind) __attribute__((always_inline)) {
            for (; u < end; ++u) {
                wait_vmcnt<0>();
                __syncthreads();
                if (u + 1 < n) issue(p, ring, u + 1, (u + 1) % C::NST);
                if constexpr (kind.value != 0) tile(u, u % C::NST, kind);
            }
        };
        run(r.ta, PackedIdle{});
        run(r.tf, PackedCut{});
        run(r.tg, PackedFull{});
        run(r.tv, PackedCut{});
        run(n, PackedIdle{});
    }
    // Zeroes a lane's overlaps with keys that its row does not see.
    __device__ __forceinline__ void mask(const PackedArgs& p, f32x16& s, int key0) const {
        const int d = row + off - key0 - p.lower;
        const uint32_t span = packed_span(p.lower, p.upper);
#pragma unroll
        for (int r = 0; r < 16; ++r)
            if ((uint32_t)(d - acc_row(r, g)) >= span) s[r] = 0.f;
    }
};

// ---------------------------------------------------------------------------
// Forward: S^T = K Q^T per 32 keys, the weights in place, O^T += V^T P^T.
// Bound by the matrix pipe at D128, by the weights' elementwise work beside it
// at D64.  Ragged bf16, 16 heads over 4: 16384 tokens D128 211 us (879 TFLOP/s),
// 8896 tokens D64 40 us (670); fp32, 1000 tokens, 8 heads D64: 18 us.
// ---------------------------------------------------------------------------
template <class E, int DP, int SPLIT>
__global__ __launch_bounds__(64 * kPackedWaves)
__attribute__((amdgpu_waves_per_eu(PackedCfg<E, DP, SPLIT>::FWD_WPE, PackedCfg<E, DP, SPLIT>::FWD_WPE)))
void born_packed_fwd_kernel(PackedArgs p) {
    using C = PackedCfg<E, DP, SPLIT>;
    using Q = PackedQueries<E, DP, SPLIT>;
    constexpr int KS = Q::Tile::KS, DB = Q::Tile::DB;
    __shared__ __attribute__((aligned(1024))) uint8_t ring[C::SMEM];
    __shared__ float zred[SPLIT][kPackedWaves / SPLIT][32];
    Q b;
    if (!b.init(p)) return;
    const int lane = b.lane, c = b.c, g = b.g, D = p.D;
    const float sc = arg_scale(p, b.h);

    u32x4 qr[KS];
    packed_load_row<E>(qr, (const uint8_t*)p.q + (int64_t)(b.sq.q0 + b.row) * p.q_st + (int64_t)b.h * p.q_sh, b.ok, D, g);
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

    const int r0 = 32 * C::SUB * b.part;  // this wave's part of every tile
    b.tiles(p, ring, [&](int u, int st, auto kind) __attribute__((always_inline)) {
        const int key0 = b.key0(u);
        const auto kt = Q::kt(ring, st), vt = Q::vt(ring, st);
#pragma unroll
        for (int nb = 0; nb < C::SUB; ++nb) {
            f32x16 s = zero16();
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) s = packed_step<E>(kt.row(r0 + 32 * nb + c, ks, g), qr[ks], s);
            if constexpr (kind.value == 2) b.mask(p, s, key0 + 32 * nb);
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
                for (int j = 0; j < 8; ++j) {
                    const float a0 = relu_f32(s[2 * j] * cf), a1 = relu_f32(s[2 * j + 1] * cf);
                    w.w[j] = F16::pack(a0 * a0, a1 * a1);
                    z = F16::sum2(w.w[j], z);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) w.w[j] = born_weight_pair<BF16>(s[2 * j], s[2 * j + 1], 1.f, z);
            }
            packed_columns<E>(vt, r0 + 32 * nb, w, acc, lane);
        }
    });

    z += __shfl_xor(z, 32);
    float s1 = std::is_same<E, F16>::value && SPLIT == 1 ? sc / cf : sc;
    if constexpr (SPLIT > 1) {
        if constexpr (std::is_same<E, F16>::value) {  // without the waves' own factors
            const float back = 1.f / (cf * cf);
            z *= back;
#pragma unroll
            for (int db = 0; db < DB; ++db) acc[db] *= back;
        }
        float* const red = reinterpret_cast<float*>(ring);
        auto share = [&](int part) { return red + ((part - 1) * C::GROUPS + b.group) * 32 * (DP + 4); };
        __syncthreads();
        if (g == 0) zred[b.part][b.group][c] = z;
        if (b.part > 0) packed_put(share(b.part), acc, c, g);
        __syncthreads();
        if (b.part > 0) return;
#pragma unroll
        for (int i = 1; i < SPLIT; ++i) {
            packed_add(acc, share(i), c, g);
            z += zred[i][b.group][c];
        }
    }
    if (!b.ok) return;
    const float s2 = s1 * s1;
    const float den = z + (p.eps == 0.f ? 0.f : p.eps / s2);
    const float inv = sc != 0.f ? packed_inverse(den) : 0.f;
    packed_store_row<E>((uint8_t*)p.out + ((size_t)(b.sq.q0 + b.row) * p.H + b.h) * D * kItem<E>, acc, inv, D, g);
    if (g == 0 && p.z != nullptr) p.z[(size_t)b.h * p.Nq + b.sq.q0 + b.row] = s2 * z + p.eps;
}

// ---------------------------------------------------------------------------
// dQ; also -delta and sign(s) s^2 / Z per row for the dK/dV kernel.  Three
// products a tile; bound by the matrix pipe: 300 us (928 TFLOP/s) for the 16384
// tokens of the forward's D128 figure.
// ---------------------------------------------------------------------------
template <class E, int DP, int SPLIT>
__global__ __launch_bounds__(64 * kPackedWaves)
__attribute__((amdgpu_waves_per_eu(PackedCfg<E, DP, SPLIT>::WPE, PackedCfg<E, DP, SPLIT>::WPE)))
void born_packed_dq_kernel(PackedArgs p) {
    using C = PackedCfg<E, DP, SPLIT>;
    using Q = PackedQueries<E, DP, SPLIT>;
    constexpr int KS = Q::Tile::KS, DB = Q::Tile::DB, IT = kItem<E>;
    __shared__ __attribute__((aligned(1024))) uint8_t ring[C::SMEM];
    Q b;
    if (!b.init(p)) return;
    const int lane = b.lane, c = b.c, g = b.g, D = p.D;
    const float sc = arg_scale(p, b.h);

    u32x4 qr[KS], dr[KS];
    packed_load_row<E>(qr, (const uint8_t*)p.q + (int64_t)(b.sq.q0 + b.row) * p.q_st + (int64_t)b.h * p.q_sh, b.ok, D, g);
    packed_load_row<E>(dr, (const uint8_t*)p.dout + (int64_t)(b.sq.q0 + b.row) * p.do_st + (int64_t)b.h * p.do_sh, b.ok, D, g);
    const size_t at = ((size_t)(b.sq.q0 + b.row) * p.H + b.h) * D * IT;  // contiguous (Nq, H, D)
    float delta = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        const int o = 32 * ks + 16 * g;
        if (!b.ok || o >= IT * D) continue;
        const u32x4 x = ldg16((const uint8_t*)p.o + at + o);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (std::is_same<E, F32>::value) delta = fmaf(__uint_as_float(x[j]), __uint_as_float(dr[ks][j]), delta);
            else delta += E::lo(x[j]) * E::lo(dr[ks][j]) + E::hi(x[j]) * E::hi(dr[ks][j]);
        }
    }
    delta += __shfl_xor(delta, 32);
    const size_t stat = (size_t)b.h * p.Nq + b.sq.q0 + b.row;
    const float zr = b.ok ? p.z[stat] : 1.f;
    float zs = zr > 0.f ? sc * fabsf(sc) / zr : 0.f;
    if (!(fabsf(zs) <= 0x1p126f / kUp<E>)) zs = 0.f;
    if (b.ok && g == 0 && b.part == 0) {
        p.ndelta[stat] = -delta;
        p.zs[stat] = kUp<E> * zs;
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
    float f = std::is_same<E, F16>::value ? kF16Start : 1.f;
    asm volatile("" : "+v"(delta));

    const int r0 = 32 * C::SUB * b.part;  // this wave's part of every tile
    b.tiles(p, ring, [&](int u, int st, auto kind) __attribute__((always_inline)) {
        const int key0 = b.key0(u);
        const auto kt = Q::kt(ring, st), vt = Q::vt(ring, st);
#pragma unroll
        for (int nb = 0; nb < C::SUB; ++nb) {
            f32x16 s = zero16(), t;
#pragma unroll
            for (int r = 0; r < 16; ++r) t[r] = -delta;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                s = packed_step<E>(kt.row(r0 + 32 * nb + c, ks, g), qr[ks], s);
                t = packed_step<E>(vt.row(r0 + 32 * nb + c, ks, g), dr[ks], t);
            }
            if constexpr (kind.value == 2) b.mask(p, s, key0 + 32 * nb);
            // Without zs, the row's factor.
            PackedWeights<E> w;
            float x[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] = relu_f32(s[r]) * t[r];
            packed_fit<E>(x, f, acc);
#pragma unroll
            for (int j = 0; j < 8; ++j) w.set(j, x[2 * j], x[2 * j + 1]);
            packed_columns<E>(kt, r0 + 32 * nb, w, acc, lane);
        }
    });
    if constexpr (SPLIT > 1) {
        packed_unfit<E>(f, acc);
        float* const red = reinterpret_cast<float*>(ring);
        auto share = [&](int part) { return red + ((part - 1) * C::GROUPS + b.group) * 32 * (DP + 4); };
        __syncthreads();
        if (b.part > 0) packed_put(share(b.part), acc, c, g);
        __syncthreads();
        if (b.part > 0) return;
#pragma unroll
        for (int i = 1; i < SPLIT; ++i) packed_add(acc, share(i), c, g);
    }
    if (!b.ok) return;
    packed_store_row<E>((uint8_t*)p.dq + at, acc, std::is_same<E, F16>::value ? 2.f * zs * (1.f / f) : 2.f * zs, D, g);
}

// A dK/dV workgroup's key head, block and heads g0 .. g1 - 1 of the group.
struct PackedHeads {
    int hk, block, split, g0, g1;
    __device__ __forceinline__ PackedHeads(const PackedArgs& p) {
        hk = blockIdx.x % p.Hkv;
        const int rest = blockIdx.x / p.Hkv;
        split = rest % p.head_splits;
        block = rest / p.head_splits;
        g0 = p.G * split / p.head_splits;
        g1 = p.G * (split + 1) / p.head_splits;
    }
};

// A key's row of dK (which = 0) or dV (1): the output, or this workgroup's part.
template <class E, int DB>
__device__ __forceinline__ void packed_store_keys(const PackedArgs& p, void* out, int which, int split, size_t at,
                                                  const f32x16 (&acc)[DB], float f, int g) {
    if (p.head_splits > 1) {
        const size_t whole = (size_t)p.Nk * p.Hkv * p.D;
        packed_store_row<F32>((uint8_t*)(p.part + (which * p.head_splits + split) * whole + at), acc, f, p.D, g);
    } else {
        packed_store_row<E>((uint8_t*)out + at * kItem<E>, acc, f, p.D, g);
    }
}

// The parts' sums, in order: 8 values a thread, dK and then dV.
template <class E>
__global__ __launch_bounds__(256) void born_packed_dkdv_join_kernel(PackedArgs p) {
    const size_t whole = (size_t)p.Nk * p.Hkv * p.D, i = ((size_t)blockIdx.x * 256 + threadIdx.x) * 8;
    if (i >= 2 * whole) return;
    const int which = i >= whole;
    const size_t at = i - which * whole;
    const float* src = p.part + which * p.head_splits * whole + at;
    f32x4 x = *reinterpret_cast<const f32x4*>(src), y = *reinterpret_cast<const f32x4*>(src + 4);
    for (int k = 1; k < p.head_splits; ++k) {
        x += *reinterpret_cast<const f32x4*>(src + k * whole);
        y += *reinterpret_cast<const f32x4*>(src + k * whole + 4);
    }
    uint8_t* out = (uint8_t*)(which ? p.dv : p.dk) + at * kItem<E>;
    if constexpr (std::is_same<E, F32>::value) {
        *reinterpret_cast<f32x4*>(out) = x;
        *reinterpret_cast<f32x4*>(out + 16) = y;
    } else {
        const u32x4 w = {E::pack(x[0], x[1]), E::pack(x[2], x[3]), E::pack(y[0], y[1]), E::pack(y[2], y[3])};
        *reinterpret_cast<u32x4*>(out) = w;
    }
}

// ---------------------------------------------------------------------------
// dK / dV of fp32, and of 16 bits above head dim 128: 32 keys per wave, whose
// rows stay in registers, one wave per SIMD; the queries of all heads of the
// group streamed.  fp32 above head dim 128 takes one launch for each (the
// registers hold the operands of both or the accumulators of both).
// ---------------------------------------------------------------------------
template <class E, int DP, int SPLIT, bool DK, bool DV>
__global__ __launch_bounds__(64 * kPackedWaves) __attribute__((amdgpu_waves_per_eu(1, 1)))
void born_packed_dkdv_kernel(PackedArgs p) {
    using C = PackedCfg<E, DP, SPLIT>;
    using Tile = PackedTile<E, DP, C::BN>;
    constexpr int KS = Tile::KS, DB = Tile::DB, BN = C::BN, NST = C::NST, SUB = C::SUB;
    __shared__ __attribute__((aligned(1024))) uint8_t ring[C::SMEM];
    __shared__ __attribute__((aligned(16))) float stats[NST][2][BN];  // -delta, zs

    const PackedHeads hd(p);
    const int hk = hd.hk;
    const PackedSeq sq = packed_seq<true, C::BM>(p, hd.block);
    const int k0 = sq.tile * C::BM;
    if (k0 >= sq.nk) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 31, g = lane >> 5;
    const int group = wave % C::GROUPS, part = wave / C::GROUPS;
    const int D = p.D, off = sq.nk - sq.nq;

    // Queries that see the block's keys, as tiles of BN, for each head.
    const int k1 = min(sq.nk, k0 + C::BM);
    const int ilo = max(0, k0 - off + p.lower), ihi = min(sq.nq - 1, k1 - 1 - off + p.upper - 1);
    const int t0 = ilo / BN, nt = ihi >= ilo ? ihi / BN - t0 + 1 : 0, n = nt * (hd.g1 - hd.g0);

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

    const int kw = k0 + 32 * group, key = kw + c;
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
    float f = std::is_same<E, F16>::value ? kF16Start : 1.f;
    const uint32_t span = packed_span(p.lower, p.upper);

    // Row values r0 + 8 j + 4 g + e.
    auto values = [&](const float* x, int r0) __attribute__((always_inline)) {
        f32x16 y;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const f32x4 a = *reinterpret_cast<const f32x4*>(x + r0 + 8 * j + 4 * g);
#pragma unroll
            for (int e = 0; e < 4; ++e) y[4 * j + e] = a[e];
        }
        return y;
    };
    // p / Z and the factor of dS of 32 queries from i0 + r0, from S and dP.
    auto elementwise = [&](int st, int i0, int r0, f32x16& s, const f32x16& dp, PackedWeights<E>& w, PackedWeights<E>& x,
                           auto kind) __attribute__((always_inline)) {
        if constexpr (kind.value == 2) {
            const int d = i0 + r0 + off - key - p.lower;
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if ((uint32_t)(d + acc_row(r, g)) >= span) s[r] = 0.f;
        }
        const f32x16 zi = values(stats[st][1], r0);
        float u[16];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float ww[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = 2 * j + e;
                const float a = relu_f32(s[r]), t = a * zi[r];
                ww[e] = fabsf(t) * a;  // zs carries the sign of s
                u[r] = t * dp[r];
            }
            if constexpr (DV) w.set(j, ww[0], ww[1]);
        }
        if constexpr (DK) {
            packed_fit<E>(u, f, dk);
#pragma unroll
            for (int j = 0; j < 8; ++j) x.set(j, u[2 * j], u[2 * j + 1]);
        }
    };

    const int r0 = 32 * SUB * part;  // this wave's part of every tile
    auto tile = [&](int t, int st, auto kind) __attribute__((always_inline)) {
        const int i0 = (t0 + t) * BN;
        const Tile q = qt(st), d = dt(st);
#pragma unroll
        for (int nb = 0; nb < SUB; ++nb) {
            const int rr = r0 + 32 * nb;
            f32x16 s = zero16(), dp = values(stats[st][0], rr);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                s = packed_step<E>(q.row(rr + c, ks, g), kr[ks], s);
                if constexpr (DK) dp = packed_step<E>(d.row(rr + c, ks, g), vr[ks], dp);
            }
            PackedWeights<E> w, x;
            elementwise(st, i0, rr, s, dp, w, x, kind);
            if constexpr (DV) packed_columns<E>(d, rr, w, dv, lane);
            if constexpr (DK) packed_columns<E>(q, rr, x, dk, lane);
        }
    };

    // Positions of the queries from the wave's first key on.
    const PackedRuns runs(nt, t0 * BN + r0 + off - kw, BN, 32 * SUB, p.lower, p.upper + 30, p.lower + 31, p.upper - 1);
    uint32_t flip = 0;  // the scale's sign, folded into K
    int u = 0;          // tiles so far
    if (n > 0) issue(hk * p.G + hd.g0, 0, 0);
    for (int gi = hd.g0; gi < hd.g1; ++gi) {
        const uint32_t fl = packed_flip<E>(arg_scale(p, hk * p.G + gi));
        if (fl != flip) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) kr[ks] ^= fl ^ flip;
            flip = fl;
        }
        int t = 0;
        auto run = [&](int end, auto kind) __attribute__((always_inline)) {
            for (; t < end; ++t, ++u) {
                wait_vmcnt<0>();
                __syncthreads();
                if (u + 1 < n) {
                    const bool last = t + 1 == nt;
                    issue(hk * p.G + gi + (last ? 1 : 0), last ? 0 : t + 1, (u + 1) % NST);
                }
                if constexpr (kind.value != 0) tile(t, u % NST, kind);
            }
        };
        run(runs.ta, PackedIdle{});
        run(runs.tf, PackedCut{});
        run(runs.tg, PackedFull{});
        run(runs.tv, PackedCut{});
        run(nt, PackedIdle{});
    }
    if constexpr (SPLIT > 1) {
        float* const red = reinterpret_cast<float*>(ring);
        auto share = [&](int i) { return red + ((i - 1) * C::GROUPS + group) * 32 * (DP + 4); };
        auto join = [&](f32x16 (&acc)[DB]) __attribute__((always_inline)) {
            __syncthreads();
            if (part > 0) packed_put(share(part), acc, c, g);
            __syncthreads();
            if (part == 0) {
#pragma unroll
                for (int i = 1; i < SPLIT; ++i) packed_add(acc, share(i), c, g);
            }
        };
        if constexpr (DK) {
            packed_unfit<E>(f, dk);
            join(dk);
        }
        if constexpr (DV) join(dv);
        if (part > 0) return;
    }
    if (!ok) return;
    const size_t at = ((size_t)(sq.k0 + key) * p.Hkv + hk) * D;  // contiguous (Nk, Hkv, D)
    if constexpr (DK) packed_store_keys<E>(p, p.dk, 0, hd.split, at, dk, std::is_same<E, F16>::value ? 2.f / kUp<E> * (1.f / f) : 2.f, g);
    if constexpr (DV) packed_store_keys<E>(p, p.dv, 1, hd.split, at, dv, 1.f / kUp<E>, g);
}

// ---------------------------------------------------------------------------
// dK / dV of 16 bits up to head dim 128: eight waves, two on each SIMD, over 128
// keys.  The stationary rows stay in LDS beside the ring, which leaves a wave
// the registers of its accumulators; four waves take 32 keys each of a tile's
// first half, four of its second.  Every tile feeds 128 keys: with 64, the
// tiles' way from L2 bounds the launch.  8 ragged sequences, 16384 tokens, 16
// heads over 4, D128, on one machine: 541 us, one wave on a SIMD over 64 or 128
// keys in registers 613 and 620.  Machines differ: 486 us (763 TFLOP/s) on
// another.  Four products a tile and the longest sequence's blocks bound it.
// ---------------------------------------------------------------------------
template <class E, int DP>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2)))
void born_packed_dkdv8_kernel(PackedArgs p) {
    constexpr int NW = 8, BM = 128, BN = 64, NST = 2;
    using Tile = PackedTile<E, DP, BN, NW>;
    using Keys = PackedTile<E, DP, BM, NW>;
    constexpr int KS = Tile::KS, DB = Tile::DB, STAGE = 2 * Tile::BYTES;
    __shared__ __attribute__((aligned(1024))) uint8_t ring[NST * STAGE + 2 * Keys::BYTES];  // and K, V
    uint8_t* const keys = ring + NST * STAGE;
    __shared__ __attribute__((aligned(16))) float stats[NST][2][BN];  // -delta, zs

    const PackedHeads hd(p);
    const int hk = hd.hk;
    const PackedSeq sq = packed_seq<true, BM>(p, hd.block);
    const int k0 = sq.tile * BM;
    if (k0 >= sq.nk) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 31, g = lane >> 5, group = wave & 3, part = wave >> 2;
    const int D = p.D, off = sq.nk - sq.nq;

    const int k1 = min(sq.nk, k0 + BM);
    const int ilo = max(0, k0 - off + p.lower), ihi = min(sq.nq - 1, k1 - 1 - off + p.upper - 1);
    const int t0 = ilo / BN, nt = ihi >= ilo ? ihi / BN - t0 + 1 : 0, n = nt * (hd.g1 - hd.g0);

    int qoff[Tile::LPW], doff[Tile::LPW];
    Tile::offsets(qoff, (int)p.q_st, D, wave, lane);
    Tile::offsets(doff, (int)p.do_st, D, wave, lane);
    auto issue = [&](int h, int t, int st) __attribute__((always_inline)) {
        const int i0 = (t0 + t) * BN, left = sq.nq - i0;
        const int64_t r = sq.q0 + i0;
        const Tile q{ring + st * STAGE}, d{ring + st * STAGE + Tile::BYTES};
        q.issue((const uint8_t*)p.q + r * p.q_st + (int64_t)h * p.q_sh, left, (int)p.q_st, D, qoff, wave);
        d.issue((const uint8_t*)p.dout + r * p.do_st + (int64_t)h * p.do_sh, left, (int)p.do_st, D, doff, wave);
        if (wave < 2) {
            const float* v = (wave == 0 ? p.ndelta : p.zs) + (size_t)h * p.Nq + r;
            i32x4 rs = buffer_rsrc(v, (uint32_t)(4 * max(0, min(left, BN))));
#pragma unroll
            for (int i = 0; i < 4; ++i) rs[i] = __builtin_amdgcn_readfirstlane(rs[i]);
            if (lane < BN / 4) dma_load16(rs, lds_addr(stats[st][wave]), 16 * lane);
        }
    };
    const Keys kt{keys}, vt{keys + Keys::BYTES};
    {
        int koff[Keys::LPW];
        const int64_t r = sq.k0 + k0;
        Keys::offsets(koff, (int)p.k_st, D, wave, lane);
        kt.issue((const uint8_t*)p.k + r * p.k_st + (int64_t)hk * p.k_sh, sq.nk - k0, (int)p.k_st, D, koff, wave);
        Keys::offsets(koff, (int)p.v_st, D, wave, lane);
        vt.issue((const uint8_t*)p.v + r * p.v_st + (int64_t)hk * p.v_sh, sq.nk - k0, (int)p.v_st, D, koff, wave);
    }
    const int kw = k0 + 32 * group, key = kw + c, r0 = 32 * part;
    f32x16 dk[DB], dv[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db) dk[db] = zero16(), dv[db] = zero16();
    float f = std::is_same<E, F16>::value ? kF16Start : 1.f;
    const uint32_t span = packed_span(p.lower, p.upper);

    auto tile = [&](int t, int st, auto kind) __attribute__((always_inline)) {
        const Tile q{ring + st * STAGE}, d{ring + st * STAGE + Tile::BYTES};
        f32x16 s = zero16(), dp;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const f32x4 a = *reinterpret_cast<const f32x4*>(&stats[st][0][r0 + 8 * j + 4 * g]);
#pragma unroll
            for (int e = 0; e < 4; ++e) dp[4 * j + e] = a[e];
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            s = E::mfma(q.row(r0 + c, ks, g), kt.row(32 * group + c, ks, g), s);
            dp = E::mfma(d.row(r0 + c, ks, g), vt.row(32 * group + c, ks, g), dp);
        }
        if constexpr (kind.value == 2) {
            const int x = (t0 + t) * BN + r0 + off - key - p.lower;
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if ((uint32_t)(x + acc_row(r, g)) >= span) s[r] = 0.f;
        }
        PackedWeights<E> w, x;
        float uu[16];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const f32x4 zi = *reinterpret_cast<const f32x4*>(&stats[st][1][r0 + 8 * j + 4 * g]);
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                float ww[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int r = 4 * j + e + i;
                    const float a = relu_f32(s[r]), y = a * zi[e + i];
                    ww[i] = fabsf(y) * a;  // zs carries the sign of s
                    uu[r] = y * dp[r];
                }
                w.set(2 * j + e / 2, ww[0], ww[1]);
            }
        }
        packed_fit<E>(uu, f, dk);
#pragma unroll
        for (int j = 0; j < 8; ++j) x.set(j, uu[2 * j], uu[2 * j + 1]);
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
            const u32x4 bw = {w.w[4 * hh], w.w[4 * hh + 1], w.w[4 * hh + 2], w.w[4 * hh + 3]};
            const u32x4 bx = {x.w[4 * hh], x.w[4 * hh + 1], x.w[4 * hh + 2], x.w[4 * hh + 3]};
#pragma unroll
            for (int db = 0; db < DB; ++db) {
                dv[db] = E::mfma(d.transposed(r0 + 16 * hh, db, lane), bw, dv[db]);
                dk[db] = E::mfma(q.transposed(r0 + 16 * hh, db, lane), bx, dk[db]);
            }
        }
    };

    // Positions of the queries from the wave's first key on.
    const PackedRuns runs(nt, t0 * BN + r0 + off - kw, BN, 32, p.lower, p.upper + 30, p.lower + 31, p.upper - 1);
    uint32_t flip = 0;  // the scale's sign, folded into K
    int u = 0;          // tiles so far
    if (n > 0) issue(hk * p.G + hd.g0, 0, 0);
    for (int gi = hd.g0; gi < hd.g1; ++gi) {
        const uint32_t fl = packed_flip<E>(arg_scale(p, hk * p.G + gi));
        if (fl != flip) {
            wait_vmcnt<0>();
            __syncthreads();  // K has arrived, and the last head's tiles are done
            for (int i = threadIdx.x; i < Keys::BYTES / 16; i += 64 * NW) reinterpret_cast<u32x4*>(keys)[i] ^= fl ^ flip;
            flip = fl;
        }
        int t = 0;
        auto run = [&](int end, auto kind) __attribute__((always_inline)) {
            for (; t < end; ++t, ++u) {
                wait_vmcnt<0>();
                __syncthreads();
                if (u + 1 < n) {
                    const bool last = t + 1 == nt;
                    issue(hk * p.G + gi + (last ? 1 : 0), last ? 0 : t + 1, (u + 1) % NST);
                }
                if constexpr (kind.value != 0) tile(t, u % NST, kind);
            }
        };
        run(runs.ta, PackedIdle{});
        run(runs.tf, PackedCut{});
        run(runs.tg, PackedFull{});
        run(runs.tv, PackedCut{});
        run(nt, PackedIdle{});
    }
    // The second half's sums to the first's waves, dK and then dV.
    static_assert(4 * 32 * (DP + 4) * 4 <= NST * STAGE + 2 * Keys::BYTES, "room for the shares");
    wait_vmcnt<0>();
    float* const red = reinterpret_cast<float*>(ring) + group * 32 * (DP + 4);
    auto join = [&](f32x16 (&acc)[DB]) __attribute__((always_inline)) {
        __syncthreads();
        if (part > 0) packed_put(red, acc, c, g);
        __syncthreads();
        if (part == 0) packed_add(acc, red, c, g);
    };
    packed_unfit<E>(f, dk);
    join(dk);
    join(dv);
    if (part > 0 || key >= sq.nk) return;
    const size_t at = ((size_t)(sq.k0 + key) * p.Hkv + hk) * D;  // contiguous (Nk, Hkv, D)
    packed_store_keys<E>(p, p.dk, 0, hd.split, at, dk, 2.f / kUp<E>, g);
    packed_store_keys<E>(p, p.dv, 1, hd.split, at, dv, 1.f / kUp<E>, g);
}

// ---------------------------------------------------------------------------
// dscale_h = (2 / s) sum_i delta_i eps / Z_i = (2 eps / |s|^3) sum_i delta_i zs_i:
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
__global__ __launch_bounds__(64) void born_packed_dscale_kernel(PackedArgs p, const double* part, float* dscale, int n_scale, double up) {
    double total = 0.0;
    for (int h = threadIdx.x; h < p.H; h += 64) {
        double x = 0.0;
        for (int i = 0; i < kPackedParts; ++i) x += part[(size_t)h * kPackedParts + i];
        const double s = fabs((double)arg_scale(p, h));
        x = s != 0.0 ? 2.0 * (double)p.eps / (s * s * s * up) * x : 0.0;
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
inline unsigned packed_blocks(int N, int S, int split) { return (unsigned)(N / packed_rows(split) + S + 1); }

// Waves that share a block's rows: the most that the ring has room for.
template <class E, int DP>
constexpr int kPackedMaxSplit = kItem<E> * DP <= 256 ? 4 : kItem<E> * DP <= 512 ? 2 : 1;

// How a launch of few blocks is divided.  The lengths are on the device, so the
// longest sequence is taken for half as long again as the mean.
struct PackedPlan {
    bool split_q, split_k;  // 32-row blocks of four waves: forward and dQ, fp32's dK/dV
    int head_splits;
};
inline PackedPlan packed_plan(int item, int64_t Nq, int64_t Nk, int64_t S, int64_t H, int64_t Hkv, int64_t D, int64_t window) {
    const int64_t rb = D <= 64 ? 64 * item : D <= 96 ? 96 * item : D <= 128 ? 128 * item : 256 * item;
    const double seqs = S > 0 ? (double)S : 1.0;
    PackedPlan r = {};
    // A block costs its start, its tiles and its end; a is the first and last
    // in 64-row tiles (fp32's are four times as long).  Split blocks walk a
    // quarter of the tiles, a third slower each, and above 128-byte rows have a
    // CU to themselves.  Measured, us unsplit and split: fp32 3 sequences of
    // 1000 tokens, 8 heads D64, forward 43 and 18, dQ 58 and 24; fp16 5
    // sequences of 3125 tokens, 6 heads D96, a window of 384: 17 and 26, 21 and 33.
    if (rb <= 512) {
        const double a = item == 2 ? 6.0 : 1.5, share = rb <= 256 ? 4.0 : 2.0;
        double longest = 1.5 * (double)Nk / seqs;
        if (longest > (double)Nk) longest = (double)Nk;
        if (window > 0 && longest > window + 128.0) longest = window + 128.0;
        const double c = longest / 64.0;
        const double whole = (double)packed_blocks((int)Nq, (int)S, 1) * H / (rb <= 256 ? 512.0 : 256.0);
        const double parts = (double)packed_blocks((int)Nq, (int)S, (int)share) * H / (rb == 128 ? 512.0 : 256.0);
        r.split_q = (parts > 1.0 ? parts : 1.0) * (a + 1.33 * c / share) < (whole > 1.0 ? whole : 1.0) * (a + c);
    }
    // fp32's dK/dV: 32-key blocks while 64-key ones would be under one a CU.
    const int64_t few = (int64_t)packed_blocks((int)Nk, (int)S, 4) * Hkv;
    r.split_k = item == 4 && rb <= 256 && few <= 512;
    // Heads of a group are shared out while that leaves a launch under four
    // blocks a CU, to even out their lengths, and a share some tiles.  Each
    // share costs its sums in fp32, written and read again.  Measured, us of
    // dK/dV and join by shares 1, 2, 4, 8: 2 sequences of 4096, 8 heads over 1,
    // D128, 776, 416, 241, 182; 4 of up to 3000, 32 heads over 8, D64, 253, 237,
    // 275.  At 548 blocks (16384 tokens, 16 heads over 4) ragged lengths would
    // still gain (D128, 541 and 509), equal ones lose (8 of 2048: D128 358 and
    // 407, D64 224 and 257; 32 of 512: 117 and 177): the lengths are not known
    // here, so the limit lies below.
    const int split = rb > 512 || (rb <= 256 && item == 2) ? 1 : r.split_k ? 4 : 2;
    const int64_t G = H / Hkv, blocks = (int64_t)packed_blocks((int)Nk, (int)S, split) * Hkv;
    double rows = 1.5 * (double)Nq / seqs;
    if (rows > (double)Nq) rows = (double)Nq;
    if (window > 0 && rows > window + 128.0) rows = window + 128.0;
    int64_t hs = 1;
    while (2 * hs <= G && 2 * hs * blocks <= 1024 && (double)(G / (2 * hs)) * rows / 64.0 >= 5.0) hs *= 2;
    r.head_splits = (int)hs;
    return r;
}
inline int64_t packed_part_bytes(const PackedPlan& r, int64_t Nk, int64_t Hkv, int64_t D) {
    return r.head_splits > 1 ? 2 * r.head_splits * Nk * Hkv * D * 4 : 0;
}

#define QDL_PACKED_DP(D, ...)                             \
    if ((D) <= 64) {                                      \
        constexpr int DPV = 64;                           \
        __VA_ARGS__                                            \
    } else if ((D) <= 96) {                               \
        constexpr int DPV = 96;                           \
        __VA_ARGS__                                            \
    } else if ((D) <= 128) {                              \
        constexpr int DPV = 128;                          \
        __VA_ARGS__                                            \
    } else {                                              \
        constexpr int DPV = 256;                          \
        __VA_ARGS__                                            \
    }

template <class E, int DP, int SPLIT>
void launch_packed_fwd_as(const PackedArgs& a, hipStream_t st) {
    const dim3 grid(packed_blocks(a.Nq, a.S, SPLIT) * (unsigned)a.H), block(64 * kPackedWaves);
    hipLaunchKernelGGL((born_packed_fwd_kernel<E, DP, SPLIT>), grid, block, 0, st, a);
}
template <class E, int DP, int SPLIT>
void launch_packed_dq_as(const PackedArgs& a, hipStream_t st) {
    const dim3 grid(packed_blocks(a.Nq, a.S, SPLIT) * (unsigned)a.H), block(64 * kPackedWaves);
    hipLaunchKernelGGL((born_packed_dq_kernel<E, DP, SPLIT>), grid, block, 0, st, a);
}
template <class E, int DP, int SPLIT, bool DK, bool DV>
void launch_packed_dkdv_as(const PackedArgs& a, hipStream_t st) {
    const dim3 grid(packed_blocks(a.Nk, a.S, SPLIT) * (unsigned)(a.Hkv * a.head_splits)), block(64 * kPackedWaves);
    hipLaunchKernelGGL((born_packed_dkdv_kernel<E, DP, SPLIT, DK, DV>), grid, block, 0, st, a);
}

template <class E>
hipError_t launch_packed_fwd(const PackedArgs& a, const PackedPlan& plan, hipStream_t st) {
    QDL_PACKED_DP(a.D, {
        if (kPackedMaxSplit<E, DPV> > 1 && plan.split_q) launch_packed_fwd_as<E, DPV, kPackedMaxSplit<E, DPV>>(a, st);
        else launch_packed_fwd_as<E, DPV, 1>(a, st);
    })
    return hipGetLastError();
}

// dQ first: it forms the rows' -delta and s^2 / Z.
template <class E>
hipError_t launch_packed_bwd(const PackedArgs& a, const PackedPlan& plan, hipStream_t st) {
    QDL_PACKED_DP(a.D, {
        if (a.Nq > 0) {
            if (kPackedMaxSplit<E, DPV> > 1 && plan.split_q) launch_packed_dq_as<E, DPV, kPackedMaxSplit<E, DPV>>(a, st);
            else launch_packed_dq_as<E, DPV, 1>(a, st);
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
        }
        if (a.Nk > 0 && a.dk != nullptr) {
            if constexpr (kItem<E> == 2 && DPV <= 128) {
                const dim3 grid(packed_blocks(a.Nk, a.S, 1) * (unsigned)(a.Hkv * a.head_splits));
                hipLaunchKernelGGL((born_packed_dkdv8_kernel<E, DPV>), grid, dim3(512), 0, st, a);
            } else if constexpr (kPackedMaxSplit<E, DPV> == 1) {
                launch_packed_dkdv_as<E, DPV, 1, true, false>(a, st);
                launch_packed_dkdv_as<E, DPV, 1, false, true>(a, st);
            } else if constexpr (kPackedMaxSplit<E, DPV> == 2) {
                launch_packed_dkdv_as<E, DPV, 2, true, true>(a, st);
            } else if (plan.split_k) {
                launch_packed_dkdv_as<E, DPV, 4, true, true>(a, st);
            } else {
                launch_packed_dkdv_as<E, DPV, 2, true, true>(a, st);
            }
        }
    })
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.Nk == 0 || a.dk == nullptr || a.head_splits == 1) return e;
    const int64_t pieces = (int64_t)a.Nk * a.Hkv * a.D / 4;  // of 8 values, dK and dV
    hipLaunchKernelGGL((born_packed_dkdv_join_kernel<E>), dim3((unsigned)((pieces + 255) / 256)), dim3(256), 0, st, a);
    return hipGetLastError();
}

// Entry points of the per-dtype translation units.
template <class E>
hipError_t packed_fwd(const PackedArgs& a, const PackedPlan& plan, hipStream_t st);
template <class E>
hipError_t packed_bwd(const PackedArgs& a, const PackedPlan& plan, hipStream_t st);

}  // namespace qdl
