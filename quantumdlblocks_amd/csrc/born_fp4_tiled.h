// Born attention of many new tokens per sequence over a paged cache in 4 bits:
// the kernel for sequences with more rows (new tokens x heads of a group) than
// the narrow one takes.
//
// 128 rows a workgroup, 32 a wave: S^T = K Q^T per 32 keys, the weights in
// place, O^T += V^T P^T, as the packed forward does it from 16 bits.  Tiles of
// keys are converted to bf16 once for the four waves: each thread has a block of
// 32 columns of K and of V, its codes loaded two tiles ahead into registers,
// converted one tile ahead into the other half of LDS, one barrier a tile.
// Sixteen lanes that write LDS together have one block of 16 keys, which the
// rows' swizzle spreads over all banks.
//
// 8 second turns (4583 tokens over 27 thousand keys, 32 heads over 8, D128 bf16):
// 330 us, 685 TFLOP/s of the formula's, and a join of 5; a large matrix product
// has 1200.  The weights' two parts make three products of the formula's two: with
// one part it was 250 us, but a row was off by 2.3e-3 in norm where the narrow
// kernel's are by 1.7e-3, so that its precision hung on what else was in the batch.
// The matrix pipe is busy in 50% of the cycles, vector instructions issue in 55:
// two workgroups a compute unit is what 256 registers leave, and with one column
// block of 32 rows a wave each operand of K from LDS feeds one product.  A higher
// priority around the overlaps' products: 328 us for 332.
//
// Keys without a page, or past the sequence, are zeros: overlaps of 0, weights
// of 0.  Few blocks of rows split their keys; the partial sums are joined in order.
#pragma once

#include "born_fp4_paged.h"

namespace qdl {

template <class E, int DP>
struct Fp4TileCfg {
    static constexpr int BN = DP == 256 ? 32 : 64, SUB = BN / 32, NB = DP / 32;
    static constexpr int BYTES = BN * DP * 2, STAGE = 2 * BYTES;
    static constexpr int UNITS = BN * NB / 256;  // blocks of K (and of V) of a thread; 0: K or V
    // Waves a SIMD.  fp32 at D128 spills some 65 vector registers, 115 with the narrow
    // part, fp16 up to 5; at D256 the narrow part makes fp16 spill some 55, fp32 150.
    static constexpr int WPE = DP == 256 ? 1 : 2;
};

// Block x of rows: part i of a sequence's.  With a lane for each sequence those
// of the longest come first, so that a launch ends with short ones (the 8 second
// turns, with one part of the weights, 264 us, in the sequences' order 327).
__device__ __forceinline__ Fp4Part fp4_block(const Fp4PagedArgs& p, const Fp4Share& share, int x) {
    if (p.items > 0 && p.B <= 64) {
        const int k = share.lane() < p.B ? share.mine.blocks(p) : 0;
        int before = 0;
        for (int j = 0; j < p.B; ++j) {
            const int n = __builtin_amdgcn_readlane(share.mine.n, j);
            if (n > share.mine.n || (n == share.mine.n && j < share.lane())) before += __builtin_amdgcn_readlane(k, j);
        }
        const uint64_t here = __ballot(before <= x && x < before + k);
        const int l = __builtin_amdgcn_readfirstlane(here != 0 ? __ffsll((long long)here) - 1 : 0);
        return Fp4Part{here != 0 ? l : -1, x - __builtin_amdgcn_readlane(before, l), 0, share.mine.of_lane(l)}.uniform();
    }
    if (p.items > 0) return fp4_part(p, share, x, [&](const Fp4Seq& s) { return s.blocks(p); });
    // Sequence s has the slots from cu[s] G / 128 + s on: never fewer than it has blocks.
    const int lane = threadIdx.x & 63;
    auto slot = [&](int s) { return (int)((int64_t)(s == 0 ? 0 : min(max(p.cu[s], 0), p.N)) * p.G / kFp4Rows) + s; };
    int lo = 0, hi = p.B + 1;
    while (hi - lo > 1) {
        const int step = (hi - lo + 63) / 64, i = lo + (lane + 1) * step;
        const bool below = i < hi && slot(i) <= x;
        lo += (int)__popcll(__ballot(below)) * step;
        hi = min(hi, lo + step);
    }
    const int s = __builtin_amdgcn_readfirstlane(lo);
    const Fp4Seq sq(p, min(s, p.B - 1));
    return Fp4Part{s < p.B ? s : -1, x - slot(s), 0, sq}.uniform();
}

template <class E, int DP, bool P16>
__device__ __forceinline__ void fp4_tiled(const Fp4PagedArgs& p, const Fp4Share& share, uint8_t* ring, int* bad_tile, int block) {
    using C = Fp4TileCfg<E, DP>;
    using Tile = PackedTile<BF16, DP, C::BN>;
    constexpr int BN = C::BN, SUB = C::SUB, NB = C::NB, KS = DP / 16, DB = DP / 32, QP = kQParts<E>, PP = kPParts<E>, IT = kItem<E>;
    const int idx = block / p.Hkv, hk = block - idx * p.Hkv, split = idx / share.wide;
    const Fp4Part blk = fp4_block(p, share, idx - split * share.wide);
    const Fp4Seq& sq = blk.sq;
    const int rows = sq.nq * p.G, m0 = blk.i * kFp4Rows;
    // Where starts do not ascend there are more blocks than slots, or some before the first.
    if (blk.b < 0 || !sq.wide(p) || (uint32_t)m0 >= (uint32_t)rows || (uint32_t)split >= (uint32_t)p.splits) return;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 31, g = lane >> 5;
    const int past = sq.n - sq.nq;  // keys before the first new token
    const int m1 = min(rows, m0 + kFp4Rows) - 1;
    // Keys that any row of the block sees, in tiles; this split's.
    const int jlo = p.window > 0 ? max(0, past + m0 / p.G - p.window + 1) : 0, jhi = min(sq.n - 1, past + m1 / p.G);
    const int first = jlo / BN, all = jhi >= jlo ? jhi / BN - first + 1 : 0;
    const int per = (all + p.splits - 1) / p.splits, t0 = first + split * per, n = max(0, min(all - split * per, per));

    // The wave's rows, the lane's.
    const int rw = m0 + 32 * wave, row = rw + c;
    const bool ok = row < rows;
    const int tok = ok ? row / p.G : 0, head = hk * p.G + (ok ? row - tok * p.G : 0);
    const int pos = past + tok;
    const float sc = arg_scale(p, head);
    f32x16 acc[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db) acc[db] = zero16();
    float z = 0.f;

    // A thread's key of each tile and its block; K and V of it, or one of them.
    constexpr bool kOne = C::UNITS == 0;
    const int key_in = DP == 256 ? 16 * (tid >> 7) + (tid & 15) : 16 * (tid >> 6) + (tid & 15);
    const int bi = DP == 256 ? (tid >> 4) & 7 : DP == 128 ? (tid >> 4) & 3 : (tid >> 4) & 1;
    const bool is_v = kOne && ((tid >> 5) & 1) != 0;
    const bool in_row = bi < p.c.nb;
    const ConstIntPtr table = (ConstIntPtr)(uintptr_t)(p.t.table + (int64_t)blk.b * p.t.table_ld);
    const uint8_t* const kc = p.c.k + (uint64_t)hk * p.c.kh + 16 * bi;
    const uint8_t* const vc = p.c.v + (uint64_t)hk * p.c.vh + 16 * bi;
    const uint8_t* const ksc = p.c.ks + (uint64_t)hk * p.c.ksh + bi;
    const uint8_t* const vsc = p.c.vs + (uint64_t)hk * p.c.vsh + bi;

    struct Codes {
        u32x4 x[kOne ? 1 : 2];
        uint32_t ks, vs;
    };
    Codes next;
    // Page of the thread's key in tile t0 + u, -1: none.
    auto page_of = [&](int u) __attribute__((always_inline)) {
        int j = (t0 + u) * BN + key_in;
        if constexpr (P16) {  // sixteen keys of a wave, one page: a scalar load
            const int k0 = (t0 + u) * BN + (DP == 256 ? 16 * (wave >> 1) : 16 * wave);
            const int i = __builtin_amdgcn_readfirstlane(fp4_page(p.c, min(k0, sq.n - 1)));
            return (int)table[i];
        } else {
            return (int)table[fp4_page(p.c, min(j, sq.n - 1))];
        }
    };
    auto fetch = [&](Codes& y, int u, int page) __attribute__((always_inline)) {
        const int j = (t0 + u) * BN + key_in;
        y.ks = y.vs = 0;
#pragma unroll
        for (int i = 0; i < (kOne ? 1 : 2); ++i) y.x[i] = u32x4{0u, 0u, 0u, 0u};
        if (!(in_row && j < sq.n && page >= 0 && page < p.c.cache_pages)) return;
        const int r = j - fp4_page(p.c, j) * p.c.page;
        y.ks = ksc[fp4_at(page, p.c.ksp, r, p.c.kst, 0, 0)];
        y.vs = vsc[fp4_at(page, p.c.vsp, r, p.c.vst, 0, 0)];
        const uint8_t *ka = kc + fp4_at(page, p.c.kp, r, p.c.kt, 0, 0), *va = vc + fp4_at(page, p.c.vp, r, p.c.vt, 0, 0);
        if constexpr (kOne) {
            y.x[0] = ldg16(is_v ? va : ka);
        } else {
            y.x[0] = ldg16(ka);
            y.x[1] = ldg16(va);
        }
    };
    auto kt = [&](int st) { return Tile{ring + st * C::STAGE}; };
    auto vt = [&](int st) { return Tile{ring + st * C::STAGE + C::BYTES}; };
    auto put = [&](const Codes& y, int u) __attribute__((always_inline)) {
        const int st = u & 1;
        const bool bad = y.ks == kFp4Bad || y.vs == kFp4Bad;
        const bool any_bad = __ballot(bad) != 0;
        if (any_bad && lane == 0) bad_tile[st] = u;
#pragma unroll
        for (int i = 0; i < (kOne ? 1 : 2); ++i) {
            const bool v = kOne ? is_v : i == 1;
            const float s = fp4_scale(v ? y.vs : y.ks);
            uint8_t* const to = ring + st * C::STAGE + (v ? C::BYTES : 0) + key_in * Tile::RB;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                u32x4 x = fp4_eight(y.x[i][w], s);
                if (any_bad && bad) x = v ? u32x4{0u, 0u, 0u, 0u} : u32x4{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u};
                *reinterpret_cast<u32x4*>(to + (((4 * bi + w) ^ Tile::swz(key_in)) << 4)) = x;
            }
        }
    };

    // The first tiles' codes are on their way before anything waits for the queries.
    int page = -1;
    Codes first_codes;
    if (n > 0) {
        page = page_of(0);
        const int page1 = n > 1 ? page_of(1) : -1;
        fetch(first_codes, 0, page);
        fetch(next, 1, page1);
        page = n > 2 ? page_of(2) : -1;
    }
    u32x4 qr[KS][QP];
    {
        const uint8_t* at = (const uint8_t*)p.q + (int64_t)(sq.q0 + tok) * p.q_st + (int64_t)head * p.q_sh;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) fp4_query<E>(at, 16 * ks + 8 * g, p.D, ok, sc < 0.f, qr[ks]);
    }
    // Rows that are not numbers, or infinite, whose sums may be NaN: 0 times them is.
    f32x16 none = zero16();
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) none = BF16::mfma(u32x4{0u, 0u, 0u, 0u}, qr[ks][0], none);
    const bool bad_rows = __ballot(none[0] != none[0]) != 0;
    auto tile = [&](int u, int st, auto kind) __attribute__((always_inline)) {
        const int key0 = (t0 + u) * BN;
        const Tile k = kt(st), v = vt(st);
        const bool bad_here = bad_rows || __builtin_amdgcn_readfirstlane(bad_tile[st]) == u;
#pragma unroll
        for (int nb = 0; nb < SUB; ++nb) {
            f32x16 s = zero16();
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const u32x4 a = k.row(32 * nb + c, ks, g);
#pragma unroll
                for (int u2 = 0; u2 < QP; ++u2) s = BF16::mfma(a, qr[ks][u2], s);
            }
            __builtin_amdgcn_s_setprio(0);
            if (bad_here) {  // the sum's NaN may have either sign, the weights take a positive one
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = s[r] == s[r] ? s[r] : __uint_as_float(0x7fc00000u);
            }
            if constexpr (kind.value == 2) {
                const uint32_t span = p.window > 0 ? (uint32_t)p.window : 0x80000000u;
                const int d = pos - key0 - 32 * nb;
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if ((uint32_t)(d - acc_row(r, g)) >= span) s[r] = 0.f;
            }
            uint32_t wt[8][PP];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float a0 = relu_f32(s[2 * j]), a1 = relu_f32(s[2 * j + 1]);
                z = (z + a0 * a0) + a1 * a1;
                fp4_parts<PP>(a0 * a0, a1 * a1, wt[j]);
            }
#pragma unroll
            for (int hh = 0; hh < 2; ++hh)
#pragma unroll
                for (int db = 0; db < DB; ++db) {
                    const u32x4 a = v.transposed(32 * nb + 16 * hh, db, lane);
#pragma unroll
                    for (int k2 = 0; k2 < PP; ++k2) {
                        const u32x4 w = {wt[4 * hh][k2], wt[4 * hh + 1][k2], wt[4 * hh + 2][k2], wt[4 * hh + 3][k2]};
                        acc[db] = BF16::mfma(a, w, acc[db]);
                    }
                }
        }
    };

    // Runs of tiles that the wave's rows see not at all, in part, whole: each
    // a loop of its own.
    const int a0 = p.window > 0 ? past + rw / p.G - p.window + 1 : 0, a1 = past + min(rw + 31, rows - 1) / p.G;
    const int b0 = p.window > 0 ? past + min(rw + 31, rows - 1) / p.G - p.window + 1 : 0, b1 = past + rw / p.G;
    const bool idle = rw >= rows;
    const PackedRuns runs(n, t0 * BN, BN, BN, idle ? 1 << 30 : a0, idle ? 1 << 30 : a1, b0, b1);
    if (n > 0) {
        if (tid < 2) bad_tile[tid] = -1;
        __syncthreads();
        put(first_codes, 0);
        int u = 0;
        auto run = [&](int end, auto kind) __attribute__((always_inline)) {
            for (; u < end; ++u) {
                __syncthreads();
                if (u + 1 < n) {
                    put(next, u + 1);
                    if (u + 2 < n) fetch(next, u + 2, page);
                    if (u + 3 < n) page = page_of(u + 3);
                }
                if constexpr (kind.value != 0) tile(u, u & 1, kind);
            }
        };
        run(runs.ta, PackedIdle{});
        run(runs.tf, PackedCut{});
        run(runs.tg, PackedFull{});
        run(runs.tv, PackedCut{});
        run(n, PackedIdle{});
    }
    z += __shfl_xor(z, 32);
    if (!ok) return;
    const int64_t at = (int64_t)(sq.q0 + tok) * p.H + head;
    if (p.splits > 1) {
        float* to = p.wide_part + (at * p.splits + split) * (p.D + 4);
        packed_store_row<F32>((uint8_t*)(to + 4), acc, 1.f, p.D, g);
        if (g == 0) to[0] = z;
    } else {
        packed_store_row<E>((uint8_t*)p.out + at * p.D * IT, acc, fp4_inverse(p, head, z), p.D, g);
    }
}

// Wide sequences alone, or sequences of all sizes in one launch (NARROW), so that
// neither kernel waits for the other: the tiled one's workgroups, the narrow one's,
// and those of the grid that the host could not know to be none.
template <class E, int DP, bool P16, bool NARROW>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(Fp4TileCfg<E, DP>::WPE)))
void born_fp4_chunk_kernel(Fp4PagedArgs p) {
    constexpr int kTiles = 2 * Fp4TileCfg<E, DP>::STAGE, kBytes = kTiles > kFp4NarrowLds<DP> || !NARROW ? kTiles : kFp4NarrowLds<DP>;
    __shared__ __attribute__((aligned(1024))) uint8_t smem[kBytes];
    __shared__ int bad_tile[2];  // the last tile of each stage that holds a token that is not a number
    if constexpr (NARROW) fp4_behind<E>(p, blockIdx.x, gridDim.x);
    const Fp4Share share(p, true);
    const int tiled = share.wide * p.splits * p.Hkv, x = blockIdx.x;
    if (x < tiled) {
        fp4_tiled<E, DP, P16>(p, share, smem, bad_tile, x);
    } else if (NARROW && x < tiled + share.units * p.Hkv) {
        const int y = x - tiled, unit = y / p.Hkv;
        fp4_narrow<E, DP, 2, false, P16>(p, share, smem, unit, y - unit * p.Hkv);
    }
}

template <class E, bool P16, bool NARROW>
void launch_fp4_chunk_dp(const Fp4PagedArgs& a, int64_t grid, hipStream_t st) {
    const dim3 g((unsigned)grid);
    if (a.D <= 64) hipLaunchKernelGGL((born_fp4_chunk_kernel<E, 64, P16, NARROW>), g, dim3(256), 0, st, a);
    else if (a.D <= 128) hipLaunchKernelGGL((born_fp4_chunk_kernel<E, 128, P16, NARROW>), g, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((born_fp4_chunk_kernel<E, 256, P16, NARROW>), g, dim3(256), 0, st, a);
}
template <class E, bool P16>
hipError_t launch_fp4_parts(const Fp4PagedArgs& a, const Fp4Plan& plan, hipStream_t st) {
    if (plan.slots > 0 && !plan.apart) {
        launch_fp4_chunk_dp<E, P16, true>(a, plan.grid, st);
        return hipGetLastError();
    }
    launch_fp4_nc<E, P16>(a, plan, st);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || plan.slots == 0) return e;
    launch_fp4_chunk_dp<E, P16, false>(a, plan.slots * plan.splits * a.Hkv, st);
    return hipGetLastError();
}

template <class E>
hipError_t launch_fp4(const Fp4PagedArgs& a, const Fp4Plan& plan, hipStream_t st) {
    const hipError_t e = fp4_p16(a.c) ? launch_fp4_parts<E, true>(a, plan, st) : launch_fp4_parts<E, false>(a, plan, st);
    return e != hipSuccess ? e : launch_fp4_join<E>(a, plan, st);
}

}  // namespace qdl
