// Born attention over a paged cache in 4 bits, for one new token per sequence
// or for several:
//
//   p_ij = (s relu(sign(s) q_i.k_j))^2 over the keys j that token i sees,
//   O_i = sum_j p_ij v_j / (sum_j p_ij + eps).
// Sequence b's tokens stand at the last of its n keys; token at position i sees
// keys max(0, i - window + 1) .. i.  G = H / Hkv query heads read one key head,
// so a sequence has new G rows for each key head: row r is head r % G of token
// r / G.
//
// Narrow kernel: 16 NC rows are the columns of S^T = K Q^T (16-key products),
// the keys split over workgroups and a workgroup's four waves, every fourth 32
// keys each.  K's codes go from memory into the A operand by conversions alone:
// a lane's 16 bytes are one block, and the order of the head dim's columns
// within a product is free, so a dword of codes is an operand.  V's rows come as
// DP / 16 columns a lane and 8 keys, are converted and paired by byte permutes.
// The 16-key products' C layout is the next product's B operand.
//
// The keys are shared out on the device, which knows the lengths: chunk = the
// keys of all sequences over the workgroups wanted, in steps of 128, and each
// sequence takes as many chunks as it needs.  Partial sums are joined in order.
//
// 32 single tokens over long caches (267 MB, 8 key heads D128, 4 heads each, bf16):
// 65 us, 4.1 TB/s, and a join of 5: K's and V's conversions make most of some 195
// vector instructions for a wave's 32 keys, beside 24 matrix and 140 scalar ones,
// and the vector instructions take half of the SIMDs' cycles beside the loads, which
// are two steps ahead.  16 sequences of 5 tokens over 51 thousand keys (4 key heads)
// 20 us and 6 where the bytes take 6: with two column sets the loads' descriptors do
// not fit the scalar registers, and each 32 keys read some 60 back; one token over
// 1531 keys 7 and 4: chains of loads, the lengths, the table's entry, the codes, the
// partial sums, a microsecond each.  Read without a page's base in scalars, 92 us
// for 73.
#pragma once

#include "born_fp4.h"
#include "fp4_plan.h"

namespace qdl {

struct Fp4PagedArgs {
    const void* q;  // rows (token, head)
    void* out;
    Fp4Cache c;
    Fp4Pages t;
    const int32_t* cu;  // B + 1 starts, or nullptr: one token per sequence
    const float* scale;
    float scale_value;
    int per_head_scale;
    int B, N, H, Hkv, G, D;
    int window;
    int items;             // units (a chunk of keys and a column block) wanted; 0: cblocks for each sequence
    int cblocks;           // column blocks of a sequence at most
    int cols;              // rows of one
    int limit;             // rows of a (sequence, key head) that the narrow kernel takes
    int splits;            // of the tiled kernel's keys
    int64_t slots;         // blocks of rows at most; 0: no sequence is wide
    float* wide_part;      // (N, H, splits, D + 4), where there are several
    float eps;
    int64_t q_st, q_sh;    // bytes
    int2* plan;            // (B): a sequence's first unit and its chunks
    float* part;           // (units, Hkv, cols, D + 4): denominator, three unused, numerators
    float* weights;        // (B, Hkv, L) or nullptr: += sum over the group of p / Z
    int64_t w_sb, w_sh;    // elements
    int w_len;
    float* raw;            // (B, H, raw_ld): p without s^2, -1 without a page, of keys from the span's first 32 on, as far as weights are kept
    int64_t raw_ld;
    int units;             // at most: `part` has room for no more
};

// A sequence: its tokens (rows of q), keys, and the first key that any token sees.
struct Fp4Seq {
    int q0, nq, n, first;
    __device__ __forceinline__ Fp4Seq(const Fp4PagedArgs& p, int b) {
        q0 = b;
        nq = 1;
        if (p.cu != nullptr) {
            q0 = b == 0 ? 0 : min(max(p.cu[b], 0), p.N);
            nq = max(min(p.cu[b + 1], p.N) - q0, 0);
        }
        n = p.c.cache_pages > 0 ? fp4_len(p.c, p.t, b) : 0;
        first = fp4_first(n, nq, p.window);
    }
    __device__ __forceinline__ Fp4Seq of_lane(int l) const {
        Fp4Seq r = *this;
        r.q0 = __builtin_amdgcn_readlane(q0, l);
        r.nq = __builtin_amdgcn_readlane(nq, l);
        r.n = __builtin_amdgcn_readlane(n, l);
        r.first = __builtin_amdgcn_readlane(first, l);
        return r;
    }
    __device__ __forceinline__ int base() const { return first & ~31; }
    __device__ __forceinline__ bool wide(const Fp4PagedArgs& p) const { return p.cu != nullptr && (int64_t)nq * p.G > p.limit; }
    // The narrow kernel's chunks are counted in steps of 128 keys.
    __device__ __forceinline__ int steps(const Fp4PagedArgs& p) const { return wide(p) ? 0 : fp4_steps(n, first); }
    // The narrow kernel's column blocks.
    __device__ __forceinline__ int columns(const Fp4PagedArgs& p) const { return wide(p) ? 0 : fp4_blocks(nq * p.G, p.cols); }
    // The tiled kernel's blocks of rows.
    __device__ __forceinline__ int blocks(const Fp4PagedArgs& p) const { return wide(p) ? (nq * p.G + kFp4Rows - 1) / kFp4Rows : 0; }
};

// Inclusive sums over the lanes of a wave: lane 63 has the total.
__device__ __forceinline__ int fp4_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);   // row_shr 1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast 15 to rows 1 and 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast 31 to rows 2 and 3
    return x;
}

// How the device shares out a call, found by every wave for itself: units (a
// chunk of the keys and a column block) of the narrow sequences, blocks of the
// wide ones' rows.
struct Fp4Share {
    int step;         // steps of 128 keys in a chunk
    int units, wide;  // how many there are
    Fp4Seq mine;      // sequence `lane`

    // totals: units and wide are wanted.
    __device__ __forceinline__ Fp4Share(const Fp4PagedArgs& p, bool totals) : step(1 << 23), units(p.B * p.cblocks), wide((int)p.slots), mine(p, min(lane(), p.B - 1)) {
        if (p.items == 0) return;  // too many sequences to look through: one chunk each, slots for blocks
        uint64_t total = 0;
        wide = 0;
        each(p, [&](const Fp4Seq& s, int b0) {
            const bool in = b0 + lane() < p.B;
            const uint64_t mine = in ? (uint64_t)(uint32_t)s.steps(p) * (uint32_t)s.columns(p) : 0;
            // Sums of 64 in 32 bits, the upper ones where there are any.
            total += (uint32_t)last(fp4_scan((int)(mine & 0xffffffu)));
            if (__ballot(mine >> 24 != 0) != 0) total += (uint64_t)(uint32_t)last(fp4_scan((int)(mine >> 24))) << 24;
            if (totals) wide += last(fp4_scan(in ? s.blocks(p) : 0));
            return false;
        });
        step = fp4_step(total, p.items);
        if (!totals) return;
        units = 0;
        each(p, [&](const Fp4Seq& s, int b0) {
            units += last(fp4_scan(b0 + lane() < p.B ? count(p, s) : 0));
            return false;
        });
    }
    __device__ __forceinline__ static int lane() { return threadIdx.x & 63; }
    __device__ __forceinline__ static int last(int scan) { return __builtin_amdgcn_readlane(scan, 63); }
    __device__ __forceinline__ int chunks(const Fp4PagedArgs& p, const Fp4Seq& s) const { return (s.steps(p) + step - 1) / step; }
    __device__ __forceinline__ int count(const Fp4PagedArgs& p, const Fp4Seq& s) const { return chunks(p, s) * s.columns(p); }
    // Every 64 sequences, until f is done.
    template <class F>
    __device__ __forceinline__ void each(const Fp4PagedArgs& p, F&& f) const {
        if (f(mine, 0)) return;
        for (int b0 = 64; b0 < p.B; b0 += 64)
            if (f(Fp4Seq(p, min(b0 + lane(), p.B - 1)), b0)) return;
    }
};

// A sequence and which of its parts: scalars.
struct Fp4Part {
    int b, i, n;  // b < 0: none; part i of n
    Fp4Seq sq;
    __device__ __forceinline__ Fp4Part uniform() const {
        return {__builtin_amdgcn_readfirstlane(b), __builtin_amdgcn_readfirstlane(i), __builtin_amdgcn_readfirstlane(n), sq.of_lane(0)};
    }
};
// Part x of all, where sequence s has parts(s) of them.
template <class F>
__device__ __forceinline__ Fp4Part fp4_part(const Fp4PagedArgs& p, const Fp4Share& share, int x, F&& parts) {
    Fp4Part r = {-1, 0, 1, share.mine};
    int before = 0;
    share.each(p, [&](const Fp4Seq& s, int b0) {
        const int k = b0 + share.lane() < p.B ? parts(s) : 0, run = fp4_scan(k), at = before + run - k;
        const uint64_t here = __ballot(at <= x && x < at + k);
        if (here != 0) {
            const int l = __builtin_amdgcn_readfirstlane(__ffsll((long long)here) - 1);
            r = {b0 + l, x - __builtin_amdgcn_readlane(at, l), __builtin_amdgcn_readlane(k, l), s.of_lane(l)};
            return true;
        }
        before += share.last(run);
        return false;
    });
    return r.uniform();
}
// Unit x: part i is column block i % columns of chunk i / columns.
__device__ __forceinline__ Fp4Part fp4_unit(const Fp4PagedArgs& p, const Fp4Share& share, int x) {
    if (p.items == 0) {
        const int b = p.cblocks > 1 ? x / p.cblocks : x;
        return {b, x - b * p.cblocks, p.cblocks, Fp4Seq(p, b)};
    }
    return fp4_part(p, share, x, [&](const Fp4Seq& s) { return share.count(p, s); });
}

__device__ __forceinline__ float fp4_inverse(const Fp4PagedArgs& p, int h, float z) {
    const float s = arg_scale(p, h), den = z + (p.eps == 0.f ? 0.f : p.eps / (s * s));
    // A denominator that is not a number stays one.
    return s != 0.f ? (den < 0x1p-126f ? 0.f : 1.0f / den) : z == z ? 0.f : z;
}

// Rows behind the last sequence: zeros, shared out over `blocks` workgroups.
template <class E>
__device__ __forceinline__ void fp4_behind(const Fp4PagedArgs& p, int block, int blocks) {
    if (p.cu == nullptr) return;
    const int last = min(max(p.cu[p.B], 0), p.N), pieces = p.H * p.D * kItem<E> / 16;
    for (int r = last + block; r < p.N; r += blocks)
        for (int i = threadIdx.x; i < pieces; i += 256)
            *reinterpret_cast<u32x4*>((uint8_t*)p.out + ((int64_t)r * pieces + i) * 16) = u32x4{0u, 0u, 0u, 0u};
}

template <class E, int DP>
struct Fp4Cfg {
    static constexpr int KB = DP == 256 ? 2 : 1;       // K: pieces of a lane's key, j4 + 4 i
    static constexpr int KW = DP == 64 ? 2 : 4;        // dwords of a piece
    static constexpr int KS = KB * KW;                 // 32-column products
    static constexpr int VC = DP / 16, VD = (VC + 7) / 8;  // columns of a lane's key, dwords of codes
};

// Waves a SIMD that the kernel's registers are held to.  One column set keeps all of
// them, and so does bf16; with two at D256 fp16 spills some 55 vector registers and
// fp32 some 145, in the loop.
template <class E>
constexpr int fp4_wpe(int DP, int NC) {
    return DP == 256 ? 1 : NC == 2 ? (kQParts<E> < 3 || DP == 64 ? 2 : 1) : kQParts<E> == 1 || DP == 64 ? 3 : 2;
}

// A wave's 32 keys, as stored.
template <class E, int DP>
struct Fp4Keys {
    using C = Fp4Cfg<E, DP>;
    uint32_t k[2][C::KB][C::KW];
    uint32_t ks[2][C::KB], kvs[2][C::KB];  // the scales of K's blocks, and of V's same ones
    uint32_t v[8][C::VD], vs[8];
    bool there[2];  // pages of 16 keys from a multiple of 16 (P16)
    uint32_t seen;  // of the keys that the lane's V rows are, else
};

template <int DW>
__device__ __forceinline__ void fp4_load(uint32_t (&to)[DW], const uint8_t* p) {
    if constexpr (DW == 4) {
        const u32x4 x = ldg16(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) to[i] = x[i];
    } else {
        const u32x2 x = *reinterpret_cast<const u32x2*>(p);
        to[0] = x[0];
        to[1] = x[1];
    }
}

// The same by a buffer's scalar base and a lane's 32-bit offset.
typedef __amdgpu_buffer_rsrc_t Fp4Rsrc;
__device__ __forceinline__ Fp4Rsrc fp4_rsrc(const uint8_t* base) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base), 0, 0x7fffffff, 0x00020000);
}
template <int DW>
__device__ __forceinline__ void fp4_fetch(uint32_t (&to)[DW], Fp4Rsrc p, uint32_t offset) {
    if constexpr (DW == 4) {
        const u32x4 x = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(p, offset, 0, 0));
#pragma unroll
        for (int i = 0; i < 4; ++i) to[i] = x[i];
    } else {
        const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(p, offset, 0, 0));
        to[0] = x[0];
        to[1] = x[1];
    }
}

// LDS of the narrow kernel: the waves' sums of 16 rows.
template <int DP>
constexpr int kFp4NarrowLds = 4 * 16 * (DP + 4 + 1) * 4;

// Unit `unit` of key head hk.  DP: 64, 128 or 256 columns; NC: 16-row column
// sets; WEIGH: the raw weights are written too (one token per sequence); P16:
// pages of a multiple of 16 tokens.
template <class E, int DP, int NC, bool WEIGH, bool P16>
__device__ __forceinline__ void fp4_narrow(const Fp4PagedArgs& p, const Fp4Share& share, uint8_t* smem, int unit, int hk) {
    using C = Fp4Cfg<E, DP>;
    constexpr int NW = 4, QP = kQParts<E>, PP = kPParts<E>, KB = C::KB, KW = C::KW, KS = C::KS, VC = C::VC, VD = C::VD;
    constexpr int IT = kItem<E>;
    auto& red = *reinterpret_cast<float(*)[NW][16][DP + 4]>(smem);
    auto& zred = *reinterpret_cast<float(*)[NW][16]>(smem + NW * 16 * (DP + 4) * 4);

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int m = lane & 15, j4 = lane >> 4;
    const Fp4Part it = fp4_unit(p, share, unit);
    const int b = it.b, chunk = share.step << 7;
    const Fp4Seq& sq = it.sq;
    if (b < 0 || sq.wide(p)) return;
    const int columns = p.items == 0 ? p.cblocks : sq.columns(p);
    const int c = columns > 1 ? it.i / columns : it.i, cb = it.i - c * columns, nsplit = p.items == 0 ? 1 : share.chunks(p, sq);
    if (it.i == 0 && hk == 0 && threadIdx.x == 0) p.plan[b] = int2{unit, nsplit};
    const int rows = sq.nq * p.G, c0 = 16 * NC * cb;
    if (c0 >= rows) return;
    const int s0 = sq.base() + (p.items == 0 ? 0 : c) * chunk, s1 = min(sq.n, s0 + chunk);

    // The keys that every row of the block sees.
    int all_hi = sq.n - 1, all_lo = sq.first;
    if (p.cu != nullptr) {
        all_hi = sq.n - sq.nq + c0 / p.G;
        if (p.window > 0) all_lo = sq.n - sq.nq + (min(c0 + 16 * NC, rows) - 1) / p.G - p.window + 1;
    }

    f32x4v acc[NC][VC];
    float z[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        z[i] = 0.f;
#pragma unroll
        for (int e = 0; e < VC; ++e) acc[i][e] = f32x4v{0.f, 0.f, 0.f, 0.f};
    }

    // A lane's pieces of K and columns of V; those past the row are read from
    // its start and taken as zeros (K) or never stored (V).
    int ko[KB], kb[KB], vo, vb;
    uint32_t kmask[KB];
#pragma unroll
    for (int a = 0; a < KB; ++a) {
        const int at = 4 * KW * (j4 + 4 * a), blk = at / 16;
        const bool in = blk < p.c.nb;
        ko[a] = in ? at : 0;
        kb[a] = in ? blk : 0;
        kmask[a] = in ? ~0u : 0u;
    }
    {
        const bool in = VC * m < kFp4Block * p.c.nb;
        vo = in ? VC * m / 2 : 0;
        vb = in ? VC * m / kFp4Block : 0;
    }
    const bool whole = kFp4Block * p.c.nb == DP;
    const uint8_t *const kc = p.c.k + (uint64_t)hk * p.c.kh, *const vc = p.c.v + (uint64_t)hk * p.c.vh;
    const uint8_t *const ksc = p.c.ks + (uint64_t)hk * p.c.ksh, *const vsc = p.c.vs + (uint64_t)hk * p.c.vsh;
    const ConstIntPtr table = (ConstIntPtr)(uintptr_t)(p.t.table + (int64_t)b * p.t.table_ld);

    // Offsets of the lane's K rows (m) and V rows (4 j4 + r) within 16 keys of a
    // page: added to scalar bases they cost nothing per load.
    uint32_t ok_[KB], oks[KB], okv[KB], ov[4], ovs[4];
    if constexpr (P16) {
#pragma unroll
        for (int a = 0; a < KB; ++a) {
            ok_[a] = m * p.c.kt + ko[a];
            oks[a] = m * p.c.kst + kb[a];
            okv[a] = m * p.c.vst + kb[a];
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            ov[r] = (4 * j4 + r) * p.c.vt + vo;
            ovs[r] = (4 * j4 + r) * p.c.vst + vb;
        }
    }
    // Keys key0 + 16 t + m for K, key0 + 16 t + 4 j4 + i for V.
    auto load = [&](Fp4Keys<E, DP>& x, int key0) __attribute__((always_inline)) {
        if constexpr (P16) {
            // Sixteen keys are rows of one page, all of them memory of the cache's;
            // without a page, or behind the last key, they are read from page 0,
            // and use() drops what no row of the block sees.
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int j = key0 + 16 * t;
                const int i = fp4_page(p.c, min(j, sq.n - 1));
                const int32_t page = table[i];
                x.there[t] = j < sq.n && page >= 0 && page < p.c.cache_pages;
                const uint32_t at = x.there[t] ? page : 0, row = x.there[t] ? j - i * p.c.page : 0;
                auto base = [&](const uint8_t* c, uint32_t sp, uint32_t st) __attribute__((always_inline)) {
                    return fp4_rsrc(c + (uint64_t)at * sp + row * st);
                };
                const Fp4Rsrc kp = base(kc, p.c.kp, p.c.kt), ksp = base(ksc, p.c.ksp, p.c.kst);
                const Fp4Rsrc vp = base(vc, p.c.vp, p.c.vt), vsp = base(vsc, p.c.vsp, p.c.vst);
#pragma unroll
                for (int a = 0; a < KB; ++a) {
                    fp4_fetch<KW>(x.k[t][a], kp, ok_[a]);
                    x.ks[t][a] = __builtin_amdgcn_raw_buffer_load_b8(ksp, oks[a], 0, 0);
                    x.kvs[t][a] = __builtin_amdgcn_raw_buffer_load_b8(vsp, okv[a], 0, 0);
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if constexpr (VC == 4) x.v[4 * t + r][0] = __builtin_amdgcn_raw_buffer_load_b16(vp, ov[r], 0, 0);
                    else if constexpr (VC == 8) x.v[4 * t + r][0] = __builtin_amdgcn_raw_buffer_load_b32(vp, ov[r], 0, 0);
                    else fp4_fetch<2>(x.v[4 * t + r], vp, ov[r]);
                    x.vs[4 * t + r] = __builtin_amdgcn_raw_buffer_load_b8(vsp, ovs[r], 0, 0);
                }
            }
        } else {
            auto find = [&](int j, uint32_t& page, uint32_t& row) {
                const bool in = j >= sq.first && j < sq.n;
                const int i = fp4_page(p.c, in ? j : 0);
                const int32_t y = in ? table[i] : -1;
                const bool ok = y >= 0 && y < p.c.cache_pages;
                page = ok ? y : 0;
                row = ok ? j - i * p.c.page : 0;
                return ok;
            };
            x.there[0] = x.there[1] = true;
            x.seen = 0;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                uint32_t page, row;
                find(key0 + 16 * t + m, page, row);
                const uint8_t *kp = kc + fp4_at(page, p.c.kp, row, p.c.kt, 0, 0), *ksp = ksc + fp4_at(page, p.c.ksp, row, p.c.kst, 0, 0);
                const uint8_t* vsp = vsc + fp4_at(page, p.c.vsp, row, p.c.vst, 0, 0);
#pragma unroll
                for (int a = 0; a < KB; ++a) {
                    fp4_load<KW>(x.k[t][a], kp + ko[a]);
                    x.ks[t][a] = ksp[kb[a]];
                    x.kvs[t][a] = vsp[kb[a]];
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                uint32_t page, row;
                if (find(key0 + 16 * (i >> 2) + 4 * j4 + (i & 3), page, row)) x.seen |= 1u << i;
                const uint8_t* vp = vc + fp4_at(page, p.c.vp, row, p.c.vt, 0, 0) + vo;
                if constexpr (VC == 4) x.v[i][0] = *reinterpret_cast<const uint16_t*>(vp);
                else if constexpr (VC == 8) x.v[i][0] = *reinterpret_cast<const uint32_t*>(vp);
                else fp4_load<2>(x.v[i], vp);
                x.vs[i] = vsc[fp4_at(page, p.c.vsp, row, p.c.vst, 0, 0) + vb];
            }
        }
    };
    // The first keys are on their way before anything waits for the queries.
    const int step = 32 * NW;
    Fp4Keys<E, DP> x, y;
    const int key_first = s0 + 32 * wave;
    if (key_first < s1) load(x, key_first);

    // This lane's rows and the keys that each sees: [lo, hi].
    int tok[NC], head[NC], lo[NC], hi[NC];
    u32x4 qr[NC][KS][QP];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const int r = c0 + 16 * i + m;
        const bool ok = r < rows;
        tok[i] = ok && p.cu != nullptr ? r / p.G : 0;
        head[i] = hk * p.G + (ok ? r - tok[i] * p.G : 0);
        hi[i] = ok ? sq.n - sq.nq + tok[i] : -1;
        lo[i] = p.window > 0 ? max(0, hi[i] - p.window + 1) : 0;
        const bool neg = arg_scale(p, head[i]) < 0.f;
        const uint8_t* row = (const uint8_t*)p.q + (int64_t)(sq.q0 + tok[i]) * p.q_st + (int64_t)head[i] * p.q_sh;
#pragma unroll
        for (int a = 0; a < KB; ++a)
#pragma unroll
            for (int w = 0; w < KW; ++w)
                fp4_query<E>(row, 8 * KW * (j4 + 4 * a) + 8 * w, p.D, ok, neg, qr[i][a * KW + w]);
    }
    auto use = [&](Fp4Keys<E, DP>& x, int key0) __attribute__((always_inline)) {
        // K, with NaN for the blocks of tokens that are not numbers in K or V.
        f32x4v s[NC][2];
        bool bad = false;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int a = 0; a < KB; ++a) bad = bad || x.ks[t][a] == kFp4Bad || x.kvs[t][a] == kFp4Bad;
        const bool any_bad = __ballot(bad) != 0;
        if (any_bad) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int a = 0; a < KB; ++a)
                    if (x.kvs[t][a] == kFp4Bad) x.ks[t][a] = kFp4Bad;
        }
        if (!whole) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int a = 0; a < KB; ++a) {
                    x.ks[t][a] &= kmask[a];
#pragma unroll
                    for (int w = 0; w < KW; ++w) x.k[t][a][w] &= kmask[a];
                }
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int i = 0; i < NC; ++i) s[i][t] = f32x4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int a = 0; a < KB; ++a) {
                const float sc = fp4_scale(x.ks[t][a]);
#pragma unroll
                for (int w = 0; w < KW; ++w) {
                    const u32x4 k = fp4_eight(x.k[t][a][w], sc);
#pragma unroll
                    for (int i = 0; i < NC; ++i)
#pragma unroll
                        for (int u = 0; u < QP; ++u) s[i][t] = mfma16<BF16>(k, qr[i][a * KW + w][u], s[i][t]);
                }
            }
        }
        // Which of the lane's 8 keys (16 t + 4 j4 + r) are there at all.
        const bool inside = key0 >= sq.first && key0 + 32 <= sq.n;
        uint32_t seen = 255;
        if constexpr (P16) {
            if (!(inside && x.there[0] && x.there[1])) {
                seen = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int key = key0 + 16 * (i >> 2) + 4 * j4 + (i & 3);
                    if (x.there[i >> 2] && key >= sq.first && key < sq.n) seen |= 1u << i;
                }
            }
        } else {
            seen = x.seen;
        }
        const bool cut = __ballot(seen != 255) != 0 || key0 + 31 > all_hi || key0 < all_lo;
        if (cut) {
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                const int key = key0 + 16 * (n >> 2) + 4 * j4 + (n & 3);
#pragma unroll
                for (int i = 0; i < NC; ++i)
                    if (!((seen >> n) & 1) || key > hi[i] || key < lo[i]) s[i][n >> 2][n & 3] = 0.f;
            }
        }
        if (cut || any_bad) {
#pragma unroll
            for (int n = 0; n < 8; ++n)
                if (!((seen >> n) & 1) || x.vs[n] == kFp4Bad) {
                    x.vs[n] = 0;
#pragma unroll
                    for (int d = 0; d < VD; ++d) x.v[n][d] = 0;
                }
        }
        u32x4 wt[NC][PP];
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            float w[8];
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                const float r = s[i][n >> 2][n & 3], a = r < 0.f ? 0.f : r;  // NaN stays
                w[n] = a * a;
                z[i] += w[n];
            }
            if constexpr (WEIGH) {
                if (c0 + 16 * i + m < rows) {
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        const int at = key0 - sq.base() + 16 * t + 4 * j4;
                        f32x4v y = {w[4 * t], w[4 * t + 1], w[4 * t + 2], w[4 * t + 3]};
                        if (cut) {  // keys without a page are marked: a denominator that is not a number is not theirs
#pragma unroll
                            for (int r = 0; r < 4; ++r) y[r] = (seen >> (4 * t + r)) & 1 ? y[r] : -1.f;
                        }
                        if (at < p.raw_ld)  // raw_ld: a multiple of 32
                            *reinterpret_cast<f32x4v*>(p.raw + ((int64_t)b * p.H + head[i]) * p.raw_ld + at) = y;
                    }
                }
            }
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                uint32_t u[PP];
                fp4_parts<PP>(w[2 * n], w[2 * n + 1], u);
#pragma unroll
                for (int k = 0; k < PP; ++k) wt[i][k][n] = u[k];
            }
        }
        // V two columns at a time: the keys' pairs of columns in bf16, regrouped
        // to pairs of keys.
        auto columns = [&](auto pair) __attribute__((always_inline)) {
            constexpr int d = decltype(pair)::value;
            uint32_t y[8];
#pragma unroll
            for (int n = 0; n < 8; ++n) y[n] = fp4_pair<d & 3>(x.v[n][d / 4], fp4_scale(x.vs[n]));
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                u32x4 a;
#pragma unroll
                for (int n = 0; n < 4; ++n) a[n] = __builtin_amdgcn_perm(y[2 * n + 1], y[2 * n], h ? 0x07060302u : 0x05040100u);
#pragma unroll
                for (int i = 0; i < NC; ++i)
#pragma unroll
                    for (int k = 0; k < PP; ++k) acc[i][2 * d + h] = mfma16<BF16>(a, wt[i][k], acc[i][2 * d + h]);
            }
        };
        columns(std::integral_constant<int, 0>{});
        columns(std::integral_constant<int, 1>{});
        if constexpr (VC >= 8) {
            columns(std::integral_constant<int, 2>{});
            columns(std::integral_constant<int, 3>{});
        }
        if constexpr (VC >= 16) {
            columns(std::integral_constant<int, 4>{});
            columns(std::integral_constant<int, 5>{});
            columns(std::integral_constant<int, 6>{});
            columns(std::integral_constant<int, 7>{});
        }
    };
    for (int key = key_first; key < s1; key += 2 * step) {
        if (key + step < s1) load(y, key + step);
        use(x, key);
        if (key + step >= s1) break;
        if (key + 2 * step < s1) load(x, key + 2 * step);
        use(y, key + step);
    }
    // The waves' sums, in order.
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        float zz = z[i];
        zz += __shfl_xor(zz, 16);
        zz += __shfl_xor(zz, 32);
        if (i > 0) __syncthreads();
        if (j4 == 0) zred[wave][m] = zz;
#pragma unroll
        for (int e = 0; e < VC; ++e)
#pragma unroll
            for (int r = 0; r < 4; ++r) red[wave][m][VC * (4 * j4 + r) + e] = acc[i][e][r];
        __syncthreads();
        const int here = min(16, rows - c0 - 16 * i);
        for (int x = threadIdx.x; x < here * (DP / 4); x += 64 * NW) {
            const int cc = x / (DP / 4), col = 4 * (x % (DP / 4));
            if (col >= p.D) continue;
            f32x4v y = *reinterpret_cast<const f32x4v*>(&red[0][cc][col]);
            float sum = zred[0][cc];
#pragma unroll
            for (int w = 1; w < NW; ++w) {
                y += *reinterpret_cast<const f32x4v*>(&red[w][cc][col]);
                sum += zred[w][cc];
            }
            const int r = c0 + 16 * i + cc, t = p.cu != nullptr ? r / p.G : 0, h = hk * p.G + r - t * p.G;
            if ((nsplit > 1 || WEIGH) && unit < p.units) {  // more only where starts do not ascend
                float* to = p.part + (((int64_t)unit * p.Hkv + hk) * (16 * NC) + 16 * i + cc) * (p.D + 4);
                *reinterpret_cast<f32x4v*>(to + 4 + col) = y;
                if (col == 0) to[0] = sum;
            }
            if (nsplit == 1) {
                y *= fp4_inverse(p, h, sum);
                fp4_store4<E>((uint8_t*)p.out + ((int64_t)(sq.q0 + t) * p.H + h) * p.D * IT, col, y);
            }
        }
    }
}

template <class E, int DP, int NC, bool WEIGH, bool P16>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(fp4_wpe<E>(DP, NC))))
void born_fp4_paged_kernel(Fp4PagedArgs p) {
    __shared__ __attribute__((aligned(16))) uint8_t smem[kFp4NarrowLds<DP>];
    const int unit = blockIdx.z * gridDim.y + blockIdx.y;
    if (blockIdx.x == 0) fp4_behind<E>(p, unit, gridDim.y * gridDim.z);
    if (unit < p.units) fp4_narrow<E, DP, NC, WEIGH, P16>(p, Fp4Share(p, false), smem, unit, blockIdx.x);
}

// A narrow row's partial sums.
struct Fp4Parts {
    const float* at;
    int64_t ld;
    int n;
    __device__ __forceinline__ Fp4Parts(const Fp4PagedArgs& p, const Fp4Seq& sq, int b, int hk, int r) {
        const int2 plan = p.plan[b];
        const int cb = r / p.cols;
        // In bounds also where starts do not ascend, and not all units had room.
        const int columns = sq.columns(p);
        n = plan.x >= 0 && plan.y > 0 && (int64_t)plan.x + (int64_t)plan.y * columns <= p.units ? plan.y : 0;
        ld = (int64_t)columns * p.Hkv * p.cols * (p.D + 4);
        at = p.part + (((int64_t)(plan.x + cb) * p.Hkv + hk) * p.cols + r - cb * p.cols) * (p.D + 4);
    }
};

// Splits joined in order.  A row's columns take `ncol` threads, its splits
// `groups` of them, 256 / (ncol groups) rows a workgroup.
// WEIGH: in the same launch, for each (sequence, key head), 256 keys at a time, the
// sum over the group of p_j / Z, the heads in order, is added to its weights; by a
// workgroup once (1), or again and again (2).
template <class E, int WEIGH>
__global__ __launch_bounds__(256) void born_fp4_join_kernel(Fp4PagedArgs p, Fp4Join q) {
    __shared__ f32x4v red[256];
    __shared__ float zred[256];
    if (WEIGH != 0 && (int)blockIdx.x >= q.blocks) {
        const int x = blockIdx.x - q.blocks, hk = x % p.Hkv, b = x / p.Hkv % p.B;
        const Fp4Seq sq(p, b);
        const int start = sq.base() + x / p.Hkv / p.B * 256, end = min(sq.n, p.w_len);
        if (start >= end) return;
        const bool once = WEIGH == 1;
        float* const weight = p.weights + (int64_t)b * p.w_sb + (int64_t)hk * p.w_sh;
        auto raw = [&](int g, int j) __attribute__((always_inline)) {
            return p.raw[((int64_t)b * p.H + hk * p.G + g) * p.raw_ld + (j - sq.base())];
        };
        auto seen = [&](int j) __attribute__((always_inline)) { return j >= sq.first && j < end; };
        auto add = [&](float& sum, float w, float inverse) __attribute__((always_inline)) {
            const float y = fmaf(w, inverse, sum);
            sum = w < 0.f ? sum : y;  // no page
        };
        // On their way before the denominators are known (16 caches of 52 thousand
        // keys, 4 key heads D64, 4 heads each: 22.4 us, after them 23.3).
        constexpr int kFirst = 4;
        float first[kFirst] = {}, old = 0.f, sum = 0.f;
        if (once && seen(start + threadIdx.x)) {
            old = weight[start + threadIdx.x];
#pragma unroll
            for (int i = 0; i < kFirst; ++i)
                if (i < p.G) first[i] = raw(i, start + threadIdx.x);
        }
        for (int g0 = 0; g0 < p.G; g0 += 256) {
            const int gn = min(256, p.G - g0);
            if ((int)threadIdx.x < gn) {
                const Fp4Parts part(p, sq, b, hk, g0 + threadIdx.x);
                float z = 0.f;
#pragma unroll 8
                for (int i = 0; i < part.n; ++i) z += part.at[i * part.ld];
                zred[threadIdx.x] = fp4_inverse(p, hk * p.G + g0 + threadIdx.x, z);
            }
            __syncthreads();
            if (once) {
                if (seen(start + threadIdx.x)) {
                    if (g0 == 0) {
#pragma unroll
                        for (int i = 0; i < kFirst; ++i)
                            if (i < gn) add(sum, first[i], zred[i]);
                    }
#pragma unroll 4
                    for (int i = g0 == 0 ? kFirst : 0; i < gn; ++i) add(sum, raw(g0 + i, start + threadIdx.x), zred[i]);
                }
            } else {
                for (int j = start + threadIdx.x; j < end; j += q.weigh * 256) {
                    if (!seen(j)) continue;
                    float more = 0.f;
#pragma unroll 4
                    for (int i = 0; i < gn; ++i) add(more, raw(g0 + i, j), zred[i]);
                    weight[j] += more;
                }
            }
            __syncthreads();
        }
        if (once && seen(start + threadIdx.x)) weight[start + threadIdx.x] = old + sum;
        return;
    }
    const int per = q.ncol * q.groups, mine = threadIdx.x / per, col = 4 * (threadIdx.x % q.ncol), group = threadIdx.x % per / q.ncol;
    const int unit = blockIdx.x * (256 / per) + mine;
    const float* from = nullptr;
    int64_t ld = 0, row = 0;  // row: token and head
    int n = 0, head = 0;
    if (unit < q.narrow + q.rows) {
        int b, hk, r;
        Fp4Seq sq(p, 0);
        if (unit < q.narrow) {
            const int rest = unit / q.most;
            r = unit - rest * q.most;
            b = rest / p.Hkv;
            hk = rest - b * p.Hkv;
            sq = Fp4Seq(p, b);
        } else {
            const int at = unit - q.narrow, t = at / p.H, h = at - t * p.H;
            b = t;
            if (p.cu != nullptr) {
                int hi = p.B;  // the last start at or before t
                b = 0;
                while (hi - b > 1) {
                    const int mid = (b + hi) / 2;
                    if (p.cu[mid] <= t) b = mid;
                    else hi = mid;
                }
            }
            sq = Fp4Seq(p, b);
            hk = h / p.G;
            r = t >= sq.q0 ? (t - sq.q0) * p.G + h - hk * p.G : INT_MAX;
        }
        if (r < sq.nq * p.G) {
            const int t = r / p.G;
            head = hk * p.G + r - t * p.G;
            row = (int64_t)(sq.q0 + t) * p.H + head;
            if (sq.wide(p)) {
                if (unit >= q.narrow) from = p.wide_part + row * p.splits * (p.D + 4), ld = p.D + 4, n = p.splits;
            } else if (unit < q.narrow || p.slots == 0) {
                const Fp4Parts part(p, sq, b, hk, r);
                if (part.n > 1) from = part.at, ld = part.ld, n = part.n;  // one: written already
            }
        }
    }
    const bool ok = col < p.D;
    f32x4v x = {0.f, 0.f, 0.f, 0.f};
    float z = 0.f;
#pragma unroll 8
    for (int i = group; i < n; i += q.groups) {
        const float* at = from + i * ld;
        z += at[0];
        if (ok) x += *reinterpret_cast<const f32x4v*>(at + 4 + col);
    }
    if (q.groups > 1) {
        red[threadIdx.x] = x;
        zred[threadIdx.x] = z;
        __syncthreads();
        if (group != 0) return;
        for (int i = 1; i < q.groups; ++i) {
            x += red[threadIdx.x + i * q.ncol];
            z += zred[threadIdx.x + i * q.ncol];
        }
    }
    if (n == 0 || !ok) return;
    x *= fp4_inverse(p, head, z);
    fp4_store4<E>((uint8_t*)p.out + row * p.D * kItem<E>, col, x);
}

template <class E>
hipError_t fp4_paged_fwd(const Fp4PagedArgs& a, const Fp4Plan& plan, hipStream_t st);

template <class E, int NC, bool WEIGH, bool P16>
void launch_fp4_dp(const Fp4PagedArgs& a, const Fp4Plan& plan, hipStream_t st) {
    // A grid's second and third dimensions hold 65535.
    const int64_t z = (plan.units + 65534) / 65535, y = (plan.units + z - 1) / z;
    const dim3 grid((unsigned)a.Hkv, (unsigned)y, (unsigned)z);
    if (a.D <= 64) hipLaunchKernelGGL((born_fp4_paged_kernel<E, 64, NC, WEIGH, P16>), grid, dim3(256), 0, st, a);
    else if (a.D <= 128) hipLaunchKernelGGL((born_fp4_paged_kernel<E, 128, NC, WEIGH, P16>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((born_fp4_paged_kernel<E, 256, NC, WEIGH, P16>), grid, dim3(256), 0, st, a);
}
template <class E, bool P16>
void launch_fp4_nc(const Fp4PagedArgs& a, const Fp4Plan& plan, hipStream_t st) {
    if (a.raw != nullptr) launch_fp4_dp<E, 1, true, P16>(a, plan, st);
    else if (plan.nc == 1) launch_fp4_dp<E, 1, false, P16>(a, plan, st);
    else launch_fp4_dp<E, 2, false, P16>(a, plan, st);
}

// Rows' offsets within a page in 31 bits.
inline bool fp4_p16(const Fp4Cache& c) {
    const int64_t far = (int64_t)1 << 31, page = c.page;
    return c.page % 16 == 0 && page * c.kt < far && page * c.vt < far && page * c.kst < far && page * c.vst < far;
}

template <class E>
hipError_t launch_fp4_join(const Fp4PagedArgs& a, const Fp4Plan& plan, hipStream_t st) {
    const Fp4Join& q = plan.join;
    if (a.raw != nullptr) {
        const dim3 grid((unsigned)(q.blocks + (int64_t)q.weigh * a.B * a.Hkv));
        if ((int64_t)q.weigh * 256 >= a.raw_ld) hipLaunchKernelGGL((born_fp4_join_kernel<E, 1>), grid, dim3(256), 0, st, a, q);
        else hipLaunchKernelGGL((born_fp4_join_kernel<E, 2>), grid, dim3(256), 0, st, a, q);
    } else if (q.blocks > 0) {
        hipLaunchKernelGGL((born_fp4_join_kernel<E, 0>), dim3(q.blocks), dim3(256), 0, st, a, q);
    }
    return hipGetLastError();
}

}  // namespace qdl
