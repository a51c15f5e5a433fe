// The paged key-value cache: appending a step's keys and values, with the
// rotation and normalisation of its queries and keys, and evicting the keys
// that the accumulated attention weighs least.
#pragma once

#include <type_traits>

#include "born_common.h"
#include "born_packed.h"

namespace qdl {

// ---------------------------------------------------------------------------
// Append.  A row (one head of one token) belongs to a group of `lpr` lanes, a
// power of two; lane i of it owns VEC columns of the first half and the
// matching ones of the second, both members of its rotation pairs:
//   y1 = x1 c - x2 s, y2 = x1 s + x2 c, out = y / sqrt(sum y^2 + eps),
// in fp32 from the 16-bit inputs on, rounded once.  Bound by memory: rows read
// and written once.  A group takes ROWS rows of one token, so that the token's
// angles are read once for them; single tokens take one row each (ROWS = 1),
// where lanes and not bytes are short.  16384 tokens, 32 heads over 8, D128: 403
// MB in 81 us (5.0 TB/s); 64 single tokens, 16 heads over 4: 5.5 us.
// ---------------------------------------------------------------------------
struct AppendArgs {
    const void *q, *k, *v;
    void *q_out, *k_cache, *v_cache;
    const float *cos, *sin;
    const int32_t* positions;  // (N) rows of the tables, or nullptr: the slot
    const int32_t* table;
    const int32_t* lens;       // (B), the appended tokens included
    const int32_t* cu;         // B + 1 starts, or nullptr: one token per sequence
    int N, B, H, Hkv, D;
    int pages, page, page_shift;
    int64_t table_ld, cache_pages;
    int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh, kp, kt, kh, vp, vt, vh;  // bytes
    int table_rows, n_freq;
    int64_t freq_ld;
    float eps;
    int lpr;
};

template <class E, int VEC>
struct RowVec {
    static constexpr int W = VEC * kItem<E> / 4;  // dwords
    uint32_t u[W];
    __device__ __forceinline__ void load(const uint8_t* p) {
        if constexpr (W == 4) {
            const u32x4 x = ldg16(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) u[i] = x[i];
        } else {
            const u32x2 x = *reinterpret_cast<const u32x2*>(p);
            u[0] = x[0];
            u[1] = x[1];
        }
    }
    __device__ __forceinline__ void store(uint8_t* p) const {
        if constexpr (W == 4) {
            const u32x4 x = {u[0], u[1], u[2], u[3]};
            *reinterpret_cast<u32x4*>(p) = x;
        } else {
            const u32x2 x = {u[0], u[1]};
            *reinterpret_cast<u32x2*>(p) = x;
        }
    }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (std::is_same<E, F32>::value) return __uint_as_float(u[i]);
        else return (i & 1) ? E::hi(u[i >> 1]) : E::lo(u[i >> 1]);
    }
    __device__ __forceinline__ void set(const float (&x)[VEC]) {
        if constexpr (std::is_same<E, F32>::value) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) u[i] = __float_as_uint(x[i]);
        } else {
#pragma unroll
            for (int i = 0; i < VEC / 2; ++i) u[i] = E::pack(x[2 * i], x[2 * i + 1]);
        }
    }
};

template <class E, int VEC, int ROWS>
__global__ __launch_bounds__(256) void born_append_kernel(AppendArgs p) {
    const int all = p.H + 2 * p.Hkv, groups = (all + ROWS - 1) / ROWS;
    const int64_t item = (int64_t)blockIdx.x * (256 / p.lpr) + threadIdx.x / p.lpr;
    const int lane = threadIdx.x & (p.lpr - 1);
    if (item >= (int64_t)p.N * groups) return;
    const int t = (int)(item / groups), r0 = (int)(item % groups) * ROWS;
    const int half = p.D >> 1;
    const bool own = lane * VEC < half;  // lanes of a group past the row's chunks
    const int o1 = lane * VEC * kItem<E>, o2 = o1 + half * kItem<E>;

    // The token's sequence, slot and row of the cache.
    int s = t, first = t, last = t + 1;
    bool in = t < p.B;
    if (p.cu != nullptr) {
        int lo = 0, hi = p.B;  // the last start at or before t
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (p.cu[mid] <= t) lo = mid;
            else hi = mid;
        }
        s = lo;
        in = p.B > 0;
        if (in) {
            first = max(p.cu[s], 0);
            last = p.cu[s + 1];
            in = t >= first && t < last;
        }
    }
    int64_t slot = -1, page = -1;
    int row = 0;
    if (in) {
        slot = (int64_t)p.lens[s] - (last - t);
        if (slot >= 0 && slot < (int64_t)p.pages * p.page) {
            const int i = p.page_shift >= 0 ? (int)slot >> p.page_shift : (int)slot / p.page;
            row = (int)slot - i * p.page;
            page = p.table[(int64_t)s * p.table_ld + i];
        }
    }
    const bool kept = page >= 0 && page < p.cache_pages;

    float c[VEC], sn[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) c[i] = 1.f, sn[i] = 0.f;
    if (p.cos != nullptr && own && r0 < p.H + p.Hkv) {
        int64_t at = p.positions != nullptr ? p.positions[t] : slot;
        at = min(max(at, (int64_t)0), (int64_t)p.table_rows - 1) * p.freq_ld;  // rows past the tables: their last
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const int f = lane * VEC + i;
            if (f < p.n_freq) c[i] = p.cos[at + f], sn[i] = p.sin[at + f];
        }
    }
    RowVec<E, VEC> x1[ROWS], x2[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int r = r0 + i;
        if (r >= all || !own) continue;
        const uint8_t* src = r < p.H          ? (const uint8_t*)p.q + (int64_t)t * p.q_st + (int64_t)r * p.q_sh
                             : r < p.H + p.Hkv ? (const uint8_t*)p.k + (int64_t)t * p.k_st + (int64_t)(r - p.H) * p.k_sh
                                               : (const uint8_t*)p.v + (int64_t)t * p.v_st + (int64_t)(r - p.H - p.Hkv) * p.v_sh;
        x1[i].load(src + o1);
        x2[i].load(src + o2);
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int r = r0 + i;
        if (r >= all) continue;  // uniform in the group
        if (r >= p.H + p.Hkv) {
            if (kept && own) {
                uint8_t* to = (uint8_t*)p.v_cache + page * p.vp + (int64_t)row * p.vt + (int64_t)(r - p.H - p.Hkv) * p.vh;
                x1[i].store(to + o1);
                x2[i].store(to + o2);
            }
            continue;
        }
        float y1[VEC], y2[VEC], ss = 0.f;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float a = own ? x1[i].get(e) : 0.f, b = own ? x2[i].get(e) : 0.f;
            y1[e] = a * c[e] - b * sn[e];
            y2[e] = a * sn[e] + b * c[e];
            ss = fmaf(y1[e], y1[e], fmaf(y2[e], y2[e], ss));
        }
        for (int o = 1; o < p.lpr; o <<= 1) ss += __shfl_xor(ss, o);
        float f = 1.0f / sqrtf(ss + p.eps);
        uint8_t* to;
        bool write = own;
        if (r < p.H) {
            to = (uint8_t*)p.q_out + ((int64_t)t * p.H + r) * p.D * kItem<E>;
        } else {
            to = (uint8_t*)p.k_cache + page * p.kp + (int64_t)row * p.kt + (int64_t)(r - p.H) * p.kh;
            write = write && kept;
        }
        if (!write) continue;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            // A token of no sequence has a zero query.
            y1[e] = in ? y1[e] * f : 0.f;
            y2[e] = in ? y2[e] * f : 0.f;
        }
        x1[i].set(y1);
        x2[i].set(y2);
        x1[i].store(to + o1);
        x2[i].store(to + o2);
    }
}

// ---------------------------------------------------------------------------
// Evict.  Two launches: the selection, one workgroup for a (sequence, key
// head), and the move of the kept rows.
//
// Selection: the `want` greatest weights among the keys before the recent
// ones, ties to the lowest index: a radix selection over the order-preserving
// 32-bit forms of the weights, four histograms of 8 bits, then one pass that
// counts the kept ones before each key.  A thread holds up to 16 weights, so up
// to 16384 keys are read once.  The weights are compared, never rounded.
// ---------------------------------------------------------------------------
struct EvictArgs {
    void *k, *v;
    const int32_t *table, *to;  // (B, pages), (B, to_pages)
    const int32_t* lens;
    const float* weight;
    float* weight_out;          // (B, Hkv, w_len)
    int32_t *lens_out, *kept;   // (B), (B, Hkv, budget)
    int B, Hkv, D, item;
    int pages, to_pages, page, page_shift;
    int64_t table_ld, to_ld, cache_pages;
    int64_t kp, kt, kh, vp, vt, vh;  // bytes
    int64_t w_sb, w_sh;              // elements
    int w_len, budget, recent;
};

__device__ __forceinline__ int evict_len(const EvictArgs& p, int b) {
    return (int)min((int64_t)max(p.lens[b], 0), (int64_t)p.pages * p.page);
}

// Unsigned order of floats; every NaN above all numbers, -0 equal to 0.
__device__ __forceinline__ uint32_t evict_key(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// 1024 threads with PER weights each: what the launch waits for is the
// instructions of one wave, so the caches' capacity picks the fewest that hold a
// row at once (4 rows of 2048 weights 6.8 us with 2 each, 128 rows of up to
// 10000 18.7 us with 16).  The whole call to a budget of 64, us with 2, 4, 8 and
// 16 each, 128 rows of 2048: 17.0, 17.2, 19.8, 24.0; of 4096: 20.0, 17.9, 20.1,
// 24.2; of 8192: 27.0, 25.3, 21.9, 26.2; of 16384: 39.6, 36.6, 36.7, 29.2.
constexpr int kEvictThreads = 1024, kEvictMost = 16;

template <int PER>
__global__ __launch_bounds__(kEvictThreads) void born_evict_select_kernel(EvictArgs p) {
    constexpr int NT = kEvictThreads, NW = NT / 64, SPAN = NT * PER, COPIES = 4;
    constexpr int CL = (PER * NW + 63) / 64;  // counts that a lane of one wave scans
    constexpr uint32_t kZero = 0x80000000u;   // the key of 0
    // Weights lie close together: four copies of each bin, one for every fourth lane.
    __shared__ __attribute__((aligned(16))) uint32_t hist[256 * COPIES];
    __shared__ uint32_t s_prefix, s_left, s_all;
    __shared__ uint32_t counts[64 * CL];  // kept for sure | ties << 16, per 64 keys
    __shared__ uint32_t s_total, s_zeros;
    const int hk = blockIdx.x % p.Hkv, b = blockIdx.x / p.Hkv;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n = evict_len(p, b), m = min(n, p.budget);
    const float* w = p.weight + (int64_t)b * p.w_sb + (int64_t)hk * p.w_sh;
    float* wo = p.weight_out + ((int64_t)b * p.Hkv + hk) * p.w_len;
    int32_t* kept = p.kept + ((int64_t)b * p.Hkv + hk) * p.budget;
    const int tail = n > m ? min(p.recent, m) : m;
    const int old = n - tail, want = m - tail;  // of the `old` first keys, `want` stay

    const int spans = (old + SPAN - 1) / SPAN;
    float x[PER];
    uint32_t key[PER];  // 0, below every number's, where there is no key
    auto load = [&](int span) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int j = span * SPAN + i * NT + tid;
            x[i] = j < old && j < p.w_len ? w[j] : 0.f;
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) key[i] = span * SPAN + i * NT + tid < old ? evict_key(x[i]) : 0u;
    };
    if (want > 0) load(0);
    if (hk == 0 && tid == 0) p.lens_out[b] = m;
    for (int i = m + tid; i < p.budget; i += NT) kept[i] = -1;
    for (int i = m + tid; i < p.w_len; i += NT) wo[i] = 0.f;
    for (int i = tid; i < tail; i += NT) {
        kept[want + i] = old + i;
        if (want + i < p.w_len) wo[want + i] = old + i < p.w_len ? w[old + i] : 0.f;
    }
    if (want == 0) return;

    if (tid == 0) s_prefix = 0, s_left = want, s_all = 0, s_zeros = 0;
    hist[tid] = 0;
    for (int i = tid; i < 64 * CL; i += NT) counts[i] = 0;
    __syncthreads();
    // The want-th greatest key, 8 bits at a time.  Keys that were never weighed
    // would all meet in one bin: they are counted by wave, in the first round.
    for (int shift = 24; shift >= 0; shift -= 8) {
        const uint32_t prefix = s_prefix, mask = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
        uint32_t zeros = 0;
        for (int sp = 0; sp < spans; ++sp) {
            if (spans > 1) load(sp);
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                if (shift == 24) zeros += (uint32_t)__popcll(__ballot(key[i] == kZero));
                if (key[i] != 0 && key[i] != kZero && (key[i] & mask) == prefix)
                    atomicAdd(&hist[((key[i] >> shift) & 255u) * COPIES + (lane & (COPIES - 1))], 1u);
            }
        }
        if (shift == 24 && lane == 0) atomicAdd(&s_zeros, zeros);
        __syncthreads();
        if (wave == 0) {
            // Lane l: bins 255 - 4 l .. 252 - 4 l, from the greatest down.
            uint32_t c[4], sum = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t bin = 255 - 4 * lane - i;
                const u32x4 h = *reinterpret_cast<const u32x4*>(&hist[bin * COPIES]);
                c[i] = h[0] + h[1] + h[2] + h[3];
                if ((kZero & mask) == prefix && ((kZero >> shift) & 255u) == bin) c[i] += s_zeros;
                sum += c[i];
            }
            uint32_t above = sum;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const uint32_t y = __shfl_up(above, o);
                if (lane >= o) above += y;
            }
            above -= sum;
            const uint32_t left = s_left;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (above < left && left <= above + c[i]) {
                    s_prefix = prefix | ((uint32_t)(255 - 4 * lane - i) << shift);
                    s_left = left - above;
                    s_all = left == above + c[i];  // the whole bin stays: nothing left to find
                }
                above += c[i];
            }
        }
        __syncthreads();
        if (s_all) break;
        hist[tid] = 0;
        __syncthreads();
    }
    // Keys above the cut stay, and the first `ties` equal to it.
    const uint32_t cut = s_all ? s_prefix - 1 : s_prefix, ties = s_all ? 0u : s_left;

    uint32_t before_gt = 0, before_eq = 0;
    for (int sp = 0; sp < spans; ++sp) {
        if (spans > 1) load(sp);
        uint64_t gt[PER], eq[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            gt[i] = __ballot(key[i] > cut);
            eq[i] = __ballot(key[i] == cut);
            if (lane == 0) counts[i * NW + wave] = (uint32_t)__popcll(gt[i]) | ((uint32_t)__popcll(eq[i]) << 16);
        }
        __syncthreads();
        if (wave == 0) {  // exclusive sums (up to 16384, which fits 16 bits)
            uint32_t c[CL], sum = 0;
#pragma unroll
            for (int i = 0; i < CL; ++i) c[i] = counts[CL * lane + i], sum += c[i];
            uint32_t run = sum;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const uint32_t y = __shfl_up(run, o);
                if (lane >= o) run += y;
            }
            if (lane == 63) s_total = run;
            run -= sum;
#pragma unroll
            for (int i = 0; i < CL; ++i) {
                counts[CL * lane + i] = run;
                run += c[i];
            }
        }
        __syncthreads();
        const uint64_t below = (1ull << lane) - 1;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const uint32_t c = counts[i * NW + wave];
            const uint32_t g = before_gt + (c & 0xffffu) + (uint32_t)__popcll(gt[i] & below);
            const uint32_t e = before_eq + (c >> 16) + (uint32_t)__popcll(eq[i] & below);
            if (key[i] > cut || (key[i] == cut && e < ties)) {
                const int to = (int)(g + min(e, ties));
                kept[to] = sp * SPAN + i * NT + tid;
                if (to < p.w_len) wo[to] = x[i];
            }
        }
        if (spans == 1) break;
        before_gt += s_total & 0xffffu;
        before_eq += s_total >> 16;
        __syncthreads();
    }
}

inline void launch_evict_select(const EvictArgs& a, unsigned units, int64_t room, hipStream_t st) {
    const dim3 grid(units), block(kEvictThreads);
    if (room <= 2 * kEvictThreads) hipLaunchKernelGGL((born_evict_select_kernel<2>), grid, block, 0, st, a);
    else if (room <= 4 * kEvictThreads) hipLaunchKernelGGL((born_evict_select_kernel<4>), grid, block, 0, st, a);
    else if (room <= 8 * kEvictThreads) hipLaunchKernelGGL((born_evict_select_kernel<8>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((born_evict_select_kernel<kEvictMost>), grid, block, 0, st, a);
}

__device__ __forceinline__ int64_t evict_at(const EvictArgs& p, const int32_t* table, int pages, int j, int64_t sp, int64_t st) {
    const int i = p.page_shift >= 0 ? j >> p.page_shift : j / p.page;
    const int64_t page = i < pages ? table[i] : -1;
    return page >= 0 && page < p.cache_pages ? page * sp + (int64_t)(j - i * p.page) * st : -1;
}

// The kept rows to other pages: 16 bytes a lane, K and V of four rows in flight
// for each.  A row whose page is missing arrives as zeros.  Bound by memory: 537
// MB in 118 us (4.5 TB/s; 16 caches cut to 4096 tokens, 8 key heads D128).
constexpr int kEvictUnroll = 4;
inline __host__ __device__ int evict_rows(int cpr) { return 256 / cpr * kEvictUnroll; }  // per workgroup

template <int>
__global__ __launch_bounds__(256) void born_evict_move_kernel(EvictArgs p) {
    const int hk = blockIdx.x % p.Hkv, rest = blockIdx.x / p.Hkv;
    const int b = rest % p.B, tile = rest / p.B;
    const int m = min(evict_len(p, b), p.budget);
    const int cpr = p.D * p.item / 16, rows = 256 / cpr;
    const int32_t* kept = p.kept + ((int64_t)b * p.Hkv + hk) * p.budget;
    const int32_t *from = p.table + (int64_t)b * p.table_ld, *to = p.to + (int64_t)b * p.to_ld;
    const int mine = threadIdx.x / cpr, o = 16 * (threadIdx.x % cpr);
    const int i0 = tile * evict_rows(cpr) + mine;
    if (mine >= rows || i0 >= m) return;
    uint8_t *kc = (uint8_t*)p.k + (int64_t)hk * p.kh + o, *vc = (uint8_t*)p.v + (int64_t)hk * p.vh + o;
    int j[kEvictUnroll];
#pragma unroll
    for (int u = 0; u < kEvictUnroll; ++u) j[u] = i0 + u * rows < m ? kept[i0 + u * rows] : -1;
    // Page and row of the row's old and new slots; page -1: none.
    int pf[kEvictUnroll], rf[kEvictUnroll], pt[kEvictUnroll], rt[kEvictUnroll];
#pragma unroll
    for (int u = 0; u < kEvictUnroll; ++u) {
        const int i = i0 + u * rows, jj = max(j[u], 0);
        const int a = p.page_shift >= 0 ? jj >> p.page_shift : jj / p.page;
        const int d = p.page_shift >= 0 ? i >> p.page_shift : i / p.page;
        rf[u] = jj - a * p.page;
        rt[u] = i - d * p.page;
        pf[u] = j[u] >= 0 && a < p.pages ? from[a] : -1;
        pt[u] = j[u] >= 0 && d < p.to_pages ? to[d] : -1;
    }
    u32x4 y[kEvictUnroll][2];
#pragma unroll
    for (int u = 0; u < kEvictUnroll; ++u) {
        y[u][0] = y[u][1] = u32x4{0u, 0u, 0u, 0u};
        if (pf[u] >= 0 && pf[u] < p.cache_pages) {
            y[u][0] = ldg16(kc + pf[u] * p.kp + rf[u] * p.kt);
            y[u][1] = ldg16(vc + pf[u] * p.vp + rf[u] * p.vt);
        }
    }
#pragma unroll
    for (int u = 0; u < kEvictUnroll; ++u)
        if (pt[u] >= 0 && pt[u] < p.cache_pages) {
            *reinterpret_cast<u32x4*>(kc + pt[u] * p.kp + rt[u] * p.kt) = y[u][0];
            *reinterpret_cast<u32x4*>(vc + pt[u] * p.vp + rt[u] * p.vt) = y[u][1];
        }
}

// The kept rows to the front of their own pages.  Rows only move down and keep
// their order, so one workgroup per (sequence, key head, K or V) walks them
// upwards: a batch is read whole before any of it is written, and what it
// writes lies below every row still to be read.  Bound by that walk where there
// are few of them: the call in place and to other pages, us: one cache of 16384
// halved, 8 key heads D128 189 and 38; 16 cut to 4096, 193 and 143; 64 of 2048
// halved, 4 key heads D64, 50 and 49.
template <int>
__global__ __launch_bounds__(1024) void born_evict_compact_kernel(EvictArgs p) {
    constexpr int U = 4;
    const int which = blockIdx.x & 1, hk = (blockIdx.x >> 1) % p.Hkv, b = (blockIdx.x >> 1) / p.Hkv;
    const int m = min(evict_len(p, b), p.budget);
    const int cpr = p.D * p.item / 16, rows = 1024 / cpr;  // whole rows per round of the workgroup
    const int32_t* kept = p.kept + ((int64_t)b * p.Hkv + hk) * p.budget;
    const int32_t* table = p.table + (int64_t)b * p.table_ld;
    const int mine = threadIdx.x / cpr, o = 16 * (threadIdx.x % cpr);
    uint8_t* cache = (uint8_t*)(which ? p.v : p.k) + (int64_t)hk * (which ? p.vh : p.kh) + o;
    const int64_t sp = which ? p.vp : p.kp, st = which ? p.vt : p.kt;
    for (int i0 = 0; i0 < m; i0 += U * rows) {
        u32x4 y[U];
        int64_t d[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * rows + mine;
            d[u] = -1;
            y[u] = u32x4{0u, 0u, 0u, 0u};
            if (mine < rows && i < m) {
                const int j = kept[i];
                if (j != i) {
                    d[u] = evict_at(p, table, p.pages, i, sp, st);
                    const int64_t a = evict_at(p, table, p.pages, j, sp, st);
                    if (a >= 0) y[u] = ldg16(cache + a);
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (d[u] >= 0) *reinterpret_cast<u32x4*>(cache + d[u]) = y[u];
        __syncthreads();
    }
}

}  // namespace qdl
