// How attention over the 4-bit cache is shared out: the host sizes launches and
// workspaces from what it knows, the device shares out what is there by the same
// rules.  Apart from the kernels, so that a host compiler takes it.
#pragma once

#include <cstdint>

namespace qdl {

constexpr int kFp4Rows = 128;  // rows (new tokens x heads of a group) of the tiled kernel's workgroups
// Rows of a (sequence, key head) up to which the narrow kernel takes it.  us with
// 32 and with 64: 32 sequences of 16 tokens over 4096 keys at most, 8 key heads
// D128, 4 heads each, 64 and 74; 4 of 64 over 8000, 4 key heads, 45 and 47; few
// rows the same.
constexpr int kFp4Narrow = 32;
// A launch of few rows goes to the narrow kernel whole, if it does not lose much
// where one sequence has all of them: every 32 rows go through the keys again, so
// rows times keys times key heads decide, whatever the number of sequences, which
// may hold empty ones.  us narrow and tiled, one sequence with all rows, D128: 512
// rows over 2000 keys of 8 heads (2^23.1) 31 and 36, over 8000 of 2 (2^23) 30 and
// 40, over 30000 of one (2^23.9) 48 and 42, over 8000 of 8 (2^25) 60 and 50, over
// 30000 of 8 161 and 105; 128 over 30000 of 8 (2^24.9) 58 and 52.  What it is for:
// 16 sequences of 5 tokens, 4 heads over 4 key heads, 27 and 30, of 8 27 and 34.
// Beyond 512 rows it is even: one sequence of 1024 rows over 1500 keys of 8 heads 45
// and 41, 32 of 8 tokens over 1000 keys of 8 heads 30 and 36.
constexpr int kFp4AllNarrow = 512;
constexpr int64_t kFp4AllWork = (int64_t)1 << 24;
// Workgroups of the narrow kernel that a launch's chunks of keys are made for: two
// rounds of as many as a compute unit holds of bf16 at D128, three with one column
// set, two with two (one column set of fp16 or fp32 there: two).  us with 512, 768, 1024, 1536, 2048: 32 single tokens over long caches 76, 72, 74,
// 65, 67; 16 sequences of 5 tokens (two column sets, before chunks of few keys were
// made fewer) 49, 51, 50, 55, 59.
constexpr int fp4_wanted(int nc) { return nc == 1 ? 1536 : 1024; }
// Narrow and wide sequences have a launch each where the keys that the tables have
// room for (the host knows no lengths), times key heads, are this many and the
// sequences' rows in the mean fit a narrow workgroup: most are narrow then, and
// their own launch has three workgroups a compute unit for two.
// us apart and together, 8 key heads D128, 4 heads each: 64 sequences of 4 tokens
// over 8192 keys at most 67 and 104; where a few are wide it costs, 31 single
// tokens beside one of 200 94 and 86, of 512 (mean 68: together) 158 and 127.
constexpr int64_t kFp4Apart = (int64_t)1 << 20;
// Workgroups that add the keys' weights up, 256 keys at a time each, at most: the
// host knows the table's room only, and more of them find no keys.  us with 2^12,
// 2^14 and any number of them: 64 sequences of 1000 keys, 8 key heads, 32 heads,
// tables of 131072 keys 37, 44, 191; of 16000 keys, tables of 16384, 325, 344, 351.
constexpr int64_t kFp4Weigh = (int64_t)1 << 12;
// Sequences that a workgroup looks through to share out the keys, which takes every
// wave two reads of all lengths.  us so and with a chunk a sequence, one token each,
// 16 heads over 4: 512 sequences of 1000 keys 81 and 48, of 16 to 4000 77 and 63, of
// 200 and one of 50000 93 and 474; 1024 of them 185 and 89, 183 and 110, 152 and
// 474; 2048 469 and 171, 460 and 188, 370 and 474.
constexpr int kFp4Shared = 1024;

// The first key that any of a sequence's nq new tokens sees, of n keys.
constexpr int fp4_first(int n, int nq, int window) {
    const int first = window > 0 && n - nq + 1 - window > 0 ? n - nq + 1 - window : 0;
    return first < n ? first : n;
}
// Chunks are counted in steps of 128 keys, from a multiple of 32 on.
constexpr int fp4_steps(int n, int first) {
    const int steps = (n - (first & ~31) + 127) >> 7;
    return steps > 1 ? steps : 1;
}
// A narrow sequence's column blocks of `cols` rows each; every one of them goes
// through every chunk of the keys.
constexpr int fp4_blocks(int64_t rows, int cols) { return (int)((rows + cols - 1) / cols); }
// Steps in a chunk, where the launch's sequences have `total` steps times column
// blocks: as many units (a chunk and a column block) as wanted, but no more than
// a third of them below 512 keys.  At least total / items, so that there are no
// more units than items and one for each column block.
constexpr int fp4_step(uint64_t total, uint32_t items) {
    if (total >= (uint64_t)1 << 31) {  // a little more, in fp32
        const float step = (float)total / (float)items * 1.001f + 1.0f;
        return step < 8388608.0f ? (int)step + 1 : 1 << 23;  // 2^30 keys: all of a sequence
    }
    const uint32_t t = (uint32_t)total, few = items / 3 > 1 ? items / 3 : 1;
    const uint32_t even = (t + items - 1) / items, some = (t + few - 1) / few;
    const uint32_t step = even > (some < 4u ? some : 4u) ? even : (some < 4u ? some : 4u);
    return (int)(step < 1u ? 1u : step < 1u << 23 ? step : 1u << 23);
}

struct Fp4Join {
    int ncol, groups, most;
    int narrow;  // rows as (sequence, key head, up to `most`): the narrow ones beside a tiled kernel's
    int rows;    // rows as (token, head): all, or the wide ones
    int blocks;  // workgroups of them
    int weigh;   // workgroups of a (sequence, key head) behind them that add its keys' weights up
};

struct Fp4Plan {
    int nc, cblocks;   // 16-row column sets of a narrow workgroup; column blocks of a sequence at most
    int items;         // units wanted; 0: cblocks for each sequence
    int64_t units;     // at most
    int most, limit;   // rows of a narrow sequence
    int splits;         // of a wide sequence's keys
    int64_t slots;      // blocks of wide rows at most; 0: no sequence is wide
    bool apart;         // narrow and wide sequences in launches of their own
    int64_t grid;       // workgroups
    Fp4Join join;
    int64_t plan_bytes, part_bytes, raw_bytes, wide_bytes, raw_ld;
    bool fits;  // the launches, in what they are counted in
    constexpr int64_t bytes() const { return plan_bytes + part_bytes + raw_bytes + wide_bytes; }
};

// packed: several tokens a sequence; weighed: the keys' weights are kept, of the
// first weight_len keys.  kMost: workgroups of a launch at most.
constexpr Fp4Plan fp4_plan(int64_t n, int64_t B, int64_t H, int64_t h_kv, int64_t D, int64_t pages, int64_t page, int64_t window,
                           bool packed, bool weighed, int64_t kMost, int64_t weight_len = (int64_t)1 << 31) {
    Fp4Plan r = {};
    const int64_t G = H / h_kv, room = pages * page;
    auto seen = [=](int64_t tokens) {  // keys that a sequence's tokens see
        const int64_t x = window > 0 && window + tokens - 1 < room ? window + tokens - 1 : room;
        return x > 1 ? x : 1;
    };
    // Else every sequence is one chunk, and blocks of wide rows have slots by their starts.
    const bool shared = B <= kFp4Shared && room > 128;
    int64_t most = G;
    r.splits = 1;
    if (packed) {
        // Few rows in all are narrow however they are shared out.
        r.limit = n * G <= kFp4AllNarrow && n * G * seen(n) * h_kv <= kFp4AllWork ? kFp4AllNarrow : kFp4Narrow;
        most = n * G < r.limit ? n * G : r.limit;
        if (n * G > r.limit) {
            const int64_t blocks = (n * G + kFp4Rows - 1) / kFp4Rows, some = n * G / (r.limit + 1);
            r.slots = n * G / kFp4Rows + (!shared ? B + 1 : B < some ? B : some);
            // Two workgroups a compute unit, none under two tiles of 64 keys (a mixed
            // step of 9 sequences 22.4 us, with four tiles 34.3, with one 21.4 and twice
            // the partial sums).
            int64_t splits = 512 / (blocks * h_kv);
            if (splits > seen(kFp4Rows) / 128) splits = seen(kFp4Rows) / 128;
            r.splits = (int)(splits < 1 ? 1 : splits);
            if (r.splits > 1) r.wide_bytes = n * H * r.splits * (D + 4) * 4;
        }
    }
    r.most = (int)most;
    r.apart = r.slots > 0 && n * G <= kFp4Narrow * B && B * seen(r.limit) * h_kv >= kFp4Apart;
    r.nc = !weighed && most > 16 && (!packed || (r.slots > 0 && !r.apart) || n * G > 16 * B) ? 2 : 1;
    r.cblocks = (r.most + 16 * r.nc - 1) / (16 * r.nc);
    r.items = (int)(!shared ? 0 : fp4_wanted(r.nc) / h_kv > 1 ? fp4_wanted(r.nc) / h_kv : 1);
    // Column blocks of all narrow sequences; none of these has more tokens than rows.
    const int64_t cols = 16 * r.nc, each_has = B * r.cblocks, by_rows = n * G / cols + B;
    const int64_t all = packed && by_rows < each_has ? by_rows : each_has;
    const int64_t longest = (seen(packed ? r.limit : 1) + 31 + 127) / 128;
    r.units = !shared ? each_has : r.items + all < all * longest ? r.items + all : all * longest;
    r.grid = (r.slots * r.splits + r.units) * h_kv;
    r.plan_bytes = (B * 8 + 15) / 16 * 16;
    if (shared || weighed) r.part_bytes = r.units * h_kv * cols * (D + 4) * 4;
    r.raw_ld = (seen(1) + 31 + 31) / 32 * 32;
    if (r.raw_ld > (weight_len + 31) / 32 * 32) r.raw_ld = (weight_len + 31) / 32 * 32;
    const bool countable = r.raw_ld < ((int64_t)1 << 60) / (B * H + 1);
    if (weighed && countable) r.raw_bytes = B * H * r.raw_ld * 4;

    r.join.most = r.most;
    r.join.ncol = 2;
    while (4 * r.join.ncol < D) r.join.ncol *= 2;
    // Threads that share a row's splits: as many as there may be, until the launch
    // fills the chip.
    const int64_t per = r.items / (B > 0 ? B : 1) + 1, each = per < longest ? per : longest;
    const int64_t narrow = shared && r.slots > 0 ? B * h_kv * r.most : 0;
    const int64_t rows = (r.slots > 0 ? r.splits > 1 : shared) ? n * H : 0;
    int64_t blocks = 0;
    for (r.join.groups = 1;; r.join.groups *= 2) {
        const int64_t each_block = 256 / (r.join.ncol * r.join.groups);
        blocks = (narrow + rows + each_block - 1) / each_block;
        if (2 * r.join.groups * r.join.ncol > 256 || r.join.groups >= each || blocks >= 1024) break;
    }
    const int64_t heads = B * h_kv, share = heads < kFp4Weigh ? kFp4Weigh / (heads > 0 ? heads : 1) : 1, keys = (r.raw_ld + 255) / 256;
    const int64_t weigh = weighed ? (keys < share ? keys : share) : 0;
    r.fits = r.grid <= kMost && (countable || !weighed) && narrow + rows < (int64_t)1 << 31 && blocks + heads * weigh <= kMost;
    if (r.fits) {
        r.join.narrow = (int)narrow;
        r.join.rows = (int)rows;
        r.join.blocks = (int)blocks;
        r.join.weigh = (int)weigh;
    }
    return r;
}

}  // namespace qdl
