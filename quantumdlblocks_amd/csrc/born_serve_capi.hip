// C ABI of the packed, paged and cache operators (declared in
// include/qdl_flash_born.h): checks the argument blocks and launches on the
// caller's stream.  No allocation, no synchronisation, no global state.
#include <stdint.h>

#include "../../include/qdl_flash_born.h"
#include "born_cache.h"
#include "born_packed.h"
#include "born_paged.h"

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
int hip_status(hipError_t e) { return e == hipSuccess ? QDL_BORN_OK : (int)e; }
bool dtype_ok(int64_t d) { return d == QDL_BORN_DTYPE_F32 || d == QDL_BORN_DTYPE_F16 || d == QDL_BORN_DTYPE_BF16; }
int64_t item(int64_t dtype) { return dtype == QDL_BORN_DTYPE_F32 ? 4 : 2; }

// A launch's threads are counted in 32 bits.
constexpr int64_t kMostBlocks = ((int64_t)1 << 24) - 1;
constexpr int64_t kMostRows = (int64_t)1 << 28;
constexpr int64_t kMostHeads = (int64_t)1 << 16;

int check_heads(int64_t dtype, int64_t H, int64_t h_kv, int64_t D) {
    if (!dtype_ok(dtype)) return QDL_BORN_E_DTYPE;
    if (D < 8 || D > 256 || D % 8 != 0) return QDL_BORN_E_HEADDIM;
    if (h_kv < 1 || H < 1 || H % h_kv != 0) return QDL_BORN_E_HEADS;
    if (H > kMostHeads) return QDL_BORN_E_SHAPE;
    return QDL_BORN_OK;
}

// Strides in elements: whole 16-byte pieces; a token's rows may not overlap.
bool stride_ok(int64_t s, int64_t it) { return s >= 0 && s <= (int64_t)1 << 40 && s * it % 16 == 0; }
bool rows_ok(const int64_t st[2], int64_t it, int64_t D) {
    return stride_ok(st[0], it) && stride_ok(st[1], it) && st[0] >= D && st[0] * it < (int64_t)1 << 24;
}

int check_cache(int64_t dtype, const int64_t ks[3], const int64_t vs[3], int64_t cache_pages, int64_t page,
                const void* k, const void* v, const int32_t* table, int64_t pages, int64_t table_ld) {
    const int64_t it = item(dtype);
    for (int i = 0; i < 3; ++i)
        if (!stride_ok(ks[i], it) || !stride_ok(vs[i], it)) return QDL_BORN_E_STRIDE;
    if (page < 1 || page > (int64_t)1 << 24 || cache_pages < 0 || cache_pages > INT32_MAX || pages < 0 || table_ld < pages ||
        pages > (int64_t)1 << 30 || pages * page > (int64_t)1 << 30)
        return QDL_BORN_E_PAGE;
    if ((pages > 0 && !table) || (cache_pages > 0 && (!k || !v))) return QDL_BORN_E_NULL;
    if (!aligned16(k) || !aligned16(v)) return QDL_BORN_E_ALIGN;
    return QDL_BORN_OK;
}

int shift_of(int64_t page) {
    for (int i = 0; i < 25; ++i)
        if (page == (int64_t)1 << i) return i;
    return -1;
}

int check_packed(const qdl_born_packed_call* c) {
    if (!c) return QDL_BORN_E_NULL;
    if (c->struct_bytes != (int64_t)sizeof(qdl_born_packed_call)) return QDL_BORN_E_SHAPE;
    const int rc = check_heads(c->dtype, c->H, c->h_kv, c->D);
    if (rc != QDL_BORN_OK) return rc;
    if (c->sequences < 0 || c->n_q < 0 || c->n_k < 0 || c->n_q > kMostRows || c->n_k > kMostRows || c->sequences > kMostRows)
        return QDL_BORN_E_SHAPE;
    if ((c->n_q / qdl::packed_rows(4) + c->sequences + 1) * c->H > kMostBlocks ||
        (c->n_k / qdl::packed_rows(4) + c->sequences + 1) * c->H > kMostBlocks || c->n_k * c->h_kv * c->D > (int64_t)1 << 33)
        return QDL_BORN_E_SHAPE;
    // dK/dV's workgroups have 512 threads.
    if ((c->n_k / qdl::packed_rows(1) + c->sequences + 1) * c->h_kv > kMostBlocks / 2) return QDL_BORN_E_SHAPE;
    if (c->scale && c->n_scale != 1 && c->n_scale != c->H) return QDL_BORN_E_SCALE;
    if (c->window_size < 0 || c->window_size > (int64_t)1 << 30) return QDL_BORN_E_WINDOW;
    if (!(c->eps >= 0.0)) return QDL_BORN_E_SHAPE;
    if (!c->cu_q || !c->cu_k) return QDL_BORN_E_NULL;
    if ((c->n_q > 0 && (!c->q || !c->out)) || (c->n_k > 0 && (!c->k || !c->v))) return QDL_BORN_E_NULL;
    if (!aligned16(c->q) || !aligned16(c->k) || !aligned16(c->v) || !aligned16(c->out)) return QDL_BORN_E_ALIGN;
    const int64_t it = item(c->dtype);
    if (!rows_ok(c->q_strides, it, c->D) || !rows_ok(c->k_strides, it, c->D) || !rows_ok(c->v_strides, it, c->D))
        return QDL_BORN_E_STRIDE;
    return QDL_BORN_OK;
}

qdl::PackedArgs packed_args(const qdl_born_packed_call* c) {
    const int64_t it = item(c->dtype);
    qdl::PackedArgs a = {};
    a.q = c->q;
    a.k = c->k;
    a.v = c->v;
    a.o = a.out = c->out;
    a.dout = c->dout;
    a.dq = c->dq;
    a.dk = c->dk;
    a.dv = c->dv;
    a.z = c->z;
    a.scale = c->scale;
    a.scale_value = (float)c->scale_value;
    a.per_head_scale = c->scale && c->n_scale > 1 ? 1 : 0;
    a.cu_q = c->cu_q;
    a.cu_k = c->cu_k;
    a.S = (int)c->sequences;
    a.Nq = (int)c->n_q;
    a.Nk = (int)c->n_k;
    a.H = (int)c->H;
    a.Hkv = (int)c->h_kv;
    a.G = (int)(c->H / c->h_kv);
    a.D = (int)c->D;
    a.lower = qdl::packed_lower(c->is_causal != 0);
    a.upper = qdl::packed_upper(c->window_size);
    a.head_splits = 1;
    a.eps = (float)c->eps;
    a.q_st = c->q_strides[0] * it;
    a.q_sh = c->q_strides[1] * it;
    a.k_st = c->k_strides[0] * it;
    a.k_sh = c->k_strides[1] * it;
    a.v_st = c->v_strides[0] * it;
    a.v_sh = c->v_strides[1] * it;
    a.do_st = c->dout_strides[0] * it;
    a.do_sh = c->dout_strides[1] * it;
    return a;
}

int64_t packed_stats(int64_t n_q, int64_t H) { return (H * n_q * 4 + 15) / 16 * 16; }

qdl::PackedPlan packed_plan(const qdl_born_packed_call* c) {
    return qdl::packed_plan((int)item(c->dtype), c->n_q, c->n_k, c->sequences, c->H, c->h_kv, c->D, c->window_size);
}
// The backward's workspace: the rows' two values, dscale's parts, and the sums
// of head splits.
int64_t packed_workspace(const qdl_born_packed_call* c) {
    return 2 * packed_stats(c->n_q, c->H) + c->H * qdl::kPackedParts * 8 + qdl::packed_part_bytes(packed_plan(c), c->n_k, c->h_kv, c->D);
}

// Splits of a paged launch: enough workgroups for four a compute unit, none
// under 128 keys (a wave's 32) or over 1024.  Eight a unit cut the chunks finer
// and mostly pay more in partial sums than they level: us at four and at eight,
// bf16, 64 sequences of 1024 keys, 8 key heads, D64 42.2 and 44.8, D128 66.4 and
// 70.8; 16 of 512..8192, 4 key heads, D64 23.7 and 23.9, D128 36.5 and 39.5.
// One ragged batch with the keys' weights gained (fp16 D64: 35.1 and 31.8),
// another of its shape did not (bf16: 32.0 and 32.2).
struct PagedPlan {
    int64_t chunk, nsplit, gblocks, raw_ld, part_bytes, raw_bytes;
    int64_t bytes() const { return part_bytes + raw_bytes; }
};
PagedPlan paged_plan(int64_t B, int64_t H, int64_t h_kv, int64_t D, int64_t pages, int64_t page, int64_t window, bool weigh) {
    PagedPlan r = {};
    const int64_t room = pages * page;
    int64_t span = window > 0 && window + 31 < room ? window + 31 : room;
    if (span < 1) span = 1;
    r.gblocks = (H / h_kv + 15) / 16;
    const int64_t units = B * h_kv * r.gblocks;
    const int64_t want = units > 0 ? (1024 + units - 1) / units : 1;
    int64_t chunk = (span + want - 1) / want;
    chunk = (chunk + 127) / 128 * 128;
    if (chunk > 1024) chunk = 1024;
    r.chunk = chunk;
    r.nsplit = (span + chunk - 1) / chunk;
    r.raw_ld = (span + 31) / 32 * 32;
    if (r.nsplit > 1 || weigh) r.part_bytes = B * H * r.nsplit * (D + 4) * 4;
    if (weigh) r.raw_bytes = B * H * r.raw_ld * 4;
    return r;
}
PagedPlan paged_plan(const qdl_born_paged_call* c) {
    return paged_plan(c->B, c->H, c->h_kv, c->D, c->pages, c->page_size, c->window_size, c->key_weight != nullptr);
}

int check_paged(const qdl_born_paged_call* c) {
    if (!c) return QDL_BORN_E_NULL;
    if (c->struct_bytes != (int64_t)sizeof(qdl_born_paged_call)) return QDL_BORN_E_SHAPE;
    int rc = check_heads(c->dtype, c->H, c->h_kv, c->D);
    if (rc != QDL_BORN_OK) return rc;
    if (c->B < 0 || c->B > kMostHeads || c->B * c->H > kMostBlocks) return QDL_BORN_E_SHAPE;
    if (c->scale && c->n_scale != 1 && c->n_scale != c->H) return QDL_BORN_E_SCALE;
    if (c->window_size < 0 || c->window_size > (int64_t)1 << 30) return QDL_BORN_E_WINDOW;
    if (!(c->eps >= 0.0)) return QDL_BORN_E_SHAPE;
    rc = check_cache(c->dtype, c->k_cache_strides, c->v_cache_strides, c->cache_pages, c->page_size, c->k_cache, c->v_cache,
                     c->block_table, c->pages, c->table_ld);
    if (rc != QDL_BORN_OK) return rc;
    const PagedPlan r = paged_plan(c);
    if (c->B * c->h_kv * r.gblocks * r.nsplit > kMostBlocks ||
        (c->key_weight && c->B * (c->H + c->h_kv * (r.raw_ld / 256 + 1)) > kMostBlocks))
        return QDL_BORN_E_SHAPE;
    if (c->key_weight && (c->weight_len < 0 || c->weight_len > INT32_MAX)) return QDL_BORN_E_SHAPE;
    return QDL_BORN_OK;
}

int64_t append_blocks(int64_t n, int64_t rows, int lpr, bool many) {
    const int64_t per = 256 / lpr;
    return (n * (many ? (rows + 3) / 4 : rows) + per - 1) / per;
}

template <class E, int VEC>
void launch_append(const qdl::AppendArgs& a, bool many, hipStream_t st) {
    const int64_t blocks = append_blocks(a.N, a.H + 2 * a.Hkv, a.lpr, many);
    if (many) hipLaunchKernelGGL((qdl::born_append_kernel<E, VEC, 4>), dim3((unsigned)blocks), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((qdl::born_append_kernel<E, VEC, 1>), dim3((unsigned)blocks), dim3(256), 0, st, a);
}

}  // namespace

extern "C" {

int qdl_flash_born_packed_forward_call(const qdl_born_packed_call* c, qdl_stream_t stream) {
    const int rc = check_packed(c);
    if (rc != QDL_BORN_OK) return rc;
    if (c->n_q == 0) return QDL_BORN_OK;
    const qdl::PackedArgs a = packed_args(c);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    switch (c->dtype) {
        case QDL_BORN_DTYPE_BF16: return hip_status(qdl::packed_fwd<qdl::BF16>(a, packed_plan(c), s));
        case QDL_BORN_DTYPE_F16: return hip_status(qdl::packed_fwd<qdl::F16>(a, packed_plan(c), s));
        default: return hip_status(qdl::packed_fwd<qdl::F32>(a, packed_plan(c), s));
    }
}

int64_t qdl_flash_born_packed_workspace_size(const qdl_born_packed_call* c) {
    return check_packed(c) == QDL_BORN_OK ? packed_workspace(c) : 0;
}

int qdl_flash_born_packed_backward_call(const qdl_born_packed_call* c, qdl_stream_t stream) {
    const int rc = check_packed(c);
    if (rc != QDL_BORN_OK) return rc;
    if ((c->n_q > 0 && (!c->dout || !c->dq || !c->z)) || (c->n_k > 0 && !c->dk != !c->dv)) return QDL_BORN_E_NULL;
    if (!aligned16(c->dout) || !aligned16(c->dq) || !aligned16(c->dk) || !aligned16(c->dv)) return QDL_BORN_E_ALIGN;
    if (c->n_q > 0 && !rows_ok(c->dout_strides, item(c->dtype), c->D)) return QDL_BORN_E_STRIDE;
    if (c->workspace_bytes < packed_workspace(c) || !c->workspace || !aligned16(c->workspace))
        return QDL_BORN_E_WORKSPACE;
    qdl::PackedArgs a = packed_args(c);
    uint8_t* ws = static_cast<uint8_t*>(c->workspace);
    a.ndelta = reinterpret_cast<float*>(ws);
    a.zs = reinterpret_cast<float*>(ws + packed_stats(c->n_q, c->H));
    double* part = reinterpret_cast<double*>(ws + 2 * packed_stats(c->n_q, c->H));
    const qdl::PackedPlan plan = packed_plan(c);
    a.head_splits = plan.head_splits;
    if (plan.head_splits > 1) a.part = reinterpret_cast<float*>(part + c->H * qdl::kPackedParts);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    hipError_t e;
    switch (c->dtype) {
        case QDL_BORN_DTYPE_BF16: e = qdl::packed_bwd<qdl::BF16>(a, plan, s); break;
        case QDL_BORN_DTYPE_F16: e = qdl::packed_bwd<qdl::F16>(a, plan, s); break;
        default: e = qdl::packed_bwd<qdl::F32>(a, plan, s); break;
    }
    if (e != hipSuccess || !c->dscale) return hip_status(e);
    hipLaunchKernelGGL((qdl::born_packed_dscale_part_kernel<0>), dim3((unsigned)a.H, qdl::kPackedParts), dim3(256), 0, s, a, part);
    e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
    hipLaunchKernelGGL((qdl::born_packed_dscale_kernel<0>), dim3(1), dim3(64), 0, s, a, part, c->dscale,
                       a.per_head_scale ? a.H : 1, c->dtype == QDL_BORN_DTYPE_F16 ? (double)qdl::kUp<qdl::F16> : 1.0);
    return hip_status(hipGetLastError());
}

int64_t qdl_flash_born_paged_workspace_size(int64_t B, int64_t H, int64_t h_kv, int64_t D, int64_t pages, int64_t page_size,
                                            int64_t window_size, int weighed) {
    if (B <= 0 || B > kMostHeads || H <= 0 || H > kMostHeads || h_kv <= 0 || H % h_kv != 0 || D <= 0 || D > 256 || pages < 0 ||
        page_size < 1 || page_size > (int64_t)1 << 24 || pages > (int64_t)1 << 30 || pages * page_size > (int64_t)1 << 30 || window_size < 0)
        return 0;
    return paged_plan(B, H, h_kv, D, pages, page_size, window_size, weighed != 0).bytes();
}

int qdl_flash_born_paged_forward_call(const qdl_born_paged_call* c, qdl_stream_t stream) {
    const int rc = check_paged(c);
    if (rc != QDL_BORN_OK) return rc;
    if (c->B == 0) return QDL_BORN_OK;
    if (!c->q || !c->out || !c->cache_lens) return QDL_BORN_E_NULL;
    if (!aligned16(c->q) || !aligned16(c->out)) return QDL_BORN_E_ALIGN;
    const int64_t it = item(c->dtype);
    if (!stride_ok(c->q_strides[0], it) || !stride_ok(c->q_strides[1], it)) return QDL_BORN_E_STRIDE;
    const PagedPlan r = paged_plan(c);
    if (r.bytes() > 0 && (!c->workspace || !aligned16(c->workspace) || c->workspace_bytes < r.bytes()))
        return QDL_BORN_E_WORKSPACE;
    qdl::PagedArgs a = {};
    a.q = c->q;
    a.k = c->k_cache;
    a.v = c->v_cache;
    a.out = c->out;
    a.table = c->block_table;
    a.lens = c->cache_lens;
    a.scale = c->scale;
    a.scale_value = (float)c->scale_value;
    a.per_head_scale = c->scale && c->n_scale > 1 ? 1 : 0;
    a.B = (int)c->B;
    a.H = (int)c->H;
    a.Hkv = (int)c->h_kv;
    a.G = (int)(c->H / c->h_kv);
    a.D = (int)c->D;
    a.pages = (int)c->pages;
    a.table_ld = c->table_ld;
    a.cache_pages = c->cache_pages;
    a.page = (int)c->page_size;
    a.page_shift = shift_of(c->page_size);
    a.window = (int)c->window_size;
    a.nsplit = (int)r.nsplit;
    a.chunk = (int)r.chunk;
    a.gblocks = (int)r.gblocks;
    a.eps = (float)c->eps;
    a.q_sb = c->q_strides[0] * it;
    a.q_sh = c->q_strides[1] * it;
    a.kp = c->k_cache_strides[0] * it;
    a.kt = c->k_cache_strides[1] * it;
    a.kh = c->k_cache_strides[2] * it;
    a.vp = c->v_cache_strides[0] * it;
    a.vt = c->v_cache_strides[1] * it;
    a.vh = c->v_cache_strides[2] * it;
    uint8_t* ws = static_cast<uint8_t*>(c->workspace);
    if (r.part_bytes > 0) a.part = reinterpret_cast<float*>(ws);
    if (r.raw_bytes > 0) {
        a.raw = reinterpret_cast<float*>(ws + r.part_bytes);
        a.raw_ld = r.raw_ld;
        a.weights = c->key_weight;
        a.w_sb = c->weight_strides[0];
        a.w_sh = c->weight_strides[1];
        a.w_len = (int)c->weight_len;
    }
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    switch (c->dtype) {
        case QDL_BORN_DTYPE_BF16: return hip_status(qdl::paged_fwd<qdl::BF16>(a, s));
        case QDL_BORN_DTYPE_F16: return hip_status(qdl::paged_fwd<qdl::F16>(a, s));
        default: return hip_status(qdl::paged_fwd<qdl::F32>(a, s));
    }
}

int qdl_flash_born_cache_append_call(const qdl_born_append_call* c, qdl_stream_t stream) {
    if (!c) return QDL_BORN_E_NULL;
    if (c->struct_bytes != (int64_t)sizeof(qdl_born_append_call)) return QDL_BORN_E_SHAPE;
    int rc = check_heads(c->dtype, c->H, c->h_kv, c->D);
    if (rc != QDL_BORN_OK) return rc;
    if (c->n < 0 || c->n > kMostRows || c->B < 0 || c->B > kMostRows || (!c->cu_seqlens && c->n != c->B)) return QDL_BORN_E_SHAPE;
    if (!(c->eps >= 0.0)) return QDL_BORN_E_SHAPE;
    rc = check_cache(c->dtype, c->k_cache_strides, c->v_cache_strides, c->cache_pages, c->page_size, c->k_cache, c->v_cache,
                     c->block_table, c->pages, c->table_ld);
    if (rc != QDL_BORN_OK) return rc;
    if (c->n == 0) return QDL_BORN_OK;
    if (!c->q || !c->k || !c->v || !c->q_out || (c->B > 0 && !c->cache_lens)) return QDL_BORN_E_NULL;
    if (!aligned16(c->q) || !aligned16(c->k) || !aligned16(c->v) || !aligned16(c->q_out)) return QDL_BORN_E_ALIGN;
    const int64_t it = item(c->dtype);
    for (int i = 0; i < 2; ++i)
        if (!stride_ok(c->q_strides[i], it) || !stride_ok(c->k_strides[i], it) || !stride_ok(c->v_strides[i], it))
            return QDL_BORN_E_STRIDE;
    if (c->cos_table && (!c->sin_table || c->table_rows < 1 || c->table_rows > INT32_MAX || c->n_freq < 0 ||
                         c->n_freq > c->D / 2 || c->freq_ld < c->n_freq))
        return QDL_BORN_E_TABLE;
    qdl::AppendArgs a = {};
    a.q = c->q;
    a.k = c->k;
    a.v = c->v;
    a.q_out = c->q_out;
    a.k_cache = c->k_cache;
    a.v_cache = c->v_cache;
    a.cos = c->cos_table;
    a.sin = c->sin_table;
    a.positions = c->positions;
    a.table = c->block_table;
    a.lens = c->cache_lens;
    a.cu = c->cu_seqlens;
    a.N = (int)c->n;
    a.B = (int)c->B;
    a.H = (int)c->H;
    a.Hkv = (int)c->h_kv;
    a.D = (int)c->D;
    a.pages = (int)c->pages;
    a.page = (int)c->page_size;
    a.page_shift = shift_of(c->page_size);
    a.table_ld = c->table_ld;
    a.cache_pages = c->cache_pages;
    a.q_st = c->q_strides[0] * it;
    a.q_sh = c->q_strides[1] * it;
    a.k_st = c->k_strides[0] * it;
    a.k_sh = c->k_strides[1] * it;
    a.v_st = c->v_strides[0] * it;
    a.v_sh = c->v_strides[1] * it;
    a.kp = c->k_cache_strides[0] * it;
    a.kt = c->k_cache_strides[1] * it;
    a.kh = c->k_cache_strides[2] * it;
    a.vp = c->v_cache_strides[0] * it;
    a.vt = c->v_cache_strides[1] * it;
    a.vh = c->v_cache_strides[2] * it;
    a.table_rows = (int)c->table_rows;
    a.n_freq = (int)c->n_freq;
    a.freq_ld = c->freq_ld;
    a.eps = (float)c->eps;
    // 16-byte pieces where half a row holds whole ones, else 8-byte pieces.
    const bool wide = c->dtype == QDL_BORN_DTYPE_F32 || c->D % 16 == 0;
    const int vec = wide && c->dtype != QDL_BORN_DTYPE_F32 ? 8 : 4;
    int lpr = 1;
    while (lpr * vec < c->D / 2) lpr *= 2;
    a.lpr = lpr;
    // Groups of four rows where single ones would fill the chip twice over
    // (256 CUs x 32 waves x 64 lanes).  us with single rows and with groups, bf16,
    // 16 heads over 4, D128: 1024 tokens 13.6 and 13.0, 4096 (under the bound)
    // 23.9 and 19.4, 8192 41.2 and 31.0; 16384, 32 over 8: 134 and 89; fp32 D64,
    // 8192: 33.7 and 28.2.
    const bool many = c->n * (c->H + 2 * c->h_kv) * lpr >= (int64_t)1 << 20;
    if (append_blocks(c->n, c->H + 2 * c->h_kv, lpr, many) > kMostBlocks) return QDL_BORN_E_SHAPE;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    switch (c->dtype) {
        case QDL_BORN_DTYPE_BF16:
            if (vec == 8) launch_append<qdl::BF16, 8>(a, many, s);
            else launch_append<qdl::BF16, 4>(a, many, s);
            break;
        case QDL_BORN_DTYPE_F16:
            if (vec == 8) launch_append<qdl::F16, 8>(a, many, s);
            else launch_append<qdl::F16, 4>(a, many, s);
            break;
        default: launch_append<qdl::F32, 4>(a, many, s); break;
    }
    return hip_status(hipGetLastError());
}

int qdl_flash_born_cache_evict_call(const qdl_born_evict_call* c, qdl_stream_t stream) {
    if (!c) return QDL_BORN_E_NULL;
    if (c->struct_bytes != (int64_t)sizeof(qdl_born_evict_call)) return QDL_BORN_E_SHAPE;
    int rc = check_heads(c->dtype, c->h_kv, c->h_kv, c->D);
    if (rc != QDL_BORN_OK) return rc;
    if (c->B < 0 || c->B > kMostRows || c->B * c->h_kv > kMostBlocks / 8) return QDL_BORN_E_SHAPE;
    rc = check_cache(c->dtype, c->k_cache_strides, c->v_cache_strides, c->cache_pages, c->page_size, c->k_cache, c->v_cache,
                     c->block_table, c->pages, c->table_ld);
    if (rc != QDL_BORN_OK) return rc;
    if (c->budget < 0 || c->recent < 0 || c->budget > (int64_t)1 << 30 || c->recent > (int64_t)1 << 30) return QDL_BORN_E_BUDGET;
    if (c->weight_len < 0 || c->weight_len > (int64_t)1 << 30) return QDL_BORN_E_SHAPE;
    if (c->out_table && (c->out_pages < 0 || c->out_pages > (int64_t)1 << 30 || c->out_table_ld < c->out_pages)) return QDL_BORN_E_PAGE;
    if (c->B == 0) return QDL_BORN_OK;
    if (!c->cache_lens || !c->lens_out || (c->budget > 0 && !c->kept) || (c->weight_len > 0 && (!c->key_weight || !c->weight_out)))
        return QDL_BORN_E_NULL;
    // Outputs that other workgroups still read as inputs.
    if (c->lens_out == c->cache_lens || (c->weight_len > 0 && c->weight_out == c->key_weight)) return QDL_BORN_E_SHAPE;
    if (c->out_table && c->out_table == c->block_table) return QDL_BORN_E_PAGE;
    const int64_t it = item(c->dtype);
    const int64_t most = c->budget < c->pages * c->page_size ? c->budget : c->pages * c->page_size;  // kept rows
    const int64_t per = qdl::evict_rows((int)(c->D * it / 16)), tiles = (most + per - 1) / per;
    if (c->out_table && tiles * c->B * c->h_kv > kMostBlocks) return QDL_BORN_E_SHAPE;
    qdl::EvictArgs a = {};
    a.k = c->k_cache;
    a.v = c->v_cache;
    a.table = c->block_table;
    a.to = c->out_table;
    a.lens = c->cache_lens;
    a.weight = c->key_weight;
    a.weight_out = c->weight_out;
    a.lens_out = c->lens_out;
    a.kept = c->kept;
    a.B = (int)c->B;
    a.Hkv = (int)c->h_kv;
    a.D = (int)c->D;
    a.item = (int)it;
    a.pages = (int)c->pages;
    a.to_pages = (int)c->out_pages;
    a.page = (int)c->page_size;
    a.page_shift = shift_of(c->page_size);
    a.table_ld = c->table_ld;
    a.to_ld = c->out_table_ld;
    a.cache_pages = c->cache_pages;
    a.kp = c->k_cache_strides[0] * it;
    a.kt = c->k_cache_strides[1] * it;
    a.kh = c->k_cache_strides[2] * it;
    a.vp = c->v_cache_strides[0] * it;
    a.vt = c->v_cache_strides[1] * it;
    a.vh = c->v_cache_strides[2] * it;
    a.w_sb = c->weight_strides[0];
    a.w_sh = c->weight_strides[1];
    a.w_len = (int)c->weight_len;
    a.budget = (int)c->budget;
    a.recent = (int)c->recent;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const unsigned units = (unsigned)(c->B * c->h_kv);
    qdl::launch_evict_select(a, units, c->pages * c->page_size, s);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || most == 0 || c->cache_pages == 0) return hip_status(e);
    if (c->out_table) hipLaunchKernelGGL((qdl::born_evict_move_kernel<0>), dim3((unsigned)tiles * units), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((qdl::born_evict_compact_kernel<0>), dim3(2 * units), dim3(1024), 0, s, a);
    return hip_status(hipGetLastError());
}

}  // extern "C"
