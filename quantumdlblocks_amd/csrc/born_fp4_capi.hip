// C ABI of the 4-bit paged cache (declared in include/qdl_flash_born.h): checks
// the argument blocks and launches on the caller's stream.  No allocation, no
// synchronisation, no global state.
#include <stdint.h>

#include "../../include/qdl_flash_born.h"
#include "born_fp4_cache.h"
#include "born_fp4_paged.h"
#include "born_fp4_tiled.h"

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
int hip_status(hipError_t e) { return e == hipSuccess ? QDL_BORN_OK : (int)e; }
int64_t item(int64_t dtype) { return dtype == QDL_BORN_DTYPE_F32 ? 4 : 2; }

// A launch's threads are counted in 32 bits.
constexpr int64_t kMostBlocks = ((int64_t)1 << 24) - 1;
constexpr int64_t kMostRows = (int64_t)1 << 28;
constexpr int64_t kMostHeads = (int64_t)1 << 16;

int check_heads(int64_t dtype, int64_t H, int64_t h_kv, int64_t D) {
    if (dtype != QDL_BORN_DTYPE_F32 && dtype != QDL_BORN_DTYPE_F16 && dtype != QDL_BORN_DTYPE_BF16) return QDL_BORN_E_DTYPE;
    if (D < 8 || D > 256 || D % 8 != 0) return QDL_BORN_E_HEADDIM;
    if (h_kv < 1 || H < 1 || H % h_kv != 0) return QDL_BORN_E_HEADS;
    if (H > kMostHeads) return QDL_BORN_E_SHAPE;
    return QDL_BORN_OK;
}

bool stride_ok(int64_t s, int64_t unit) { return s >= 0 && s <= (int64_t)1 << 40 && s % unit == 0; }
bool cache_stride_ok(int64_t s, int64_t unit) { return stride_ok(s, unit) && s < (int64_t)1 << 32; }
bool rows_ok(const int64_t st[2], int64_t it) { return stride_ok(st[0] * it, 16) && stride_ok(st[1] * it, 16); }

int check_cache(const qdl_born_fp4_cache& c, int64_t B) {
    for (int i = 0; i < 3; ++i)
        if (!cache_stride_ok(c.k_strides[i], 16) || !cache_stride_ok(c.v_strides[i], 16) || !cache_stride_ok(c.k_scale_strides[i], 1) ||
            !cache_stride_ok(c.v_scale_strides[i], 1))
            return QDL_BORN_E_STRIDE;
    if (c.page_size < 1 || c.page_size > (int64_t)1 << 24 || c.cache_pages < 0 || c.cache_pages > INT32_MAX || c.pages < 0 ||
        c.table_ld < c.pages || c.pages > (int64_t)1 << 30 || c.pages * c.page_size > (int64_t)1 << 30)
        return QDL_BORN_E_PAGE;
    if (B > 0 && ((c.pages > 0 && !c.block_table) || !c.cache_lens || (c.cache_pages > 0 && (!c.k || !c.v || !c.k_scale || !c.v_scale))))
        return QDL_BORN_E_NULL;
    if (!aligned16(c.k) || !aligned16(c.v)) return QDL_BORN_E_ALIGN;
    return QDL_BORN_OK;
}

int shift_of(int64_t page) {
    for (int i = 0; i < 25; ++i)
        if (page == (int64_t)1 << i) return i;
    return -1;
}

void set_cache(qdl::Fp4Cache& a, qdl::Fp4Pages& t, const qdl_born_fp4_cache& c, int64_t D) {
    a.k = static_cast<uint8_t*>(c.k);
    a.v = static_cast<uint8_t*>(c.v);
    a.ks = static_cast<uint8_t*>(c.k_scale);
    a.vs = static_cast<uint8_t*>(c.v_scale);
    a.kp = (uint32_t)c.k_strides[0], a.kt = (uint32_t)c.k_strides[1], a.kh = (uint32_t)c.k_strides[2];
    a.vp = (uint32_t)c.v_strides[0], a.vt = (uint32_t)c.v_strides[1], a.vh = (uint32_t)c.v_strides[2];
    a.ksp = (uint32_t)c.k_scale_strides[0], a.kst = (uint32_t)c.k_scale_strides[1], a.ksh = (uint32_t)c.k_scale_strides[2];
    a.vsp = (uint32_t)c.v_scale_strides[0], a.vst = (uint32_t)c.v_scale_strides[1], a.vsh = (uint32_t)c.v_scale_strides[2];
    a.cache_pages = (int)c.cache_pages;
    a.page = (int)c.page_size;
    a.page_shift = shift_of(c.page_size);
    a.nb = (int)((D + qdl::kFp4Block - 1) / qdl::kFp4Block);
    t.table = c.block_table;
    t.lens = c.cache_lens;
    t.table_ld = c.table_ld;
    t.pages = (int)c.pages;
}

int64_t append_blocks(int64_t n, int64_t rows, int lanes) {
    const int64_t per = 256 / lanes;
    return (n * rows + per - 1) / per;
}

template <class E, int VEC, bool WHOLE>
void launch_append(const qdl::Fp4AppendArgs& a, bool many, int64_t blocks, hipStream_t st) {
    if (many) hipLaunchKernelGGL((qdl::born_fp4_append_kernel<E, VEC, 4, WHOLE>), dim3((unsigned)blocks), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((qdl::born_fp4_append_kernel<E, VEC, 1, WHOLE>), dim3((unsigned)blocks), dim3(256), 0, st, a);
}

}  // namespace

extern "C" {

int qdl_flash_born_fp4_append_call(const qdl_born_fp4_append_call* c, qdl_stream_t stream) {
    if (!c) return QDL_BORN_E_NULL;
    if (c->struct_bytes != (int64_t)sizeof(qdl_born_fp4_append_call)) return QDL_BORN_E_SHAPE;
    int rc = check_heads(c->dtype, c->H, c->h_kv, c->D);
    if (rc != QDL_BORN_OK) return rc;
    if (c->n < 0 || c->n > kMostRows || c->B < 0 || c->B > kMostRows || (!c->cu_seqlens && c->n != c->B)) return QDL_BORN_E_SHAPE;
    if (!(c->eps >= 0.0)) return QDL_BORN_E_SHAPE;
    rc = check_cache(c->cache, c->B);
    if (rc != QDL_BORN_OK) return rc;
    if (c->n == 0) return QDL_BORN_OK;
    if (!c->q || !c->k || !c->v || !c->q_out) return QDL_BORN_E_NULL;
    if (!aligned16(c->q) || !aligned16(c->k) || !aligned16(c->v) || !aligned16(c->q_out)) return QDL_BORN_E_ALIGN;
    const int64_t it = item(c->dtype);
    if (!rows_ok(c->q_strides, it) || !rows_ok(c->k_strides, it) || !rows_ok(c->v_strides, it)) return QDL_BORN_E_STRIDE;
    if (c->cos_table && (!c->sin_table || c->table_rows < 1 || c->table_rows > INT32_MAX || c->n_freq < 0 ||
                         c->n_freq > c->D / 2 || c->freq_ld < c->n_freq))
        return QDL_BORN_E_TABLE;
    qdl::Fp4AppendArgs a = {};
    set_cache(a.c, a.t, c->cache, c->D);
    a.q = c->q;
    a.k = c->k;
    a.v = c->v;
    a.q_out = c->q_out;
    a.cos = c->cos_table;
    a.sin = c->sin_table;
    a.positions = c->positions;
    a.cu = c->cu_seqlens;
    a.N = (int)c->n;
    a.B = (int)c->B;
    a.H = (int)c->H;
    a.Hkv = (int)c->h_kv;
    a.D = (int)c->D;
    a.q_st = c->q_strides[0] * it;
    a.q_sh = c->q_strides[1] * it;
    a.k_st = c->k_strides[0] * it;
    a.k_sh = c->k_strides[1] * it;
    a.v_st = c->v_strides[0] * it;
    a.v_sh = c->v_strides[1] * it;
    a.table_rows = (int)c->table_rows;
    a.n_freq = (int)c->n_freq;
    a.freq_ld = c->freq_ld;
    a.wide_tables = c->cos_table && c->freq_ld % 4 == 0 && aligned16(c->cos_table) && aligned16(c->sin_table) ? 1 : 0;
    a.eps = c->eps;
    // 16-byte pieces where half a row holds whole ones, else 8-byte pieces.
    const bool whole = c->D % 16 == 0;
    const int vec = c->dtype != QDL_BORN_DTYPE_F32 && whole ? 8 : 4;
    a.lpr = 1;
    while (a.lpr * vec < c->D / 2) a.lpr *= 2;
    a.lpw = 4;
    while (a.lpw < 4 * a.c.nb) a.lpw *= 2;
    // Groups of four heads where single ones would fill the chip twice over (16384
    // tokens, 32 heads over 8, D128, read back too: 100 us, with single ones 144).
    const bool many = c->n * c->H * a.lpr >= (int64_t)1 << 20;
    const int64_t queries = append_blocks(c->n, many ? (c->H + 3) / 4 : c->H, a.lpr);
    const int each = many ? qdl::kFp4AppendHeads<4> : qdl::kFp4AppendHeads<1>;
    a.heads = (int)((c->h_kv + each - 1) / each);
    a.tokens = (int)append_blocks(c->n, 1, a.lpw);
    const int64_t blocks = queries + (c->cache.cache_pages > 0 ? 2 * (int64_t)a.heads * a.tokens : 0);
    if (blocks > kMostBlocks) return QDL_BORN_E_SHAPE;
    a.q_blocks = (int)queries;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    switch (c->dtype) {
        case QDL_BORN_DTYPE_BF16:
            if (whole) launch_append<qdl::BF16, 8, true>(a, many, blocks, s);
            else launch_append<qdl::BF16, 4, false>(a, many, blocks, s);
            break;
        case QDL_BORN_DTYPE_F16:
            if (whole) launch_append<qdl::F16, 8, true>(a, many, blocks, s);
            else launch_append<qdl::F16, 4, false>(a, many, blocks, s);
            break;
        default:
            if (whole) launch_append<qdl::F32, 4, true>(a, many, blocks, s);
            else launch_append<qdl::F32, 4, false>(a, many, blocks, s);
            break;
    }
    return hip_status(hipGetLastError());
}

int qdl_flash_born_fp4_read_call(const qdl_born_fp4_read_call* c, qdl_stream_t stream) {
    if (!c) return QDL_BORN_E_NULL;
    if (c->struct_bytes != (int64_t)sizeof(qdl_born_fp4_read_call)) return QDL_BORN_E_SHAPE;
    int rc = check_heads(c->dtype, c->h_kv, c->h_kv, c->D);
    if (rc != QDL_BORN_OK) return rc;
    if (c->n < 0 || c->n > kMostRows || c->B < 0 || c->B > kMostRows) return QDL_BORN_E_SHAPE;
    rc = check_cache(c->cache, c->B);
    if (rc != QDL_BORN_OK) return rc;
    if (c->n == 0) return QDL_BORN_OK;
    if (!c->k_out || !c->v_out || !c->cu_seqlens) return QDL_BORN_E_NULL;
    if (!aligned16(c->k_out) || !aligned16(c->v_out)) return QDL_BORN_E_ALIGN;
    qdl::Fp4ReadArgs a = {};
    set_cache(a.c, a.t, c->cache, c->D);
    a.cu = c->cu_seqlens;
    a.k = c->k_out;
    a.v = c->v_out;
    a.N = (int)c->n;
    a.B = (int)c->B;
    a.Hkv = (int)c->h_kv;
    a.D = (int)c->D;
    a.lpr = 1;
    while (a.lpr * 8 < c->D) a.lpr *= 2;
    a.heads = (int)((c->h_kv + qdl::kFp4ReadHeads - 1) / qdl::kFp4ReadHeads);
    const int64_t blocks = append_blocks(c->n, 1, a.lpr) * a.heads;
    if (blocks > kMostBlocks) return QDL_BORN_E_SHAPE;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    switch (c->dtype) {
        case QDL_BORN_DTYPE_BF16: hipLaunchKernelGGL((qdl::born_fp4_read_kernel<qdl::BF16>), dim3((unsigned)blocks), dim3(256), 0, s, a); break;
        case QDL_BORN_DTYPE_F16: hipLaunchKernelGGL((qdl::born_fp4_read_kernel<qdl::F16>), dim3((unsigned)blocks), dim3(256), 0, s, a); break;
        default: hipLaunchKernelGGL((qdl::born_fp4_read_kernel<qdl::F32>), dim3((unsigned)blocks), dim3(256), 0, s, a); break;
    }
    return hip_status(hipGetLastError());
}

int64_t qdl_flash_born_fp4_paged_workspace_size(int64_t n, int64_t B, int64_t H, int64_t h_kv, int64_t D, int64_t pages,
                                                int64_t page_size, int64_t window_size, int packed, int weighed) {
    if (n <= 0 || n > kMostRows || B < 0 || B > kMostHeads || H <= 0 || H > kMostHeads || h_kv <= 0 || H % h_kv != 0 || D <= 0 || D > 256 ||
        pages < 0 || page_size < 1 || page_size > (int64_t)1 << 24 || pages > (int64_t)1 << 30 ||
        pages * page_size > (int64_t)1 << 30 || window_size < 0 || weighed < 0)
        return 0;
    const qdl::Fp4Plan r = qdl::fp4_plan(n, B, H, h_kv, D, pages, page_size, window_size, packed != 0, weighed != 0, kMostBlocks,
                                         weighed > 1 ? weighed : INT32_MAX);
    return r.fits ? r.bytes() : 0;
}

int qdl_flash_born_fp4_paged_forward_call(const qdl_born_fp4_paged_call* c, qdl_stream_t stream) {
    if (!c) return QDL_BORN_E_NULL;
    if (c->struct_bytes != (int64_t)sizeof(qdl_born_fp4_paged_call)) return QDL_BORN_E_SHAPE;
    int rc = check_heads(c->dtype, c->H, c->h_kv, c->D);
    if (rc != QDL_BORN_OK) return rc;
    if (c->n < 0 || c->n > kMostRows || c->B < 0 || c->B > kMostHeads || (c->B == 0 && c->n > 0) || (!c->cu_seqlens && c->n != c->B))
        return QDL_BORN_E_SHAPE;
    if (c->scale && c->n_scale != 1 && c->n_scale != c->H) return QDL_BORN_E_SCALE;
    if (c->window_size < 0 || c->window_size > (int64_t)1 << 30) return QDL_BORN_E_WINDOW;
    if (!(c->eps >= 0.0) || (c->key_weight && (c->cu_seqlens || c->weight_len < 0 || c->weight_len > INT32_MAX))) return QDL_BORN_E_SHAPE;
    rc = check_cache(c->cache, c->B);
    if (rc != QDL_BORN_OK) return rc;
    if (c->n == 0) return QDL_BORN_OK;
    if (!c->q || !c->out) return QDL_BORN_E_NULL;
    if (!aligned16(c->q) || !aligned16(c->out)) return QDL_BORN_E_ALIGN;
    const int64_t it = item(c->dtype);
    if (!rows_ok(c->q_strides, it)) return QDL_BORN_E_STRIDE;
    const bool weighed = c->key_weight != nullptr && c->weight_len > 0;
    const qdl::Fp4Plan r = qdl::fp4_plan(c->n, c->B, c->H, c->h_kv, c->D, c->cache.pages, c->cache.page_size, c->window_size,
                                         c->cu_seqlens != nullptr, weighed, kMostBlocks, weighed ? c->weight_len : 0);
    if (!r.fits) return QDL_BORN_E_SHAPE;
    if (!c->workspace || !aligned16(c->workspace) || c->workspace_bytes < r.bytes()) return QDL_BORN_E_WORKSPACE;
    qdl::Fp4PagedArgs a = {};
    set_cache(a.c, a.t, c->cache, c->D);
    a.q = c->q;
    a.out = c->out;
    a.cu = c->cu_seqlens;
    a.scale = c->scale;
    a.scale_value = (float)c->scale_value;
    a.per_head_scale = c->scale && c->n_scale > 1 ? 1 : 0;
    a.B = (int)c->B;
    a.N = (int)c->n;
    a.H = (int)c->H;
    a.Hkv = (int)c->h_kv;
    a.G = (int)(c->H / c->h_kv);
    a.D = (int)c->D;
    a.window = (int)c->window_size;
    a.items = r.items;
    a.cblocks = r.cblocks;
    a.units = (int)r.units;
    a.cols = 16 * r.nc;
    a.limit = r.limit;
    a.splits = r.splits;
    a.slots = r.slots;
    a.eps = (float)c->eps;
    a.q_st = c->q_strides[0] * it;
    a.q_sh = c->q_strides[1] * it;
    uint8_t* ws = static_cast<uint8_t*>(c->workspace);
    a.plan = reinterpret_cast<int2*>(ws);
    a.part = reinterpret_cast<float*>(ws + r.plan_bytes);
    a.wide_part = reinterpret_cast<float*>(ws + r.plan_bytes + r.part_bytes + r.raw_bytes);
    if (weighed) {
        a.raw = reinterpret_cast<float*>(ws + r.plan_bytes + r.part_bytes);
        a.raw_ld = r.raw_ld;
        a.weights = c->key_weight;
        a.w_sb = c->weight_strides[0];
        a.w_sh = c->weight_strides[1];
        a.w_len = (int)c->weight_len;
    }
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    switch (c->dtype) {
        case QDL_BORN_DTYPE_BF16: return hip_status(qdl::fp4_paged_fwd<qdl::BF16>(a, r, s));
        case QDL_BORN_DTYPE_F16: return hip_status(qdl::fp4_paged_fwd<qdl::F16>(a, r, s));
        default: return hip_status(qdl::fp4_paged_fwd<qdl::F32>(a, r, s));
    }
}

int qdl_flash_born_fp4_evict_call(const qdl_born_fp4_evict_call* c, qdl_stream_t stream) {
    if (!c) return QDL_BORN_E_NULL;
    if (c->struct_bytes != (int64_t)sizeof(qdl_born_fp4_evict_call)) return QDL_BORN_E_SHAPE;
    int rc = check_heads(QDL_BORN_DTYPE_BF16, c->h_kv, c->h_kv, c->D);
    if (rc != QDL_BORN_OK) return rc;
    if (c->B < 0 || c->B > kMostRows || c->B * c->h_kv > kMostBlocks / 8) return QDL_BORN_E_SHAPE;
    rc = check_cache(c->cache, c->B);
    if (rc != QDL_BORN_OK) return rc;
    if (c->budget < 0 || c->recent < 0 || c->budget > (int64_t)1 << 30 || c->recent > (int64_t)1 << 30) return QDL_BORN_E_BUDGET;
    if (c->weight_len < 0 || c->weight_len > (int64_t)1 << 30) return QDL_BORN_E_SHAPE;
    if (c->out_table && (c->out_pages < 0 || c->out_pages > (int64_t)1 << 30 || c->out_table_ld < c->out_pages)) return QDL_BORN_E_PAGE;
    if (c->B == 0) return QDL_BORN_OK;
    if (!c->lens_out || (c->budget > 0 && !c->kept) || (c->weight_len > 0 && (!c->key_weight || !c->weight_out))) return QDL_BORN_E_NULL;
    // Outputs that other workgroups still read as inputs.
    if (c->lens_out == c->cache.cache_lens || (c->weight_len > 0 && c->weight_out == c->key_weight)) return QDL_BORN_E_SHAPE;
    if (c->out_table && c->out_table == c->cache.block_table) return QDL_BORN_E_PAGE;
    qdl::Fp4EvictArgs a = {};
    qdl::Fp4Pages t;
    set_cache(a.c, t, c->cache, c->D);
    const int64_t room = c->cache.pages * c->cache.page_size, most = c->budget < room ? c->budget : room;  // kept rows
    const int64_t per = qdl::fp4_evict_rows(a.c.nb), tiles = (most + per - 1) / per;
    if (c->out_table && tiles * c->B * c->h_kv > kMostBlocks) return QDL_BORN_E_SHAPE;
    a.s.table = t.table;
    a.s.to = c->out_table;
    a.s.lens = t.lens;
    a.s.weight = c->key_weight;
    a.s.weight_out = c->weight_out;
    a.s.lens_out = c->lens_out;
    a.s.kept = c->kept;
    a.s.B = (int)c->B;
    a.s.Hkv = (int)c->h_kv;
    a.s.pages = t.pages;
    a.s.to_pages = (int)c->out_pages;
    a.s.page = a.c.page;
    a.s.page_shift = a.c.page_shift;
    a.s.table_ld = t.table_ld;
    a.s.to_ld = c->out_table_ld;
    a.s.cache_pages = c->cache.cache_pages;
    a.s.w_sb = c->weight_strides[0];
    a.s.w_sh = c->weight_strides[1];
    a.s.w_len = (int)c->weight_len;
    a.s.budget = (int)c->budget;
    a.s.recent = (int)c->recent;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const unsigned units = (unsigned)(c->B * c->h_kv);
    qdl::launch_evict_select(a.s, units, room, s);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || most == 0 || c->cache.cache_pages == 0) return hip_status(e);
    if (c->out_table) hipLaunchKernelGGL((qdl::born_fp4_evict_move_kernel<0>), dim3((unsigned)tiles * units), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((qdl::born_fp4_evict_compact_kernel<0>), dim3(units), dim3(1024), 0, s, a);
    return hip_status(hipGetLastError());
}

}  // extern "C"
