// vc_rt_paged.cu - the C ABI of voxtral_cuda.h, the operators over a paged
// cache in 8 bits (rotary append, attention, copies of pages): argument checks
// and launches.  None of them allocates, waits for the host or keeps a
// workspace, so calls on different streams are independent and a call may be
// captured into a CUDA graph.
#include "vc_rt_check.h"

#include <algorithm>
#include <limits.h>

using namespace vc;
using namespace vc::rt;

namespace {

// table: the call follows the streams' pages
int check_pool(const char *who, const vox_cuda_paged_cache *c, bool table, PagedView *out) {
    if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale || (table && !c->table)) {
        set_error("%s: no cache, or one without scales or table", who);
        return VOX_CUDA_ERR_ARG;
    }
    if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128) {
        set_error("%s: page_size must be 16, 32, 64 or 128, not %d", who, c->page_size);
        return VOX_CUDA_ERR_ARG;
    }
    if (c->n_layers < 1 || c->n_layers > 32767 || c->n_pages < 1 || c->n_kv_heads < 1 || c->n_kv_heads > 4096 ||
        (table && (c->n_streams < 1 || c->n_streams > 65535 || c->table_stride < 1 ||
                   c->table_stride > kMaxPosition / c->page_size))) {
        set_error("%s: bad cache shape (%d layers, %d pages, %d heads, %d streams of %d pages)", who, c->n_layers, c->n_pages,
                  c->n_kv_heads, c->n_streams, c->table_stride);
        return VOX_CUDA_ERR_ARG;
    }
    if (c->head_dim != 64 && c->head_dim != 128) {
        set_error("%s: head_dim must be 64 or 128, not %d", who, c->head_dim);
        return VOX_CUDA_ERR_ARG;
    }
    PagedView v = {};
    v.k = static_cast<unsigned char *>(c->k);
    v.v = static_cast<unsigned char *>(c->v);
    v.k_scale = c->k_scale;
    v.v_scale = c->v_scale;
    v.table = c->table;
    v.table_stride = c->table_stride;
    v.n_layers = c->n_layers;
    v.n_pages = c->n_pages;
    v.page = c->page_size;
    v.page_shift = c->page_size == 16 ? 4 : c->page_size == 32 ? 5 : c->page_size == 64 ? 6 : 7;
    v.n_streams = c->n_streams;
    v.n_kv_heads = c->n_kv_heads;
    v.head_dim = c->head_dim;
    v.slot_stride = c->slot_stride ? c->slot_stride : c->head_dim;
    v.head_stride = c->head_stride ? c->head_stride : (long long)c->page_size * v.slot_stride;
    const double span = std::max((double)c->n_kv_heads * v.head_stride, (double)c->page_size * v.slot_stride);   // of a page, whichever is outside
    v.page_stride = c->page_stride ? c->page_stride : (long long)std::min(span, 1e16);
    v.layer_stride = c->layer_stride ? c->layer_stride : (long long)std::min(std::max((double)c->n_pages * v.page_stride, span), 1e16);
    const long long st[4] = {v.slot_stride, v.head_stride, v.page_stride, v.layer_stride};
    for (long long s : st)
        if (s < c->head_dim || s % 16 != 0) {
            set_error("%s: cache strides must be multiples of 16 bytes, of a head at least (%lld)", who, s);
            return VOX_CUDA_ERR_ARG;
        }
    const double extent = (double)v.layer_stride * v.n_layers + (double)v.page_stride * v.n_pages +
                          (double)v.head_stride * v.n_kv_heads + (double)v.slot_stride * v.page;
    if (extent > 1e15) {
        set_error("%s: cache strides are too large", who);
        return VOX_CUDA_ERR_ARG;
    }
    // each axis steps over all that the ones inside it hold, whatever their order
    struct Axis {
        long long stride, n;
    } axes[4] = {{v.slot_stride, v.page}, {v.head_stride, v.n_kv_heads}, {v.page_stride, v.n_pages}, {v.layer_stride, v.n_layers}};
    std::sort(axes, axes + 4, [](const Axis &a, const Axis &b) { return a.stride < b.stride; });
    long long inside = c->head_dim;
    for (const Axis &a : axes) {
        if (a.n == 1) continue;
        if (a.stride < inside) {
            set_error("%s: cache strides must keep slots, heads, pages and layers apart (%lld bytes over %lld)", who, a.stride, inside);
            return VOX_CUDA_ERR_ARG;
        }
        inside += a.stride * (a.n - 1);
    }
    if (!aligned16(c->k) || !aligned16(c->v) || !aligned4(c->k_scale) || !aligned4(c->v_scale) || (table && !aligned4(c->table))) {
        set_error("%s: the cache must be 16-byte aligned, its scales as fp32 is, its table as int is", who);
        return VOX_CUDA_ERR_ARG;
    }
    *out = v;
    return VOX_CUDA_OK;
}

int check_paged_rows(const char *who, const vox_cuda_rows *r, const PagedView &c, RowsView *out) {
    const int rc = check_rows(who, r, c.n_streams, INT_MAX, 0, out);
    if (rc) return rc;
    if (r->max_rows > (long long)c.table_stride * c.page) {
        set_error("%s: %d pages of %d positions cannot hold %d rows", who, c.table_stride, c.page, r->max_rows);
        return VOX_CUDA_ERR_CAPACITY;
    }
    return VOX_CUDA_OK;
}

int check_q_type(const char *who, int type) {
    if (type == ELEM_BF16 || type == ELEM_F16) return VOX_CUDA_OK;
    set_error("%s: q must be bf16 or fp16", who);
    return VOX_CUDA_ERR_ARG;
}

int attention(const char *who, const vox_cuda_paged_cache *cache, int layer, const vox_cuda_rows *rows, const void *q, int q_type,
              int n_heads, int window, int n_sink, float scale, void *out, float *lse, void *stream, int stall_ms = 0,
              RowsPlan *only = nullptr) {
    PagedAttnParams p = {};
    int rc = check_pool(who, cache, true, &p.c);
    if (rc || (rc = check_paged_rows(who, rows, p.c, &p.r)) || (rc = check_layer(who, layer, p.c.n_layers)) ||
        (rc = check_heads(who, n_heads, p.c.n_kv_heads)) || (rc = check_q_type(who, q_type)))
        return rc;
    if (window < 0 || n_sink < 0 || !(fabsf(scale) <= 2.0e38f)) {
        set_error("%s: bad window, sinks or scale", who);
        return VOX_CUDA_ERR_ARG;
    }
    if (p.r.n_rows == 0) return VOX_CUDA_OK;
    if (!q || !out || !aligned16(q) || !aligned16(out) || !aligned4(lse)) {
        set_error("%s: q and out must be 16-byte aligned device pointers", who);
        return VOX_CUDA_ERR_ARG;
    }
    const double lines = (double)p.r.n_rows * n_heads, bytes = lines * p.c.head_dim * 2;
    if ((q != out && overlap(q, bytes, out, bytes)) || overlap(lse, lines * sizeof(float), q, bytes) ||
        overlap(lse, lines * sizeof(float), out, bytes)) {   // CTAs would read what others have written
        set_error("%s: out is q itself or apart from it, lse apart from both", who);
        return VOX_CUDA_ERR_ARG;
    }
    if ((long long)p.r.max_rows * (n_heads / p.c.n_kv_heads) > (1 << 28)) {
        set_error("%s: too many rows of a stream (%d)", who, p.r.max_rows);
        return VOX_CUDA_ERR_ARG;
    }
    DevCtx *c = cur_ctx();
    if (!c) return VOX_CUDA_ERR_UNAVAILABLE;
    DeviceGuard guard(c->device);
    if (!guard.ok()) return launched(who, cudaGetLastError());
    if (!only && (rc = check_waits(who, c))) return rc;
    p.err = c->op_err + op_slot();
    p.stall_ns = stall_ms * 1000000ull;
    p.layer = layer;
    p.q = q;
    p.out = out;
    p.q_type = q_type;
    p.lse = lse;
    p.n_heads = n_heads;
    p.group = n_heads / p.c.n_kv_heads;
    const int room = p.c.table_stride * p.c.page;
    p.window = window < room ? window : 0;   // a stream has no more positions: no limit (and no sum overflows)
    p.n_sink = p.window > 0 ? min(n_sink, room) : 0;
    p.scale_log2 = (scale == 0.f ? 1.0f / sqrtf((float)p.c.head_dim) : scale) * 1.4426950408889634f;
    return launched(who, launch_paged_attn(p, c->sms, stream ? (cudaStream_t)stream : c->stream, only));
}

}  // namespace

extern "C" int vox_cuda_rope_append_paged_dev(const vox_cuda_paged_cache *cache, int layer, const vox_cuda_rows *rows,
                                              const void *qkv, int qkv_type, int n_heads, long long qkv_stride,
                                              const float *q_norm, const float *k_norm, float eps, float theta, void *q_out,
                                              int q_type, void *stream) {
    const char *who = "rope_append_paged";
    PagedAppendParams p = {};
    int rc = check_pool(who, cache, true, &p.c);
    if (rc || (rc = check_paged_rows(who, rows, p.c, &p.r)) || (rc = check_layer(who, layer, p.c.n_layers)) ||
        (rc = check_heads(who, n_heads, p.c.n_kv_heads)) || (rc = check_q_type(who, q_type)))
        return rc;
    if (qkv_type != ELEM_F32 && qkv_type != q_type) {
        set_error("%s: q|k|v must be fp32 or of q's type", who);
        return VOX_CUDA_ERR_ARG;
    }
    const int elem = elem_size(qkv_type);
    const long long width = (long long)(n_heads + 2 * p.c.n_kv_heads) * p.c.head_dim;
    const long long ld = qkv_stride ? qkv_stride : width;
    if (ld < width || ld * elem % 16 != 0 || ld > (1ll << 40)) {
        set_error("%s: rows of %lld elements need a stride of as many, a multiple of 16 bytes (not %lld)", who, width, ld);
        return VOX_CUDA_ERR_ARG;
    }
    if (!(eps >= 0.f) || !(theta >= 0.f) || !(theta <= 3.0e38f)) {
        set_error("%s: eps and theta must not be negative", who);
        return VOX_CUDA_ERR_ARG;
    }
    if (p.r.n_rows == 0) return VOX_CUDA_OK;
    if (!qkv || !q_out || !aligned16(qkv) || !aligned16(q_out) || !aligned16(q_norm) || !aligned16(k_norm)) {
        set_error("%s: q|k|v, q_out and the norm weights must be 16-byte aligned device pointers", who);
        return VOX_CUDA_ERR_ARG;
    }
    if (overlap(qkv, (double)ld * p.r.n_rows * elem, q_out, (double)p.r.n_rows * n_heads * p.c.head_dim * 2)) {
        set_error("%s: q_out must not overlap q|k|v", who);
        return VOX_CUDA_ERR_ARG;
    }
    DevCtx *c = cur_ctx();
    if (!c) return VOX_CUDA_ERR_UNAVAILABLE;
    DeviceGuard guard(c->device);
    if (!guard.ok()) return launched(who, cudaGetLastError());
    p.layer = layer;
    p.qkv = qkv;
    p.src_type = qkv_type;
    p.ld = ld;
    p.n_heads = n_heads;
    p.q_norm = q_norm;
    p.k_norm = k_norm;
    p.eps = eps;
    p.rotate = theta > 0.f;
    p.log2_theta = theta > 0.f ? log2((double)theta) : 0.0;
    p.q_out = q_out;
    p.q_type = q_type;
    return launched(who, launch_paged_append(p, stream ? (cudaStream_t)stream : c->stream));
}

extern "C" int vox_cuda_attention_paged_dev(const vox_cuda_paged_cache *cache, int layer, const vox_cuda_rows *rows,
                                            const void *q, int q_type, int n_heads, int window, int n_sink, float scale,
                                            void *out, float *lse, void *stream) {
    return attention("attention_paged", cache, layer, rows, q, q_type, n_heads, window, n_sink, scale, out, lse, stream);
}

extern "C" int vox_cuda_selftest_attention_paged_plan(const vox_cuda_paged_cache *cache, const vox_cuda_rows *rows, int q_type,
                                                      int n_heads, int window, int n_sink, int *plan) {
    const char *who = "selftest_attention_paged_plan";
    if (!plan || !rows || rows->n_rows < 1) {
        set_error("%s: no rows, or no place for the answer", who);
        return VOX_CUDA_ERR_ARG;
    }
    RowsPlan form = {};
    void *some = cache ? cache->k : nullptr;   // (an aligned address; nothing is launched)
    const int rc = attention(who, cache, 0, rows, some, q_type, n_heads, window, n_sink, 0.f, some, nullptr, nullptr, 0, &form);
    if (rc) return rc;
    plan[0] = form.rows;
    plan[1] = form.ctas;
    plan[2] = form.shares;
    return VOX_CUDA_OK;
}

extern "C" int vox_cuda_selftest_attention_paged_timeout(const vox_cuda_paged_cache *cache, int layer, const vox_cuda_rows *rows,
                                                         const void *q, int q_type, int n_heads, void *out, float *lse, int wait_ms,
                                                         void *stream) {
    const char *who = "selftest_attention_paged_timeout";
    int plan[3];
    const int rc = vox_cuda_selftest_attention_paged_plan(cache, rows, q_type, n_heads, 0, 0, plan);
    if (rc) return rc;
    if (wait_ms < 1 || wait_ms > 10000 || plan[0] < 128) {
        set_error("%s: wait_ms must be 1..10000, the rows many (the few-rows kernel has no waits)", who);
        return VOX_CUDA_ERR_ARG;
    }
    return attention(who, cache, layer, rows, q, q_type, n_heads, 0, 0, 0.f, out, lse, stream, wait_ms);
}

extern "C" int vox_cuda_kv_copy_pages_dev(const vox_cuda_paged_cache *cache, const int *src, const int *dst, int n, void *stream) {
    const char *who = "kv_copy_pages";
    PagedCopyParams p = {};
    int rc = check_pool(who, cache, false, &p.c);
    if (rc) return rc;
    if (n < 0 || n > p.c.n_pages || (n > 0 && (!src || !dst))) {
        set_error("%s: bad arguments (0 to %d pairs)", who, p.c.n_pages);
        return VOX_CUDA_ERR_ARG;
    }
    if (n == 0) return VOX_CUDA_OK;
    if (!aligned4(src) || !aligned4(dst)) {
        set_error("%s: the pages' numbers must be aligned as int is", who);
        return VOX_CUDA_ERR_ARG;
    }
    DevCtx *c = cur_ctx();
    if (!c) return VOX_CUDA_ERR_UNAVAILABLE;
    DeviceGuard guard(c->device);
    if (!guard.ok()) return launched(who, cudaGetLastError());
    p.src = src;
    p.dst = dst;
    p.n = n;
    return launched(who, launch_paged_copy(p, c->sms, stream ? (cudaStream_t)stream : c->stream));
}
