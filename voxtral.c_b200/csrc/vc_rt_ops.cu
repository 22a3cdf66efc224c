// vc_rt_ops.cu - the C ABI of voxtral_cuda.h, the row operators over a cache
// slab (rotary append, window and tree attention, commit, fork) and the token
// log probabilities: argument checks and launches.  None of them allocates,
// waits for the host or keeps a workspace, so calls on different streams are
// independent and a call may be captured into a CUDA graph.
#include "vc_rt_check.h"

using namespace vc;
using namespace vc::rt;

namespace {

int check_cache(const char *who, const vox_cuda_kv_cache *c, CacheView *out) {
    if (!c || !c->k || !c->v) {
        set_error("%s: no cache", who);
        return VOX_CUDA_ERR_ARG;
    }
    if (!known_type(c->dtype)) {
        set_error("%s: unknown cache type %d", who, c->dtype);
        return VOX_CUDA_ERR_ARG;
    }
    if (c->n_layers < 1 || c->n_layers > 32767 || c->n_streams < 1 || c->n_streams > 65535 || c->n_kv_heads < 1 ||
        c->n_kv_heads > 4096 || c->cap < 1 || c->cap > kMaxPosition) {
        set_error("%s: bad cache shape (%d layers, %d streams, %d slots, %d heads)", who, c->n_layers, c->n_streams, c->cap,
                  c->n_kv_heads);
        return VOX_CUDA_ERR_ARG;
    }
    if (c->head_dim != 64 && c->head_dim != 128) {
        set_error("%s: head_dim must be 64 or 128, not %d", who, c->head_dim);
        return VOX_CUDA_ERR_ARG;
    }
    if (c->n_sink < 0 || c->n_sink >= c->cap) {
        set_error("%s: %d sinks leave no ring in %d slots", who, c->n_sink, c->cap);
        return VOX_CUDA_ERR_ARG;
    }
    CacheView v = {};
    v.k = static_cast<char *>(c->k);
    v.v = static_cast<char *>(c->v);
    v.dtype = c->dtype;
    v.n_layers = c->n_layers;
    v.n_streams = c->n_streams;
    v.cap = c->cap;
    v.n_kv_heads = c->n_kv_heads;
    v.head_dim = c->head_dim;
    v.n_sink = c->n_sink;
    v.ring = c->cap - c->n_sink;
    v.head_stride = c->head_stride ? c->head_stride : c->head_dim;
    v.slot_stride = c->slot_stride ? c->slot_stride : (long long)c->n_kv_heads * c->head_dim;
    v.stream_stride = c->stream_stride ? c->stream_stride : (long long)c->cap * v.slot_stride;
    v.layer_stride = c->layer_stride ? c->layer_stride : (long long)c->n_streams * v.stream_stride;
    const int per16 = 16 / elem_size(c->dtype);
    const long long st[4] = {v.head_stride, v.slot_stride, v.stream_stride, v.layer_stride};
    for (long long s : st)
        if (s < c->head_dim || s % per16 != 0) {
            set_error("%s: cache strides must be multiples of 16 bytes, of a head at least (%lld elements)", who, s);
            return VOX_CUDA_ERR_ARG;
        }
    const double extent = (double)v.layer_stride * v.n_layers + (double)v.stream_stride * v.n_streams +
                          (double)v.slot_stride * v.cap + (double)v.head_stride * v.n_kv_heads;
    if (extent > 1e15) {
        set_error("%s: cache strides are too large", who);
        return VOX_CUDA_ERR_ARG;
    }
    if (!aligned16(c->k) || !aligned16(c->v)) {
        set_error("%s: the cache must be 16-byte aligned", who);
        return VOX_CUDA_ERR_ARG;
    }
    *out = v;
    return VOX_CUDA_OK;
}

int attention(const char *who, bool tree, const vox_cuda_kv_cache *cache, int layer, const vox_cuda_rows *rows, const void *q,
              int n_heads, int window, float scale, void *out, float *lse, void *stream, int stall_ms = 0,
              RowsPlan *only = nullptr) {
    RowsAttnParams p = {};
    int rc = check_cache(who, cache, &p.c);
    if (rc || (rc = check_rows(who, rows, p.c.n_streams, p.c.ring, tree ? 2 : 0, &p.r)) ||
        (rc = check_layer(who, layer, p.c.n_layers)) || (rc = check_heads(who, n_heads, p.c.n_kv_heads)))
        return rc;
    if (window < 0 || !(fabsf(scale) <= 2.0e38f)) {
        set_error("%s: bad window or scale", who);
        return VOX_CUDA_ERR_ARG;
    }
    if (p.r.n_rows == 0) return VOX_CUDA_OK;
    if (!q || !out || !aligned16(q) || !aligned16(out)) {
        set_error("%s: q and out must be 16-byte aligned device pointers", who);
        return VOX_CUDA_ERR_ARG;
    }
    const double lines = (double)p.r.n_rows * n_heads, bytes = lines * p.c.head_dim * elem_size(p.c.dtype);
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
    p.layer_off = (long long)layer * p.c.layer_stride;
    p.q = q;
    p.out = out;
    p.lse = lse;
    p.n_heads = n_heads;
    p.group = n_heads / p.c.n_kv_heads;
    p.window = window < p.c.ring ? window : 0;   // the ring holds no more: no limit (and no sum overflows)
    p.scale_log2 = (scale == 0.f ? 1.0f / sqrtf((float)p.c.head_dim) : scale) * 1.4426950408889634f;
    return launched(who, launch_attn_rows(p, stream ? (cudaStream_t)stream : c->stream, only));
}

}  // namespace

extern "C" int vox_cuda_attention_window_dev(const vox_cuda_kv_cache *cache, int layer, const vox_cuda_rows *rows,
                                             const void *q, int n_heads, int window, float scale, void *out, float *lse,
                                             void *stream) {
    return attention("attention_window", false, cache, layer, rows, q, n_heads, window, scale, out, lse, stream);
}

extern "C" int vox_cuda_attention_tree_dev(const vox_cuda_kv_cache *cache, int layer, const vox_cuda_rows *rows,
                                           const void *q, int n_heads, int window, float scale, void *out, float *lse,
                                           void *stream) {
    return attention("attention_tree", true, cache, layer, rows, q, n_heads, window, scale, out, lse, stream);
}

extern "C" int vox_cuda_selftest_attention_timeout(const vox_cuda_kv_cache *cache, int layer, const vox_cuda_rows *rows,
                                                   const void *q, int n_heads, void *out, float *lse, int wait_ms,
                                                   void *stream) {
    const char *who = "selftest_attention_timeout";
    if (wait_ms < 1 || wait_ms > 10000 || (cache && cache->dtype == ELEM_F32)) {
        set_error("%s: wait_ms must be 1..10000, the cache of 16 bits (the fp32 kernels have no waits)", who);
        return VOX_CUDA_ERR_ARG;
    }
    return attention(who, false, cache, layer, rows, q, n_heads, 0, 0.f, out, lse, stream, wait_ms);
}

extern "C" int vox_cuda_selftest_attention_plan(const vox_cuda_kv_cache *cache, const vox_cuda_rows *rows, int n_heads,
                                                int window, int *plan) {
    const char *who = "selftest_attention_plan";
    if (!plan || !rows || rows->n_rows < 1) {
        set_error("%s: no rows, or no place for the answer", who);
        return VOX_CUDA_ERR_ARG;
    }
    RowsPlan form = {};
    void *some = cache ? cache->k : nullptr;   // (an aligned address; nothing is launched)
    const int rc = attention(who, rows->parent != nullptr, cache, 0, rows, some, n_heads, window, 0.f, some, nullptr, nullptr, 0,
                             &form);
    if (rc) return rc;
    plan[0] = form.rows;
    plan[1] = form.ctas;
    plan[2] = form.shares;
    return VOX_CUDA_OK;
}

extern "C" int vox_cuda_rope_append_dev(const vox_cuda_kv_cache *cache, int layer, const vox_cuda_rows *rows,
                                        const void *qkv, int qkv_type, int n_heads, long long qkv_stride,
                                        const float *q_norm, const float *k_norm, float eps, float theta, void *q_out,
                                        void *stream) {
    const char *who = "rope_append";
    AppendParams p = {};
    int rc = check_cache(who, cache, &p.c);
    if (rc || (rc = check_rows(who, rows, p.c.n_streams, p.c.ring, 1, &p.r)) ||
        (rc = check_layer(who, layer, p.c.n_layers)) || (rc = check_heads(who, n_heads, p.c.n_kv_heads)))
        return rc;
    if (qkv_type != ELEM_F32 && qkv_type != p.c.dtype) {
        set_error("%s: q|k|v must be fp32 or of the cache's type", who);
        return VOX_CUDA_ERR_ARG;
    }
    const int elem = elem_size(qkv_type), cell = elem_size(p.c.dtype);
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
    if (overlap(qkv, (double)ld * p.r.n_rows * elem, q_out, (double)p.r.n_rows * n_heads * p.c.head_dim * cell)) {
        set_error("%s: q_out must not overlap q|k|v", who);
        return VOX_CUDA_ERR_ARG;
    }
    DevCtx *c = cur_ctx();
    if (!c) return VOX_CUDA_ERR_UNAVAILABLE;
    DeviceGuard guard(c->device);
    if (!guard.ok()) return launched(who, cudaGetLastError());
    p.layer_off = (long long)layer * p.c.layer_stride;
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
    return launched(who, launch_rope_append(p, stream ? (cudaStream_t)stream : c->stream));
}

extern "C" int vox_cuda_kv_commit_dev(const vox_cuda_kv_cache *cache, const int *pos, const int *path, int path_stride,
                                      const int *n_accept, int max_accept, int *new_pos, void *stream) {
    const char *who = "kv_commit";
    CommitParams p = {};
    int rc = check_cache(who, cache, &p.c);
    if (rc) return rc;
    if (!pos || !path || !n_accept || max_accept < 1 || max_accept > kTreeMax || path_stride < max_accept) {
        set_error("%s: bad path (1 to %d rows of a stream, a stride of as many)", who, kTreeMax);
        return VOX_CUDA_ERR_ARG;
    }
    const double n = (double)p.c.n_streams * sizeof(int);
    if (overlap(new_pos, n, pos, n) || overlap(new_pos, n, n_accept, n) || overlap(new_pos, n, path, n * path_stride)) {
        set_error("%s: new_pos must not overlap pos, path or n_accept", who);
        return VOX_CUDA_ERR_ARG;
    }
    DevCtx *c = cur_ctx();
    if (!c) return VOX_CUDA_ERR_UNAVAILABLE;
    DeviceGuard guard(c->device);
    if (!guard.ok()) return launched(who, cudaGetLastError());
    p.pos = pos;
    p.path = path;
    p.path_ld = path_stride;
    p.n_accept = n_accept;
    p.max_accept = max_accept;
    p.new_pos = new_pos;
    return launched(who, launch_kv_commit(p, stream ? (cudaStream_t)stream : c->stream));
}

extern "C" int vox_cuda_kv_fork_dev(const vox_cuda_kv_cache *cache, const int *src, const int *dst, int n, const int *pos,
                                    void *stream) {
    const char *who = "kv_fork";
    ForkParams p = {};
    int rc = check_cache(who, cache, &p.c);
    if (rc) return rc;
    if (n < 0 || n > kForkMax || !pos || (n > 0 && (!src || !dst))) {
        set_error("%s: bad arguments (0 to %d pairs)", who, kForkMax);
        return VOX_CUDA_ERR_ARG;
    }
    for (int i = 0; i < n; i++) {
        if (src[i] < 0 || src[i] >= p.c.n_streams || dst[i] < 0 || dst[i] >= p.c.n_streams) {
            set_error("%s: pair %d (%d to %d) of %d streams", who, i, src[i], dst[i], p.c.n_streams);
            return VOX_CUDA_ERR_ARG;
        }
        for (int j = 0; j < n; j++)
            if (dst[i] == src[j] || (i != j && dst[i] == dst[j])) {
                set_error("%s: stream %d is written while another pair reads or writes it", who, dst[i]);
                return VOX_CUDA_ERR_ARG;
            }
        p.src[i] = (unsigned short)src[i];
        p.dst[i] = (unsigned short)dst[i];
    }
    if (n == 0) return VOX_CUDA_OK;
    DevCtx *c = cur_ctx();
    if (!c) return VOX_CUDA_ERR_UNAVAILABLE;
    DeviceGuard guard(c->device);
    if (!guard.ok()) return launched(who, cudaGetLastError());
    p.n = n;
    p.pos = pos;
    return launched(who, launch_kv_fork(p, c->sms, stream ? (cudaStream_t)stream : c->stream));
}

extern "C" int vox_cuda_token_logprobs_dev(const void *logits, int type, int n_rows, int vocab, long long row_stride,
                                           const int *tokens, int n_top, float *logprob, float *entropy, int *top_ids,
                                           float *top_logprob, void *stream) {
    const char *who = "token_logprobs";
    const long long ld = row_stride ? row_stride : vocab;
    if (!known_type(type) || n_rows < 0 || n_rows > (1 << 26) || vocab < 1 || vocab > kMaxPosition || ld < vocab ||
        ld > (1ll << 40)) {
        set_error("%s: bad logits (type %d, %d rows of %d, stride %lld)", who, type, n_rows, vocab, ld);
        return VOX_CUDA_ERR_ARG;
    }
    if (n_top < 0 || n_top > kTopMax || n_top > vocab || (n_top > 0 && !top_ids) || (n_top == 0 && top_logprob)) {
        set_error("%s: 0 to %d alternatives, with a place for their ids (not %d)", who, kTopMax, n_top);
        return VOX_CUDA_ERR_ARG;
    }
    if ((logprob != nullptr) != (tokens != nullptr)) {
        set_error("%s: tokens and logprob go together", who);
        return VOX_CUDA_ERR_ARG;
    }
    if (n_rows == 0) return VOX_CUDA_OK;
    if (!logits || ((uintptr_t)logits % elem_size(type)) != 0 || (!logprob && !entropy && n_top == 0)) {
        set_error("%s: no logits, or nothing asked for", who);
        return VOX_CUDA_ERR_ARG;
    }
    DevCtx *c = cur_ctx();
    if (!c) return VOX_CUDA_ERR_UNAVAILABLE;
    DeviceGuard guard(c->device);
    if (!guard.ok()) return launched(who, cudaGetLastError());
    LogprobParams p = {};
    p.logits = logits;
    p.dtype = type;
    p.n_rows = n_rows;
    p.vocab = vocab;
    p.ld = ld;
    p.tokens = tokens;
    p.n_top = n_top;
    p.logprob = logprob;
    p.entropy = entropy;
    p.top_ids = top_ids;
    p.top_logprob = top_logprob;
    return launched(who, launch_token_logprobs(p, c->sms, stream ? (cudaStream_t)stream : c->stream));
}
