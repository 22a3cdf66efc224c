// vc_cache.cu - a cache slab's own operators: rotary append (with the
// optional norm of each query and key head), commit of an accepted path,
// fork of a stream.
#include "vc_rows.cuh"

#include <algorithm>

namespace vc {

namespace {

// ---------------------------------------------------------------------------
// Rotary append: one row's q | k | v heads are read once; q and k are
// normalised (x / sqrt(mean(x^2) + eps) * g, if g is given) and rotated in
// interleaved pairs, (a, b) -> (a cos - b sin, a sin + b cos), q goes to
// q_out, k and v to the row's cache slot.
//
// Bound by HBM for long chunks, by launch latency for a step.  The row's
// cosines and sines are computed once, by one thread per pair: the angle in
// turns in fp64 (a far position times a frequency keeps its fraction only
// there), its fraction to sincospi in fp32; the first heads are on their way
// meanwhile, each later group while the one before is worked on.  A head is
// HD / 8 lanes with 8 values each, so the shuffles of a norm serve two or four
// heads.  4 streams of up to 1021 rows of 48 heads of 128, fp32 to bf16: 24.9 us, 0.80 of the
// copy rate (lanes of 4 values, no load ahead: 28.7; of 8: 26.6).
// ---------------------------------------------------------------------------

constexpr int kApThreads = 256;

template <typename TS, typename TC, int HD>
__global__ void __launch_bounds__(kApThreads) rope_append_kernel(const AppendParams p) {
    __shared__ float2 cs[HD / 2];
    __shared__ short parent[kTreeMax];
    __shared__ int depth_s;
    const int i = blockIdx.x, stream = blockIdx.z;
    const RowSpan s = row_span(p.r, stream);
    if (i >= s.n) return;
    int at = s.pos + i;
    if (p.r.parent) {
        load_parents(parent, p.r, s, threadIdx.x, kApThreads);
        __syncthreads();
        if (threadIdx.x == 0) {
            int d = -1;
            for (int a = i; a >= 0; a = parent[a]) d++;
            depth_s = d;
        }
        __syncthreads();
        at = s.pos + depth_s;
    }
    constexpr int LH = HD / 8;   // lanes of a head
    const int sub = threadIdx.x % LH, d[2] = {sub * 4, HD / 2 + sub * 4};
    const long long row = s.r0 + i;
    const TS *src = static_cast<const TS *>(p.qkv) + row * p.ld;
    const int n = p.n_heads + 2 * p.c.n_kv_heads;
    constexpr int kAtOnce = kApThreads / LH;   // heads per block and step
    float4 next[2] = {};   // the first heads are on their way under the angles
    auto load = [&](int h) {
        if (h < n)
#pragma unroll
            for (int e = 0; e < 2; e++) next[e] = load4<TS>(src + h * HD + d[e]);
    };
    load(blockIdx.y * kAtOnce + threadIdx.x / LH);
    if (threadIdx.x < HD / 2) {
        float2 v = make_float2(1.f, 0.f);
        if (p.rotate) {
            const double turns = (double)at * exp2(-2.0 * threadIdx.x / HD * p.log2_theta) * 0.15915494309189535;
            sincospif(2.f * (float)(turns - rint(turns)), &v.y, &v.x);
        }
        cs[threadIdx.x] = v;
    }
    __syncthreads();

    const float2 c[2][2] = {{cs[sub * 2], cs[sub * 2 + 1]}, {cs[HD / 4 + sub * 2], cs[HD / 4 + sub * 2 + 1]}};
    TC *q = static_cast<TC *>(p.q_out) + row * p.n_heads * HD;
    const long long slot = p.layer_off + (long long)stream * p.c.stream_stride +
                           (long long)cache_slot(p.c, s.pos + i) * p.c.slot_stride;
    TC *k = reinterpret_cast<TC *>(p.c.k) + slot, *v = reinterpret_cast<TC *>(p.c.v) + slot;
    // whole warps stay in the loop: the norm's shuffles cover every lane
    for (int h0 = blockIdx.y * kAtOnce; h0 < n; h0 += gridDim.y * kAtOnce) {
        const int h = h0 + threadIdx.x / LH;
        float4 x[2] = {next[0], next[1]};
        load(h + gridDim.y * kAtOnce);
        const bool is_q = h < p.n_heads, is_v = h >= p.n_heads + p.c.n_kv_heads;
        const float *g = is_q ? p.q_norm : is_v ? nullptr : p.k_norm;
        if (p.q_norm || p.k_norm) {
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < 2; e++) ss += (x[e].x * x[e].x + x[e].y * x[e].y) + (x[e].z * x[e].z + x[e].w * x[e].w);
#pragma unroll
            for (int o = LH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            if (g) {
                const float r = rsqrtf(ss * (1.0f / HD) + p.eps);
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const float4 gv = __ldg(reinterpret_cast<const float4 *>(g + d[e]));
                    x[e] = make_float4(x[e].x * r * gv.x, x[e].y * r * gv.y, x[e].z * r * gv.z, x[e].w * r * gv.w);
                }
            }
        }
        if (h >= n) continue;
        if (!is_v)
#pragma unroll
            for (int e = 0; e < 2; e++)
                x[e] = make_float4(x[e].x * c[e][0].x - x[e].y * c[e][0].y, x[e].x * c[e][0].y + x[e].y * c[e][0].x,
                                   x[e].z * c[e][1].x - x[e].w * c[e][1].y, x[e].z * c[e][1].y + x[e].w * c[e][1].x);
        TC *const to = is_q ? q + h * HD
                            : is_v ? v + (long long)(h - p.n_heads - p.c.n_kv_heads) * p.c.head_stride
                                   : k + (long long)(h - p.n_heads) * p.c.head_stride;
#pragma unroll
        for (int e = 0; e < 2; e++) store4<TC>(to + d[e], x[e]);
    }
}

// ---------------------------------------------------------------------------
// Commit: the rows at positions pos + path[k] move to pos + k, for every
// layer.  path[k] >= k and the path ascends, so a thread that moves its 16
// bytes of every row in the order of k never overwrites a row it still has to
// read: a batch's targets lie below every later source.  A few MB at most:
// bound by latency, so a batch of 8 rows is read before it is written.  5 rows
// of 8 streams, 26 layers of 8 heads of 128, fp32 (14 MB moved): 6.1 us.
// ---------------------------------------------------------------------------

constexpr int kCmThreads = 128;
constexpr int kCmBatch = 8;

__global__ void __launch_bounds__(kCmThreads) kv_commit_kernel(const CommitParams p, int elem, int chunks) {
    __shared__ int path[kTreeMax];
    __shared__ int count;
    const int layer = blockIdx.x, stream = blockIdx.y;
    const int pos = __ldg(p.pos + stream);
    const bool out = pos < 0 || pos > kMaxPosition;   // the stream sits out
    const int want = out ? 0 : min(max(__ldg(p.n_accept + stream), 0), p.max_accept);
    for (int k = threadIdx.x; k < want; k += kCmThreads) path[k] = __ldg(p.path + (long long)stream * p.path_ld + k);
    __syncthreads();
    if (threadIdx.x == 0) {
        // the path ends before the first entry that does not ascend or that no tree holds
        int n = 0, last = -1;
        while (n < want && path[n] > last && path[n] < min(kTreeMax, p.c.ring)) last = path[n++];
        count = n;
        if (p.new_pos && layer == 0 && blockIdx.z == 0) p.new_pos[stream] = pos + n;
    }
    __syncthreads();
    const int n = count;
    const int e = blockIdx.z * kCmThreads + threadIdx.x;   // 16-byte chunk of K's row, then of V's
    if (e >= 2 * chunks) return;
    char *base = e < chunks ? p.c.k : p.c.v;
    const int ch = e < chunks ? e : e - chunks;
    const int per_head = p.c.head_dim * elem / 16;
    base += (cache_base(p.c, layer, stream) + (long long)(ch / per_head) * p.c.head_stride) * elem + ch % per_head * 16;
    const long long slot_bytes = p.c.slot_stride * elem;
    for (int k0 = 0; k0 < n; k0 += kCmBatch) {
        uint4 v[kCmBatch];
#pragma unroll
        for (int b = 0; b < kCmBatch; b++)
            if (k0 + b < n && path[k0 + b] != k0 + b)
                v[b] = *reinterpret_cast<const uint4 *>(base + cache_slot(p.c, pos + path[k0 + b]) * slot_bytes);
#pragma unroll
        for (int b = 0; b < kCmBatch; b++)
            if (k0 + b < n && path[k0 + b] != k0 + b)
                *reinterpret_cast<uint4 *>(base + cache_slot(p.c, pos + k0 + b) * slot_bytes) = v[b];
    }
}

// ---------------------------------------------------------------------------
// Fork: the slots that a stream uses - its first pos, or all of them - copied
// to another stream, for every layer.  Bound by HBM: 16-byte loads, four in
// flight per thread.  1.75 GB moved: 290 us, 0.93 of the copy rate.
// ---------------------------------------------------------------------------

constexpr int kFkThreads = 256;
constexpr int kFkLoads = 4;

__global__ void __launch_bounds__(kFkThreads) kv_fork_kernel(const ForkParams p, int elem, int chunks) {
    const int pair = blockIdx.z, src = p.src[pair], dst = p.dst[pair];
    const int pos = __ldg(p.pos + src);
    if (pos < 0 || pos > kMaxPosition) return;
    const int layer = blockIdx.y >> 1;
    char *base = (blockIdx.y & 1) ? p.c.v : p.c.k;
    const char *from = base + cache_base(p.c, layer, src) * elem;
    char *to = base + cache_base(p.c, layer, dst) * elem;
    const int per_head = p.c.head_dim * elem / 16;
    const long long slot_bytes = p.c.slot_stride * elem, head_bytes = p.c.head_stride * elem;
    const long long n = (long long)min(pos, p.c.cap) * chunks;
    const long long step = (long long)gridDim.x * kFkThreads;
    for (long long e0 = (long long)blockIdx.x * kFkThreads + threadIdx.x; e0 < n; e0 += step * kFkLoads) {
        uint4 v[kFkLoads];
        long long off[kFkLoads];
#pragma unroll
        for (int b = 0; b < kFkLoads; b++) {
            const long long e = e0 + b * step;
            const long long slot = e / chunks;
            const int ch = (int)(e - slot * chunks);
            off[b] = slot * slot_bytes + ch / per_head * head_bytes + ch % per_head * 16;
            if (e < n) v[b] = *reinterpret_cast<const uint4 *>(from + off[b]);
        }
#pragma unroll
        for (int b = 0; b < kFkLoads; b++)
            if (e0 + b * step < n) *reinterpret_cast<uint4 *>(to + off[b]) = v[b];
    }
}

template <typename TS, typename TC>
cudaError_t append_typed(const AppendParams &p, cudaStream_t st) {
    const int hd = p.c.head_dim, at_once = kApThreads / (hd / 8);
    const int steps = (p.n_heads + 2 * p.c.n_kv_heads + at_once - 1) / at_once;
    // few rows: a block per group of heads (a step of 8 rows: 5.2 us, launch
    // bound); from 512 on, which fill the SMs' 8 blocks half, a block per row,
    // so that its cosines and sines serve every head
    const long long rows = (long long)p.r.max_rows * p.c.n_streams;
    const int split = (int)(rows >= 512 ? 1 : steps);
    const dim3 grid(p.r.max_rows, split, p.c.n_streams);
    if (hd == 64) rope_append_kernel<TS, TC, 64><<<grid, kApThreads, 0, st>>>(p);
    else rope_append_kernel<TS, TC, 128><<<grid, kApThreads, 0, st>>>(p);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_rope_append(const AppendParams &p, cudaStream_t st) {
    if (p.src_type == ELEM_F32) {
        if (p.c.dtype == ELEM_F32) return append_typed<float, float>(p, st);
        if (p.c.dtype == ELEM_BF16) return append_typed<float, __nv_bfloat16>(p, st);
        return append_typed<float, __half>(p, st);
    }
    if (p.c.dtype == ELEM_BF16) return append_typed<__nv_bfloat16, __nv_bfloat16>(p, st);
    return append_typed<__half, __half>(p, st);
}

cudaError_t launch_kv_commit(const CommitParams &p, cudaStream_t st) {
    const int elem = p.c.dtype == ELEM_F32 ? 4 : 2;
    const int chunks = p.c.n_kv_heads * p.c.head_dim * elem / 16;
    const dim3 grid(p.c.n_layers, p.c.n_streams, (2 * chunks + kCmThreads - 1) / kCmThreads);
    kv_commit_kernel<<<grid, kCmThreads, 0, st>>>(p, elem, chunks);
    return cudaGetLastError();
}

cudaError_t launch_kv_fork(const ForkParams &p, int sms, cudaStream_t st) {
    const int elem = p.c.dtype == ELEM_F32 ? 4 : 2;
    const int chunks = p.c.n_kv_heads * p.c.head_dim * elem / 16;
    const long long most = ((long long)p.c.cap * chunks + kFkThreads * kFkLoads - 1) / (kFkThreads * kFkLoads);
    const long long rest = (long long)p.c.n_layers * 2 * p.n;   // blocks of the other axes
    const long long x = std::max<long long>(1, std::min(most, (16ll * sms + rest - 1) / rest));
    kv_fork_kernel<<<dim3((unsigned)x, p.c.n_layers * 2, p.n), kFkThreads, 0, st>>>(p, elem, chunks);
    return cudaGetLastError();
}

}  // namespace vc
