// vc_paged_cache.cu - a paged cache's own operators: rotary append with the
// rounding to e4m3, copies of pages.
#include "vc_paged.cuh"

#include <algorithm>

namespace vc {

namespace {

// ---------------------------------------------------------------------------
// Rotary append.  A CTA has the rows of one (page of a stream, KV head): their
// K and V head and the group's q heads, so that the largest value of the page's
// new K (or V) is found in the CTA and nothing is read twice.  q and k are
// normalised (x / sqrt(mean(x^2) + eps) * g, if g is given) and rotated in
// interleaved pairs, (a, b) -> (a cos - b sin, a sin + b cos): the angle in
// turns in fp64, its fraction to sincospi in fp32, once per row for the K and q
// heads.  Then the scale 2^e that puts the maximum under 448, the earlier slots
// of the page again where it grew, and the new ones.
// ---------------------------------------------------------------------------

constexpr int kPaThreads = 256;
constexpr int kLeastExp = -100;   // of a scale

// 2^e with e the smallest whole number >= kLeastExp and a <= 448 * 2^e; a >= 0, finite
__device__ __forceinline__ float scale_for(float a) {
    const uint32_t bits = __float_as_uint(a);   // a = 1.m * 2^x: 448 = 1.75 * 2^8
    const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u);
    return __uint_as_float((uint32_t)(max(e, kLeastExp) + 127) << 23);
}

__device__ __forceinline__ float finite_abs(float x) {
    const float a = fabsf(x);
    return a < INFINITY ? a : 0.f;
}

// RPT: rows of a page that a thread takes, its lanes hold 8 values of each
template <typename TS, typename TQ, int HD, int RPT>
__global__ void __launch_bounds__(kPaThreads) paged_append_kernel(const PagedAppendParams p) {
    constexpr int LH = HD / 8;                    // lanes of a head
    constexpr int kSlots = kPaThreads / LH;       // rows of a step
    __shared__ float most_s[kPaThreads / 32];
    const int kvh = blockIdx.y, stream = blockIdx.z, P = p.c.page;
    const RowSpan s = paged_span(p.r, p.c, stream);
    const int index = (s.pos >> p.c.page_shift) + blockIdx.x;   // of the page
    const int j0 = max(s.pos, index * P), j1 = min(s.pos + s.n, (index + 1) * P);
    if (s.n == 0 || j0 >= j1) return;
    const int page = page_at(p.c, stream, index);
    const int sub = threadIdx.x % LH, r0 = threadIdx.x / LH;
    double turn[4];   // turns of the lane's four pairs per position
#pragma unroll
    for (int e = 0; e < 4; e++)
        turn[e] = p.rotate ? exp2(-2.0 * (sub * 4 + e) / HD * p.log2_theta) * 0.15915494309189535 : 0.0;

    auto load = [&](int j, int head, float (&x)[8]) {
        const TS *src = static_cast<const TS *>(p.qkv) + (s.r0 + j - s.pos) * p.ld + (long long)head * HD + sub * 8;
        const float4 a = load4<TS>(src), b = load4<TS>(src + 4);
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
        x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    };
    auto norm = [&](float (&x)[8], const float *g) {   // whole warps: shuffles among the head's lanes
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; e += 2) ss += x[e] * x[e] + x[e + 1] * x[e + 1];
#pragma unroll
        for (int o = LH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float r = rsqrtf(ss * (1.0f / HD) + p.eps);
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] *= r * __ldg(g + sub * 8 + e);
    };
    // the CTA's maximum, the page's scale, the earlier slots, the new ones
    auto store = [&](const float (&x)[RPT][8], unsigned char *pool, float *scales) {
        float most = 0.f;
#pragma unroll
        for (int i = 0; i < RPT; i++)
#pragma unroll
            for (int e = 0; e < 8; e++) most = fmaxf(most, finite_abs(x[i][e]));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        __syncthreads();
        if (threadIdx.x % 32 == 0) most_s[threadIdx.x / 32] = most;
        __syncthreads();
        if (page < 0) return;
#pragma unroll
        for (int w = 0; w < kPaThreads / 32; w++) most = fmaxf(most, most_s[w]);
        float *const at = scales + scale_at(p.c, p.layer, page, kvh);
        const int lo = j0 & (P - 1);
        const float was = lo ? *at : 0.f, need = scale_for(most);
        const bool keep = lo > 0 && was >= need && was < INFINITY;
        const float now = keep ? was : need, inv = 1.0f / now;
        unsigned char *const base = pool + page_base(p.c, p.layer, page, kvh);
        if (!keep) {
            const float ratio = was * inv;
            for (int e = threadIdx.x; e < lo * (HD / 4); e += kPaThreads) {
                uint32_t *w = reinterpret_cast<uint32_t *>(base + e / (HD / 4) * p.c.slot_stride + e % (HD / 4) * 4);
                const float4 v = from_e4m3x4(*w);
                *w = to_e4m3x4(make_float4(v.x * ratio, v.y * ratio, v.z * ratio, v.w * ratio));
            }
        }
#pragma unroll
        for (int i = 0; i < RPT; i++) {
            const int j = j0 + r0 + i * kSlots;
            if (j < j1)
                *reinterpret_cast<uint2 *>(base + (j & (P - 1)) * p.c.slot_stride + sub * 8) =
                    make_uint2(to_e4m3x4(make_float4(x[i][0] * inv, x[i][1] * inv, x[i][2] * inv, x[i][3] * inv)),
                               to_e4m3x4(make_float4(x[i][4] * inv, x[i][5] * inv, x[i][6] * inv, x[i][7] * inv)));
        }
        __syncthreads();   // (all have read the scale)
        if (threadIdx.x == 0 && !keep) *at = now;
    };

    float x[RPT][8];
#pragma unroll
    for (int i = 0; i < RPT; i++) {
        const int j = j0 + r0 + i * kSlots;
        float c[4], sn[4], y[8];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const double t = (double)j * turn[e];
            sincospif(2.f * (float)(t - rint(t)), &sn[e], &c[e]);
        }
        auto rotate = [&](float (&v)[8]) {
            if (!p.rotate) return;   // (0 times an infinity would be NaN)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float a = v[2 * e], b = v[2 * e + 1];
                v[2 * e] = a * c[e] - b * sn[e];
                v[2 * e + 1] = a * sn[e] + b * c[e];
            }
        };
        for (int h = 0; h < p.group; h++) {
            const int head = kvh * p.group + h;
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] = 0.f;
            if (j < j1) load(j, head, y);
            if (p.q_norm) norm(y, p.q_norm);
            rotate(y);
            if (j < j1)
                *reinterpret_cast<uint4 *>(static_cast<TQ *>(p.q_out) + ((long long)(s.r0 + j - s.pos) * p.n_heads + head) * HD +
                                           sub * 8) =
                    make_uint4(pack2<TQ>(y[0], y[1]), pack2<TQ>(y[2], y[3]), pack2<TQ>(y[4], y[5]), pack2<TQ>(y[6], y[7]));
        }
#pragma unroll
        for (int e = 0; e < 8; e++) x[i][e] = 0.f;
        if (j < j1) load(j, p.n_heads + kvh, x[i]);
        if (p.k_norm) norm(x[i], p.k_norm);
        rotate(x[i]);
    }
    store(x, p.c.k, p.c.k_scale);
#pragma unroll
    for (int i = 0; i < RPT; i++) {
        const int j = j0 + r0 + i * kSlots;
#pragma unroll
        for (int e = 0; e < 8; e++) x[i][e] = 0.f;
        if (j < j1) load(j, p.n_heads + p.c.n_kv_heads + kvh, x[i]);
    }
    store(x, p.c.v, p.c.v_scale);
}

// ---------------------------------------------------------------------------
// Copies of pages: a CTA has one pair of one layer, K or V of some heads, or
// the scales.  Bound by HBM.
// ---------------------------------------------------------------------------

constexpr int kPcThreads = 256;
constexpr int kPcLoads = 4;

__global__ void __launch_bounds__(kPcThreads) paged_copy_kernel(const PagedCopyParams p) {
    const int layer = blockIdx.y >> 1, per_row = p.c.head_dim / 16;
    const bool is_v = blockIdx.y & 1;
    for (int i = blockIdx.z; i < p.n; i += gridDim.z) {
        const int src = __ldg(p.src + i), dst = __ldg(p.dst + i);
        if (src < 0 || src >= p.c.n_pages || dst < 0 || dst >= p.c.n_pages) continue;
        unsigned char *const base = is_v ? p.c.v : p.c.k;
        float *const scales = is_v ? p.c.v_scale : p.c.k_scale;
        const unsigned char *const from = base + page_base(p.c, layer, src, 0);
        unsigned char *const to = base + page_base(p.c, layer, dst, 0);
        const int n = p.c.n_kv_heads * p.c.page * per_row, step = gridDim.x * kPcThreads;
        for (int e0 = blockIdx.x * kPcThreads + threadIdx.x; e0 < n; e0 += step * kPcLoads) {
            uint4 v[kPcLoads];
            long long off[kPcLoads];
#pragma unroll
            for (int b = 0; b < kPcLoads; b++) {
                const int e = e0 + b * step, row = e / per_row;
                off[b] = (row >> p.c.page_shift) * p.c.head_stride + (row & (p.c.page - 1)) * p.c.slot_stride + e % per_row * 16;
                if (e < n) v[b] = *reinterpret_cast<const uint4 *>(from + off[b]);
            }
#pragma unroll
            for (int b = 0; b < kPcLoads; b++)
                if (e0 + b * step < n) *reinterpret_cast<uint4 *>(to + off[b]) = v[b];
        }
        if (blockIdx.x == 0)
            for (int h = threadIdx.x; h < p.c.n_kv_heads; h += kPcThreads)
                scales[scale_at(p.c, layer, dst, h)] = scales[scale_at(p.c, layer, src, h)];
    }
}

template <typename TS, typename TQ, int HD, int RPT>
cudaError_t append_rows(const PagedAppendParams &p, cudaStream_t st) {
    // the pages that max_rows positions can touch, wherever they begin
    const dim3 grid((p.r.max_rows + p.c.page - 2) / p.c.page + 1, p.c.n_kv_heads, p.c.n_streams);
    paged_append_kernel<TS, TQ, HD, RPT><<<grid, kPaThreads, 0, st>>>(p);
    return cudaGetLastError();
}
template <typename TS, typename TQ, int HD>
cudaError_t append_dim(const PagedAppendParams &p, cudaStream_t st) {
    constexpr int kSlots = kPaThreads / (HD / 8);
    const int rows = std::min(p.r.max_rows, p.c.page), per = (rows + kSlots - 1) / kSlots;
    if (per <= 1) return append_rows<TS, TQ, HD, 1>(p, st);
    if (per <= 2) return append_rows<TS, TQ, HD, 2>(p, st);
    if (per <= 4) return append_rows<TS, TQ, HD, 4>(p, st);
    if constexpr (HD == 128) return append_rows<TS, TQ, HD, 8>(p, st);
    return cudaErrorInvalidValue;   // (heads of 64: 32 rows a step, pages of 128 at most)
}
template <typename TS, typename TQ>
cudaError_t append_typed(const PagedAppendParams &p, cudaStream_t st) {
    return p.c.head_dim == 64 ? append_dim<TS, TQ, 64>(p, st) : append_dim<TS, TQ, 128>(p, st);
}

}  // namespace

cudaError_t launch_paged_append(const PagedAppendParams &p, cudaStream_t st) {
    if (p.q_type == ELEM_BF16)
        return p.src_type == ELEM_F32 ? append_typed<float, __nv_bfloat16>(p, st)
                                      : append_typed<__nv_bfloat16, __nv_bfloat16>(p, st);
    return p.src_type == ELEM_F32 ? append_typed<float, __half>(p, st) : append_typed<__half, __half>(p, st);
}

cudaError_t launch_paged_copy(const PagedCopyParams &p, int sms, cudaStream_t st) {
    const long long chunks = (long long)p.c.n_kv_heads * p.c.page * (p.c.head_dim / 16);
    const long long most = (chunks + kPcThreads * kPcLoads - 1) / (kPcThreads * kPcLoads);
    const long long rest = (long long)p.c.n_layers * 2 * p.n;   // blocks of the other axes
    const long long x = std::max<long long>(1, std::min(most, (16ll * sms + rest - 1) / rest));
    paged_copy_kernel<<<dim3((unsigned)x, p.c.n_layers * 2, std::min(p.n, 65535)), kPcThreads, 0, st>>>(p);
    return cudaGetLastError();
}

}  // namespace vc
