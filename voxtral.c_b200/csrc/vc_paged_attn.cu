// vc_paged_attn.cu - attention of a call's rows over a paged cache in 8 bits.
#include "vc_paged.cuh"

namespace vc {

namespace {

// A CTA has one row and the query heads of a KV head, a warp every fourth key:
// a lane holds HD / 32 dims of q, K and V, and the running maximum, sum and
// output of its warp's keys, which the CTA joins at the end.
constexpr int kPtWarps = 4;

template <typename T, int HD>
__global__ void __launch_bounds__(kPtWarps * 32) paged_attn_kernel(const PagedAttnParams p) {
    constexpr int D = HD / 32;
    __shared__ float o_s[kPtWarps][HD], m_s[kPtWarps], l_s[kPtWarps];
    const int i = blockIdx.x, kvh = blockIdx.y, stream = blockIdx.z, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const RowSpan s = paged_span(p.r, p.c, stream);
    if (i >= s.n) return;
    const int at = s.pos + i, low = p.window > 0 ? max(0, at - p.window + 1) : 0;
    for (int h = kvh * p.group; h < (kvh + 1) * p.group; h++) {
        const long long line = (long long)(s.r0 + i) * p.n_heads + h;
        float q[D], o[D], m = -INFINITY, l = 0.f;
#pragma unroll
        for (int d = 0; d < D; d++) {
            q[d] = (float)static_cast<const T *>(p.q)[line * HD + lane * D + d] * p.scale_log2;
            o[d] = 0.f;
        }
        for (int j = warp; j <= at; j += kPtWarps) {
            if (j >= p.n_sink && j < low) continue;
            const int page = page_at(p.c, stream, j >> p.c.page_shift);
            if (page < 0) continue;
            const long long sc = scale_at(p.c, p.layer, page, kvh);
            const long long off = page_base(p.c, p.layer, page, kvh) + (j & (p.c.page - 1)) * p.c.slot_stride + lane * D;
            float x = 0.f, v[D];
#pragma unroll
            for (int d = 0; d < D; d += 2) {
                const float2 kk = __half22float2(from_e4m3x2(*reinterpret_cast<const uint16_t *>(p.c.k + off + d)));
                const float2 vv = __half22float2(from_e4m3x2(*reinterpret_cast<const uint16_t *>(p.c.v + off + d)));
                x += q[d] * kk.x + q[d + 1] * kk.y;
                v[d] = vv.x;
                v[d + 1] = vv.y;
            }
            x = warp_sum(x) * p.c.k_scale[sc];
            const float mn = fmaxf(m, x), base = mn == -INFINITY ? 0.f : mn;
            const float f = exp2f(m - base), w = exp2f(x - base), vs = p.c.v_scale[sc];
            m = mn;
            l = l * f + w;
#pragma unroll
            for (int d = 0; d < D; d++) o[d] = o[d] * f + w * vs * v[d];
        }
        __syncthreads();
#pragma unroll
        for (int d = 0; d < D; d++) o_s[warp][lane * D + d] = o[d];
        if (lane == 0) {
            m_s[warp] = m;
            l_s[warp] = l;
        }
        __syncthreads();
        float gm = -INFINITY, gl = 0.f;
        for (int w = 0; w < kPtWarps; w++) gm = fmaxf(gm, m_s[w]);
        const float base = gm == -INFINITY ? 0.f : gm;
        for (int w = 0; w < kPtWarps; w++) gl += l_s[w] * exp2f(m_s[w] - base);
        for (int d = threadIdx.x; d < HD; d += kPtWarps * 32) {
            float a = 0.f;
            for (int w = 0; w < kPtWarps; w++) a += o_s[w][d] * exp2f(m_s[w] - base);
            static_cast<T *>(p.out)[line * HD + d] = (T)(gl == 0.f ? 0.f : a / gl);
        }
        if (p.lse && threadIdx.x == 0) p.lse[line] = gl == 0.f ? -INFINITY : (gm + log2f(gl)) * 0.69314718055994531f;
    }
}

template <typename T>
cudaError_t attn_typed(const PagedAttnParams &p, cudaStream_t st) {
    const dim3 grid(p.r.max_rows, p.c.n_kv_heads, p.c.n_streams);
    if (p.c.head_dim == 64) paged_attn_kernel<T, 64><<<grid, kPtWarps * 32, 0, st>>>(p);
    else paged_attn_kernel<T, 128><<<grid, kPtWarps * 32, 0, st>>>(p);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_paged_attn(const PagedAttnParams &p, cudaStream_t st) {
    return p.q_type == ELEM_BF16 ? attn_typed<__nv_bfloat16>(p, st) : attn_typed<__half>(p, st);
}

}  // namespace vc
