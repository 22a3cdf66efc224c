// vc_paged_cache.cu - a paged cache's own operators: rotary append with the
// rounding to e4m3, copies of pages.
#include "vc_paged.cuh"

#include <algorithm>

namespace vc {

namespace {

// ---------------------------------------------------------------------------
// Rotary append, two kinds of CTA in one launch, each reading its part once:
//   K and V  the rows of one (page of a stream, KV head), so that the largest
//            value of the page's new K, and of its V, is found in the CTA: both
//            heads' rows are loaded before anything is done with them, then comes
//            the scale 2^e that puts the maximum under 448, the earlier slots of the
//            page again where it grew, and the new ones
//   q        some rows' q heads, which need no scale and share their rows' angles
// q and k are normalised (x / sqrt(mean(x^2) + eps) * g, if g is given) and rotated
// in interleaved pairs, (a, b) -> (a cos - b sin, a sin + b cos): the angle in quarter
// turns in fp64 (a far position times a frequency keeps its fraction only there).  A
// head is HD / 8 lanes with 8 values each.
//
// Bound by HBM for long chunks, by the launch and three dependent reads (position,
// page, keys) for a step.  4 streams of up to 1021 rows of 32 / 8 heads of 128, fp32 to
// bf16: 29.5 us, 0.63 of the copy rate (issue 54% busy); an encoder chunk of 1500 rows
// of 32 / 32 heads of 64, fp16: 16 us, 0.29 (issue 65% busy); one token of 8 streams
// 3.1 us on the device.  All heads of a page and KV head in one kind of CTA, as their
// angles ask for, took 33 and 18 us: few loads at a time.
// ---------------------------------------------------------------------------

constexpr int kLeastExp = -100;   // of a scale

// 2^e with e the smallest whole number >= kLeastExp and a <= 448 * 2^e; a >= 0, finite
__device__ __forceinline__ float scale_for(float a) {
    const uint32_t bits = __float_as_uint(a);   // a = 1.m * 2^x: 448 = 1.75 * 2^8
    const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u);
    return __uint_as_float((uint32_t)(max(e, kLeastExp) + 127) << 23);
}

// The largest |x| of a thread's values: infinity if one is, NaN passed over.
template <int N>
__device__ __forceinline__ float largest(const float (&x)[N], float most) {
#pragma unroll
    for (int e = 0; e < N; e++) most = fmaxf(most, fabsf(x[e]));
    return most;
}
// The same without the infinities.
template <int N>
__device__ __forceinline__ float largest_finite(const float (&x)[N], float most) {
#pragma unroll
    for (int e = 0; e < N; e++) most = fmaxf(most, fabsf(x[e]) < INFINITY ? fabsf(x[e]) : 0.f);
    return most;
}

// Quarter turns per position of pair d of a head, in fp64.
__device__ __forceinline__ double quarters_of(const PagedAppendParams &p, int d, int hd) {
    return p.rotate ? exp2(-2.0 * d / hd * p.log2_theta) * 0.6366197723675814 : 0.0;
}
// Cosine and sine of an angle in quarter turns, 2^-23.7 off at most over a million
// angles: what is left of the nearest whole number, r in [-1/2, 1/2], is taken in fp64
// and kept in two parts; sin(pi r / 2) / r and cos(pi r / 2) are minimax polynomials
// in r^2 (own Remez fits, 2^-27 and 2^-34), pi / 2 in two parts, and what goes to a
// leading term is added last.  An angle that is 2^-21 off (the hardware's sine; 2 us
// faster for the encoder chunk) rounds a key in a million to the other neighbour.
__device__ __forceinline__ float2 cos_sin(double quarters) {
    const double whole = rint(quarters), rest = quarters - whole;
    const int n = (int)(long long)whole;
    const float r = (float)rest, lo = (float)(rest - (double)r), u = r * r;
    const float q = fmaf(fmaf(fmaf(0.000903631677f, u, -0.0208600722f), u, 0.253669202f), u, -1.23370051f);
    const float c = 1.0f + fmaf(q, u, r * lo * -2.46740110f);
    const float t = fmaf(fmaf(fmaf(-0.00460217707f, u, 0.0796802267f), u, -0.64596349f), u, -4.37113883e-8f);
    const float s = fmaf(r, 1.57079637f, fmaf(c * 1.57079637f, lo, r * t));
    const float a = n & 1 ? s : c, b = n & 1 ? c : s;   // the angle's cosine and sine but for their signs
    return make_float2(__uint_as_float(__float_as_uint(a) ^ ((uint32_t)(n + 1) << 30 & 0x80000000u)),
                       __uint_as_float(__float_as_uint(b) ^ ((uint32_t)n << 30 & 0x80000000u)));
}

template <typename TS>
struct Eight {   // 8 values as they come
    static constexpr int kWords = sizeof(TS) / 2;
    uint4 w[kWords];
    __device__ __forceinline__ void load(const TS *p, bool ok) {
#pragma unroll
        for (int i = 0; i < kWords; i++) w[i] = ok ? *reinterpret_cast<const uint4 *>(p + i * 4 * (4 / sizeof(TS))) : make_uint4(0u, 0u, 0u, 0u);
    }
    __device__ __forceinline__ void values(float (&x)[8]) const {
        if constexpr (sizeof(TS) == 4) {
            const uint32_t v[8] = {w[0].x, w[0].y, w[0].z, w[0].w, w[1].x, w[1].y, w[1].z, w[1].w};
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = __uint_as_float(v[e]);
        } else {
            const uint32_t v[4] = {w[0].x, w[0].y, w[0].z, w[0].w};
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float2 f = unpack2<TS>(v[e]);
                x[2 * e] = f.x;
                x[2 * e + 1] = f.y;
            }
        }
    }
};

// A lane's weights of a norm.
__device__ __forceinline__ void load_weights(float (&w)[8], const float *g, int sub) {
    const float4 a = __ldg(reinterpret_cast<const float4 *>(g + sub * 8)), b = __ldg(reinterpret_cast<const float4 *>(g + sub * 8 + 4));
    w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
    w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
}
// Whole warps: shuffles among the head's lanes.
template <int HD>
__device__ __forceinline__ void normalise(float (&x)[8], const float (&w)[8], float eps) {
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; e += 2) ss += x[e] * x[e] + x[e + 1] * x[e + 1];
#pragma unroll
    for (int o = HD / 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float r = rsqrtf(ss * (1.0f / HD) + eps);
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] *= r * w[e];
}
__device__ __forceinline__ void rotate8(float (&x)[8], const float2 (&c)[4]) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const float a = x[2 * e], b = x[2 * e + 1];
        x[2 * e] = __fsub_rn(__fmul_rn(a, c[e].x), __fmul_rn(b, c[e].y));   // rounded as written: a key's e4m3 does not
        x[2 * e + 1] = __fadd_rn(__fmul_rn(a, c[e].y), __fmul_rn(b, c[e].x));   // depend on what was contracted
    }
}

template <int HD, int NT>
struct AppendSmem {
    double turn[HD / 2];              // quarter turns per position
    float2 cs[2 * NT / HD][HD / 2];   // q: cosines and sines of its rows
    float most[2][NT / 32];
};

// K and V of one page and head; RPT: rows of a page that a thread takes
template <typename TS, int HD, int RPT, int NT>
__device__ __forceinline__ void append_kv(const PagedAppendParams &p, AppendSmem<HD, NT> &sh, const RowSpan &s, int stream, int nth, int kvh) {
    constexpr int LH = HD / 8, kSlots = NT / LH;   // lanes of a head, rows of a step
    const int P = p.c.page, index = (s.pos >> p.c.page_shift) + nth;   // of the page
    const int j0 = max(s.pos, index * P), j1 = min(s.pos + s.n, (index + 1) * P);
    if (s.n == 0 || j0 >= j1) return;
    const int sub = threadIdx.x % LH, r0 = threadIdx.x / LH;
    Eight<TS> raw[2][RPT];   // on their way under the page's look-up
#pragma unroll
    for (int i = 0; i < RPT; i++) {
        const int j = j0 + r0 + i * kSlots;
        const TS *src = static_cast<const TS *>(p.qkv) + (s.r0 + j - s.pos) * p.ld + (long long)(p.n_heads + kvh) * HD + sub * 8;
        raw[0][i].load(src, j < j1);
        raw[1][i].load(src + (long long)p.c.n_kv_heads * HD, j < j1);
    }
    const int page = page_at(p.c, stream, index);
    if (page < 0) return;
    float *const at[2] = {p.c.k_scale + scale_at(p.c, p.layer, page, kvh), p.c.v_scale + scale_at(p.c, p.layer, page, kvh)};
    const int lo = j0 & (P - 1);
    const float was[2] = {lo ? *at[0] : 0.f, lo ? *at[1] : 0.f};
    if (threadIdx.x < HD / 2) sh.turn[threadIdx.x] = quarters_of(p, threadIdx.x, HD);
    __syncthreads();
    float x[RPT][8], most[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < RPT; i++) {
        raw[0][i].values(x[i]);
        if (p.k_norm) {
            float weight[8];
            load_weights(weight, p.k_norm, sub);
            normalise<HD>(x[i], weight, p.eps);
        }
        if (p.rotate) {   // (0 times an infinity would be NaN)
            float2 c[4];
#pragma unroll
            for (int e = 0; e < 4; e++) c[e] = cos_sin((double)(j0 + r0 + i * kSlots) * sh.turn[sub * 4 + e]);
            rotate8(x[i], c);
        }
        float v[8];
        raw[1][i].values(v);
        most[0] = largest(x[i], most[0]);
        most[1] = largest(v, most[1]);
    }
    // infinities are looked for where there is one: they count for nothing, and become NaN
    const bool inf[2] = {most[0] == INFINITY, most[1] == INFINITY};
    if (inf[0] || inf[1]) {
        most[0] = most[1] = 0.f;
#pragma unroll
        for (int i = 0; i < RPT; i++) {
            float v[8];
            raw[1][i].values(v);
            most[0] = largest_finite(x[i], most[0]);
            most[1] = largest_finite(v, most[1]);
        }
    }
#pragma unroll
    for (int w = 0; w < 2; w++) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) most[w] = fmaxf(most[w], __shfl_xor_sync(0xffffffffu, most[w], o));
        if (threadIdx.x % 32 == 0) sh.most[w][threadIdx.x / 32] = most[w];
    }
    __syncthreads();   // (all have read the scales, too)
    const long long base = page_base(p.c, p.layer, page, kvh);
#pragma unroll
    for (int w = 0; w < 2; w++) {
#pragma unroll
        for (int o = 0; o < NT / 32; o++) most[w] = fmaxf(most[w], sh.most[w][o]);
        const float need = scale_for(most[w]);
        const bool keep = lo > 0 && was[w] >= need && was[w] < INFINITY;
        const float now = keep ? was[w] : need, inv = 1.0f / now;
        unsigned char *const to = (w ? p.c.v : p.c.k) + base;
        if (!keep) {
            const float ratio = was[w] * inv;
            for (int e = threadIdx.x; e < lo * (HD / 16); e += NT) {
                uint4 *at16 = reinterpret_cast<uint4 *>(to + e / (HD / 16) * p.c.slot_stride + e % (HD / 16) * 16);
                const uint4 u = *at16;
                auto again = [&](uint32_t four) {
                    const float4 f = from_e4m3x4(four);
                    return to_e4m3x4(make_float4(f.x * ratio, f.y * ratio, f.z * ratio, f.w * ratio));
                };
                *at16 = make_uint4(again(u.x), again(u.y), again(u.z), again(u.w));
            }
            if (threadIdx.x == 0) *at[w] = now;
        }
#pragma unroll
        for (int i = 0; i < RPT; i++) {
            const int j = j0 + r0 + i * kSlots;
            float v[8];
            if (w) raw[1][i].values(v);
            else {
#pragma unroll
                for (int e = 0; e < 8; e++) v[e] = x[i][e];
            }
            if (inf[w])
#pragma unroll
                for (int e = 0; e < 8; e++) v[e] = fabsf(v[e]) < INFINITY ? v[e] : NAN;
            if (j < j1)
                *reinterpret_cast<uint2 *>(to + (j & (P - 1)) * p.c.slot_stride + sub * 8) =
                    make_uint2(to_e4m3x4(make_float4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv)),
                               to_e4m3x4(make_float4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv)));
        }
    }
}

// The q heads of rows [i0, i0 + R): every split-th group of heads from `part` on
template <typename TS, typename TQ, int HD, int NT>
__device__ __forceinline__ void append_q(const PagedAppendParams &p, AppendSmem<HD, NT> &sh, const RowSpan &s, int i0, int R, int part, int split) {
    constexpr int LH = HD / 8, kAtOnce = NT / LH;   // heads of a step
    const int rows = min(R, s.n - i0);
    if (rows <= 0) return;
    const int sub = threadIdx.x % LH, h0 = threadIdx.x / LH;
    // a group of heads of a row after the other; the next two are on their way
    // while one is worked on
    const int first = part * kAtOnce + h0, step = split * kAtOnce;
    struct Item {
        int row, head;   // the thread's
        __device__ bool next(int heads, int first, int step) {   // whether the row is done: by groups, so that a warp stays together
            head += step;
            const bool done = head / kAtOnce * kAtOnce >= heads;
            if (done) {
                head = first;
                row++;
            }
            return done;
        }
    };
    Eight<TS> raw[2];
    const TS *row_src = static_cast<const TS *>(p.qkv) + (long long)(s.r0 + i0) * p.ld + sub * 8;
    TQ *row_dst = static_cast<TQ *>(p.q_out) + (long long)(s.r0 + i0) * p.n_heads * HD + sub * 8;
    Item at = {0, first}, ahead = at;
    auto fetch = [&](Eight<TS> &to) {
        to.load(row_src + ahead.head * HD, ahead.row < rows && ahead.head < p.n_heads);
        if (ahead.next(p.n_heads, first, step)) row_src += p.ld;
    };
    float weight[8];
    if (p.q_norm) load_weights(weight, p.q_norm, sub);
    fetch(raw[0]);
    fetch(raw[1]);
    if (p.rotate) {
        if (threadIdx.x < HD / 2) sh.turn[threadIdx.x] = quarters_of(p, threadIdx.x, HD);
        __syncthreads();
        for (int e = threadIdx.x; e < rows * (HD / 2); e += NT)
            sh.cs[e / (HD / 2)][e % (HD / 2)] = cos_sin((double)(s.pos + i0 + e / (HD / 2)) * sh.turn[e % (HD / 2)]);
        __syncthreads();
    }
    while (at.row < rows) {   // (the same for all lanes of a head, and of a warp)
        float x[8];
        raw[0].values(x);
        raw[0] = raw[1];
        fetch(raw[1]);
        if (p.q_norm) normalise<HD>(x, weight, p.eps);
        if (p.rotate) {
            const float4 a = *reinterpret_cast<const float4 *>(&sh.cs[at.row][sub * 4]), b = *reinterpret_cast<const float4 *>(&sh.cs[at.row][sub * 4 + 2]);
            const float2 c[4] = {make_float2(a.x, a.y), make_float2(a.z, a.w), make_float2(b.x, b.y), make_float2(b.z, b.w)};
            rotate8(x, c);
        }
        if (at.head < p.n_heads)
            *reinterpret_cast<uint4 *>(row_dst + at.head * HD) =
                make_uint4(pack2<TQ>(x[0], x[1]), pack2<TQ>(x[2], x[3]), pack2<TQ>(x[4], x[5]), pack2<TQ>(x[6], x[7]));
        if (at.next(p.n_heads, first, step)) row_dst += (long long)p.n_heads * HD;
    }
}

// A stream's CTAs: x page of y < n_kv_heads, the KV head; those behind, in turn, its
// rows' q by R rows and `split` CTAs.
template <typename TS, typename TQ, int HD, int RPT, int NT>
__global__ void __launch_bounds__(NT, 1024 / NT) paged_append_kernel(const PagedAppendParams p, int R, int split) {
    __shared__ __align__(16) AppendSmem<HD, NT> sh;
    const int stream = blockIdx.z, over = blockIdx.y - p.c.n_kv_heads;
    const RowSpan s = paged_span(p.r, p.c, stream);
    if (over < 0) {
        append_kv<TS, HD, RPT, NT>(p, sh, s, stream, blockIdx.x, blockIdx.y);
    } else {
        const int i = over * gridDim.x + blockIdx.x, of = split == 1 ? i : i / split;   // (its rows end before 2^30)
        append_q<TS, TQ, HD, NT>(p, sh, s, of * R, R, i - of * split, split);
    }
}

// ---------------------------------------------------------------------------
// Copies of pages: a CTA has one pair of one layer, K or V: some of its 16-byte
// chunks, four in flight per thread, and the scales.  Bound by HBM: 1.75 GB moved 267
// us, 1.0 of the copy rate; 55 MB 9.9, 0.84.
// ---------------------------------------------------------------------------

constexpr int kPcThreads = 256;
constexpr int kPcLoads = 4;

__global__ void __launch_bounds__(kPcThreads) paged_copy_kernel(const PagedCopyParams p) {
    const int layer = blockIdx.y >> 1, row_shift = p.c.head_dim == 64 ? 2 : 3;   // 16-byte chunks of a row
    const bool is_v = blockIdx.y & 1;
    for (int i = blockIdx.z; i < p.n; i += gridDim.z) {
        const int src = __ldg(p.src + i), dst = __ldg(p.dst + i);
        if (src < 0 || src >= p.c.n_pages || dst < 0 || dst >= p.c.n_pages) continue;
        unsigned char *const base = is_v ? p.c.v : p.c.k;
        float *const scales = is_v ? p.c.v_scale : p.c.k_scale;
        const unsigned char *const from = base + page_base(p.c, layer, src, 0);
        unsigned char *const to = base + page_base(p.c, layer, dst, 0);
        const int n = p.c.n_kv_heads * p.c.page << row_shift, step = gridDim.x * kPcThreads;
        for (int e0 = blockIdx.x * kPcThreads + threadIdx.x; e0 < n; e0 += step * kPcLoads) {
            uint4 v[kPcLoads];
            long long off[kPcLoads];
#pragma unroll
            for (int b = 0; b < kPcLoads; b++) {
                const int e = e0 + b * step, row = e >> row_shift;
                off[b] = (row >> p.c.page_shift) * p.c.head_stride + (row & (p.c.page - 1)) * p.c.slot_stride + (e & ((1 << row_shift) - 1)) * 16;
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

template <typename TS, typename TQ, int HD, int RPT, int NT>
cudaError_t append_rows(const PagedAppendParams &p, cudaStream_t st) {
    // the pages that max_rows positions can touch, wherever they begin
    const int pages = (p.r.max_rows + p.c.page - 2) / p.c.page + 1;
    // q: few rows: a CTA per group of heads; from 512 on, a few CTAs to an SM, a row;
    // many: several, up to as many as a CTA has threads for their angles
    constexpr int kAtOnce = NT / (HD / 8);
    const long long rows = (long long)p.r.max_rows * p.c.n_streams;
    const int R = (int)std::max(1ll, std::min(2ll * NT / HD, rows / 512)), split = rows < 512 ? std::min(64, (p.n_heads + kAtOnce - 1) / kAtOnce) : 1;
    const long long q = ((p.r.max_rows + R - 1ll) / R) * split, y = p.c.n_kv_heads + (q + pages - 1) / pages;   // < 4096 + 64 * 128
    paged_append_kernel<TS, TQ, HD, RPT, NT><<<dim3(pages, (unsigned)y, p.c.n_streams), NT, 0, st>>>(p, R, split);
    return cudaGetLastError();
}
// As many threads as give each two rows of a page at most, so that 64 registers do
// and an SM holds 32 warps.
template <typename TS, typename TQ, int HD>
cudaError_t append_dim(const PagedAppendParams &p, cudaStream_t st) {
    const int lanes = std::min(p.r.max_rows, p.c.page) * (HD / 8);
    if (lanes <= 256) return append_rows<TS, TQ, HD, 1, 256>(p, st);
    if (lanes <= 512) return append_rows<TS, TQ, HD, 2, 256>(p, st);
    if (lanes <= 1024) return append_rows<TS, TQ, HD, 2, 512>(p, st);
    if constexpr (HD == 128) return append_rows<TS, TQ, HD, 2, 1024>(p, st);
    return cudaErrorInvalidValue;   // (pages of 128 at most)
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
