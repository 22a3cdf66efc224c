// vc_logprobs.cu - log probabilities of given tokens, the entropy and the top
// alternatives of rows of logits.
//
//   log p_t = x_t - m - ln Z          Z = sum_i e^(x_i - m)
//   H       = ln Z - S / Z            S = sum_i e^(x_i - m) (x_i - m)
//
// One pass over a row: each thread keeps a running maximum with Z and S in
// fp32, rescaled when a batch of its values raises the maximum.  A row with a
// NaN or +inf, or without a finite logit, has no distribution: NaN.  Bound by HBM
// for many rows, by latency for one: a row is shared by the CTAs of a cluster
// when there are fewer rows than SMs.
//
// The alternatives cost no second pass: the threads also leave each batch's
// maximum in shared memory.  The n_top-th largest of 32 group maxima is a
// value that at least n_top logits reach, so only batches that reach it -
// about n_top of them - are looked at again; their values go into a sorted
// list that a warp holds across its lanes.  Lists order by value, then by the
// lowest id, and merge by rank.
#include "vc_rows.cuh"
#include "vc_tc.cuh"

#include <algorithm>
#include <atomic>
#include <float.h>

namespace vc {

using namespace tc;

namespace {

constexpr int kLpThreads = 256;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpLoads = 4;      // 16-byte loads of a thread's batch
constexpr int kLpSlots = 16;     // batch maxima kept per thread; batch b in slot b % 16
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLpFloor = -200.f;   // x - m below this: e^(x - m) is 0 in fp32

// A logit and its id as one number: larger is better, ties go to the lower id.
typedef unsigned long long Key;
__device__ __forceinline__ Key make_key(float x, int id) {
    const uint32_t b = __float_as_uint(x + 0.0f);   // -0 and +0 are equal
    const uint32_t o = b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
    return ((Key)o << 32) | (uint32_t)(0x7fffffff - id);
}
__device__ __forceinline__ float key_value(Key k) {
    const uint32_t o = (uint32_t)(k >> 32);
    return __uint_as_float((o & 0x80000000u) ? o ^ 0x80000000u : ~o);
}
__device__ __forceinline__ int key_id(Key k) { return 0x7fffffff - (int)(uint32_t)k; }

struct LpSmem {
    float batch_max[kLpSlots][kLpThreads];
    Key lists[kLpWarps][kTopMax];   // the warps' best, then (list 0) the CTA's
    Key merged[kTopMax];
    float group_max[32];
    float red[kLpWarps][4];
    float stat[4];                  // the CTA's (m, top, rest, S)
    float floor;                    // n_top logits of the CTA's share reach this
};

// A thread's vectors of a row: 16-byte vectors from the first aligned
// element, the unaligned head as vector -1, the rest as the last one.
template <typename T>
struct RowView {
    static constexpr int V = 16 / (int)sizeof(T);
    const T *x;
    int head, full, vocab;   // head elements, whole vectors, all elements
    __device__ RowView(const T *row, int n) : x(row), vocab(n) {
        head = (int)((16u - ((uint32_t)(uintptr_t)row & 15u)) & 15u) / (int)sizeof(T);
        head = min(head, n);
        full = (n - head) / V;
    }
    // vectors -1 .. full; element 0 of vector v
    __device__ int first(int v) const { return v < 0 ? 0 : head + v * V; }
    __device__ int count(int v) const { return v < 0 ? head : v < full ? V : vocab - head - full * V; }
    __device__ void get(int v, float (&f)[V]) const {
        if (v >= 0 && v < full) {
            const uint4 u = __ldg(reinterpret_cast<const uint4 *>(x + head) + v);
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
            if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int i = 0; i < 4; i++) f[i] = __uint_as_float(w[i]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float2 a = unpack2<T>(w[i]);
                    f[2 * i] = a.x;
                    f[2 * i + 1] = a.y;
                }
            }
        } else {
            const int n = count(v), b = first(v);
#pragma unroll
            for (int i = 0; i < V; i++) f[i] = i < n ? (float)x[b + i] : -INFINITY;   // adds nothing
        }
    }
};

// the larger value, or NaN if either is
__device__ __forceinline__ float fmax_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Adds a second part (m2, ...) of a row to the first.
__device__ __forceinline__ void fold(float &m, float &top, float &rest, float &mom, float m2, float top2, float rest2,
                                     float mom2) {
    if (m2 == m) {
        top += top2;
        rest += rest2;
        mom += mom2;
        return;
    }
    const bool up = m2 > m;   // the second part's maximum is the larger: it keeps its top
    const float d = fmax_nan(up ? m - m2 : m2 - m, kLpFloor), w = exp2_approx(d * kLog2e);
    const float low = up ? rest + top : rest2 + top2, low_mom = up ? mom : mom2;
    mom = (up ? mom2 : mom) + w * fmaf(low, d, low_mom);
    rest = (up ? rest2 : rest) + w * low;
    if (up) {
        top = top2;
        m = m2;
    }
}

// Puts a key into the list that the warp's lanes hold in descending order.
__device__ __forceinline__ void list_insert(Key &mine, Key k, int lane) {
    const int at = __popc(__ballot_sync(0xffffffffu, mine > k));
    const Key up = __shfl_up_sync(0xffffffffu, mine, 1);
    if (lane == at) mine = k;
    else if (lane > at) mine = up;
}

// How many of a descending list's keys are better than k.
__device__ __forceinline__ int better(const Key *list, int n, Key k) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (list[mid] > k) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

template <typename T>
__global__ void __launch_bounds__(kLpThreads) token_logprobs_kernel(const LogprobParams p, int Z) {
    using R = RowView<T>;
    constexpr int V = R::V;
    __shared__ LpSmem sh;
    __shared__ Key all[16 * kTopMax];   // rank 0: the cluster's lists
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row = blockIdx.x / Z, z = blockIdx.x % Z;
    const R x(static_cast<const T *>(p.logits) + (long long)row * p.ld, p.vocab);
    // this CTA's vectors, of -1 .. full
    const int nv = x.full + 2;
    const int v0 = (int)((long long)z * nv / Z) - 1, v1 = (int)((long long)(z + 1) * nv / Z) - 1;
    const int K = p.n_top;

    // Z = top + rest: `top` counts the logits equal to m, the others' e^(x - m)
    // add up apart from it, so that a confident row's ln Z and H keep their
    // leading digits (ln Z = log1p(rest)).
    float m = -FLT_MAX, top = 0.f, rest = 0.f, mom = 0.f, best = -INFINITY;
    for (int s = 0; s < kLpSlots; s++) sh.batch_max[s][threadIdx.x] = -INFINITY;
    int b = 0;
    for (int vb = v0; vb < v1; vb += kLpThreads * kLpLoads, b++) {
        float f[kLpLoads][V];
#pragma unroll
        for (int u = 0; u < kLpLoads; u++) {
            const int v = vb + u * kLpThreads + threadIdx.x;
            if (v < v1) x.get(v, f[u]);
            else {
#pragma unroll
                for (int i = 0; i < V; i++) f[u][i] = -INFINITY;
            }
        }
        float bm = -INFINITY;
#pragma unroll
        for (int u = 0; u < kLpLoads; u++)
#pragma unroll
            for (int i = 0; i < V; i++) bm = fmaxf(bm, f[u][i]);
        if (K > 0) {
            float &slot = sh.batch_max[b % kLpSlots][threadIdx.x];
            slot = fmaxf(slot, bm);
            best = fmaxf(best, bm);
        }
        if (bm > m) {
            const float d = fmax_nan(m - bm, kLpFloor), w = exp2_approx(d * kLog2e);
            rest += top;
            mom = w * fmaf(rest, d, mom);
            rest *= w;
            top = 0.f;
            m = bm;
        }
        if (bm == m) {
#pragma unroll
            for (int u = 0; u < kLpLoads; u++)
#pragma unroll
                for (int i = 0; i < V; i++) top += f[u][i] == m ? 1.f : 0.f;
        }
#pragma unroll
        for (int u = 0; u < kLpLoads; u++)
#pragma unroll
            for (int i = 0; i < V; i++) {
                const float d = fmax_nan(f[u][i] - m, kLpFloor), e = exp2_approx(d * kLog2e);
                if (!(d == 0.f)) rest += e;
                mom = fmaf(e, d, mom);
            }
    }

    // the CTA's (m, top, rest, S)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        fold(m, top, rest, mom, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, top, o),
             __shfl_xor_sync(0xffffffffu, rest, o), __shfl_xor_sync(0xffffffffu, mom, o));
    if (lane == 0) {
        sh.red[warp][0] = m;
        sh.red[warp][1] = top;
        sh.red[warp][2] = rest;
        sh.red[warp][3] = mom;
    }
    if (K > 0) {
        float g = best;
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, o));
        if ((lane & 7) == 0) sh.group_max[warp * 4 + lane / 8] = g;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kLpWarps; w++)
            fold(m, top, rest, mom, sh.red[w][0], sh.red[w][1], sh.red[w][2], sh.red[w][3]);
        sh.stat[0] = m;
        sh.stat[1] = top;
        sh.stat[2] = rest;
        sh.stat[3] = mom;
    }
    if (K > 0) {
        if (warp == 1) {   // the K-th largest group maximum: K - 1 others are at least as large
            const float g = sh.group_max[lane];
            int rank = 0;
            for (int o = 0; o < 32; o++) {
                const float h = __shfl_sync(0xffffffffu, g, o);
                rank += h > g || (h == g && o < lane);
            }
            if (rank == K - 1) sh.floor = g;
        }
        __syncthreads();
        const float floor = sh.floor;
        Key mine = 0;   // lane i: the warp's i-th best
        for (int s = 0; s < kLpSlots; s++) {
            bool hit = sh.batch_max[s][threadIdx.x] >= floor;
            if (!__any_sync(0xffffffffu, hit)) continue;
            for (int vb = v0 + s * kLpThreads * kLpLoads; vb < v1; vb += kLpSlots * kLpThreads * kLpLoads) {
                float f[kLpLoads][V];
#pragma unroll
                for (int u = 0; u < kLpLoads; u++) {
                    const int v = vb + u * kLpThreads + threadIdx.x;
                    if (hit && v < v1) x.get(v, f[u]);
                    else {
#pragma unroll
                        for (int i = 0; i < V; i++) f[u][i] = -INFINITY;
                    }
                }
#pragma unroll
                for (int u = 0; u < kLpLoads; u++) {
                    const int v = vb + u * kLpThreads + threadIdx.x;
                    const int id0 = x.first(v), n = hit && v < v1 ? x.count(v) : 0;
#pragma unroll
                    for (int i = 0; i < V; i++) {
                        bool cand = i < n && f[u][i] >= floor;
                        if (!__any_sync(0xffffffffu, cand)) continue;
                        const Key k = make_key(f[u][i], id0 + i);
                        for (;;) {
                            const Key last = __shfl_sync(0xffffffffu, mine, K - 1);
                            const unsigned todo = __ballot_sync(0xffffffffu, cand && k > last);
                            if (!todo) break;
                            const int from = __ffs(todo) - 1;
                            list_insert(mine, __shfl_sync(0xffffffffu, k, from), lane);
                            if (lane == from) cand = false;
                        }
                    }
                }
            }
        }
        sh.lists[warp][lane] = lane < K ? mine : 0;
        __syncthreads();
        if (threadIdx.x < kTopMax) sh.merged[threadIdx.x] = 0;
        __syncthreads();
        if (lane < K && mine != 0) {   // the rank of each key among the 8 lists
            int rank = 0;
            for (int w = 0; w < kLpWarps; w++) rank += better(sh.lists[w], K, mine);
            if (rank < K) sh.merged[rank] = mine;
        }
    }
    if (Z > 1) cluster_sync_all();
    else __syncthreads();

    if (z == 0) {
        // the cluster's (m, top, rest, S), in every thread
        float gm = sh.stat[0], gn = sh.stat[1], gr = sh.stat[2], gt = sh.stat[3];
        for (int r = 1; r < Z; r++) {
            const uint32_t a = mapa_shared(smem_u32(sh.stat), r);
            fold(gm, gn, gr, gt, ld_dsmem_f1(a), ld_dsmem_f1(a + 4), ld_dsmem_f1(a + 8), ld_dsmem_f1(a + 12));
        }
        const float lz = gn == 1.f ? log1pf(gr) : logf(gn + gr);
        if (threadIdx.x == 0) {
            if (p.logprob) {
                const int tok = p.tokens ? __ldg(p.tokens + row) : -1;
                // a row without a finite logit has no distribution: NaN
                p.logprob[row] = tok >= 0 && tok < p.vocab ? ((float)x.x[tok] - gm) - lz : NAN;
            }
            if (p.entropy) p.entropy[row] = lz - gt / (gn + gr);
        }
        if (K > 0) {
            const Key *lists = sh.merged;
            if (Z > 1) {
                for (int e = threadIdx.x; e < Z * kTopMax; e += kLpThreads) {
                    const uint32_t a = mapa_shared(smem_u32(sh.merged + e % kTopMax), e / kTopMax);
                    const float2 v = ld_dsmem_f2(a);
                    all[e] = ((Key)__float_as_uint(v.y) << 32) | __float_as_uint(v.x);
                }
                __syncthreads();
                lists = all;
            }
            if (threadIdx.x < K) {   // NaN logits are no alternatives: places that nothing fills
                int found = 0;
                for (int r = 0; r < Z; r++) found += better(lists + r * kTopMax, K, 0);
                if (threadIdx.x >= found) {
                    p.top_ids[(long long)row * K + threadIdx.x] = -1;
                    if (p.top_logprob) p.top_logprob[(long long)row * K + threadIdx.x] = NAN;
                }
            }
            for (int e = threadIdx.x; e < Z * kTopMax; e += kLpThreads) {
                const Key k = lists[e];
                if (k == 0) continue;
                int rank = 0;
                for (int r = 0; r < Z; r++) rank += better(lists + r * kTopMax, K, k);
                if (rank < K) {
                    p.top_ids[(long long)row * K + rank] = key_id(k);
                    if (p.top_logprob) p.top_logprob[(long long)row * K + rank] = (key_value(k) - gm) - lz;
                }
            }
        }
    }
    if (Z > 1) cluster_sync_all();   // no CTA leaves while rank 0 still reads its share
}

template <typename T>
cudaError_t launch_typed(const LogprobParams &p, int Z, cudaStream_t st) {
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (!(done.load() & bit)) {
        e = cudaFuncSetAttribute(token_logprobs_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
        done.fetch_or(bit);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(p.n_rows * Z));
    cfg.blockDim = dim3(kLpThreads);
    cfg.stream = st;
    cudaLaunchAttribute a[1];
    a[0].id = cudaLaunchAttributeClusterDimension;
    a[0].val.clusterDim.x = Z;
    a[0].val.clusterDim.y = 1;
    a[0].val.clusterDim.z = 1;
    cfg.attrs = a;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T>, p, Z);
}

}  // namespace

cudaError_t launch_token_logprobs(const LogprobParams &p, int sms, cudaStream_t st) {
    // shares of a row: as many as fill the SMs twice, each with a batch of
    // work for its threads, at most a cluster's 16
    const int elem = p.dtype == ELEM_F32 ? 4 : 2;
    const long long batch = (long long)kLpThreads * 16 / elem;
    const long long by_work = std::max<long long>(1, p.vocab / batch);
    const long long by_sms = std::max<long long>(1, 2ll * sms / p.n_rows);
    const int Z = (int)std::min<long long>(16, std::min(by_work, by_sms));
    switch (p.dtype) {
        case ELEM_F32: return launch_typed<float>(p, Z, st);
        case ELEM_BF16: return launch_typed<__nv_bfloat16>(p, Z, st);
        default: return launch_typed<__half>(p, Z, st);
    }
}

}  // namespace vc
