// vc_logprobs.cu - log probabilities of given tokens, the entropy and the top
// alternatives of rows of logits.
//
//   log p_t = x_t - m - ln Z          Z = sum_i e^(x_i - m)
//   H       = ln Z - S / Z            S = sum_i e^(x_i - m) (x_i - m)
//
// One pass over a row: each warp keeps a running maximum, its threads Z and S in
// fp32, rescaled when a batch of values raises the maximum.  Per value about 5
// instructions, pairs of values where one does for two, and one exponential.  A row with a
// NaN or +inf, or without a finite logit, has no distribution: NaN.  Bound by HBM
// for many rows, by latency for one: a row is shared by the CTAs of a cluster
// when there are fewer rows than SMs.
//
// The alternatives cost no second pass: the threads also leave each batch's
// maximum in shared memory.  The n_top-th largest of 64 group maxima is a
// value that at least n_top logits reach, so only batches that reach it -
// 1 to 1.5 n_top of them - are looked at again, and their few values that reach it
// are ranked by counting.  Keys order by value, then by the lowest id; the
// shares of a row rank their lists against each other's.
#include "vc_rows.cuh"
#include "vc_tc.cuh"

#include <algorithm>
#include <atomic>
#include <math.h>
#include <type_traits>

namespace vc {

using namespace tc;

namespace {

// Threads of a CTA: 256 up to a row per SM, where a row is shared by CTAs and
// latency counts; 128 beyond, a row to a CTA, seven to an SM, and one row's end
// hides under the others.  There each thread copies its next batch into shared
// memory of its own while it works on this one (bf16, 131072 logits, 20
// alternatives, of 1001 rows: 76 -> 68 us; without alternatives 66 -> 57, of
// 4000 rows 235 -> 177, 0.92 of the copy rate; two batches ahead with six CTAs
// on an SM: 76).
constexpr int kLpFew = 256, kLpMany = 128;
constexpr int kLpCtas = 7;       // CTAs of kLpMany threads on an SM
constexpr int kLpLoads = 4;      // 16-byte loads of a thread's batch
constexpr int kLpAhead = 1;      // batches that a thread has on their way (many rows)
constexpr int kLpKept = 8192;    // bytes of batch maxima kept, batch b of a thread in slot b % slots.  As many bytes in
                                 // either size of type: with 16 KB of fp32 maxima only five CTAs fit an SM (1001
                                 // rows of 131072 fp32 logits, 20 alternatives 138 -> 119 us, 4000 rows 363 -> 353)
constexpr int kLpFound = 256;    // candidates, and batches with some, kept
constexpr int kLpShares = 16;    // CTAs of a row at most
constexpr int kLpGroups = 64;    // groups of threads whose maxima give the floor
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLpFloor = -300.f;   // 2^x below this is 0 in fp32

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

template <typename T, int NTH>
struct LpSmem {
    static constexpr int kWarps = NTH / 32, kSlots = kLpKept / (int)sizeof(T) / NTH;
    static constexpr bool kAhead = NTH == kLpMany;
    uint4 ahead[kAhead ? kLpAhead + 1 : 1][kAhead ? kLpLoads : 1][kAhead ? NTH : 1];   // batches on their way, each thread's own
    T batch_max[kSlots][NTH];
    Key found[kLpFound];            // candidates, in any order
    Key lists[kWarps][kTopMax];   // the warps' best, where `found` overflowed
    Key merged[kTopMax];            // the CTA's best
    float group_max[kLpGroups];
    float red[kWarps][4];
    float stat[5];                  // the CTA's (m, top, rest, S) and its largest logit
    float floor;                    // n_top logits of the CTA's share reach this
    int hit[kLpFound], hits;        // batches with candidates: batch * NTH + thread
    int count;                      // candidates
};
struct LpCluster {                  // what the shares of a row show each other
    Key lists[kLpShares][kTopMax];
    float stat[kLpShares][5];
    int rank[kTopMax];
};

// 16 bytes of T as they lie in memory.  The exponentials take values of at
// least kLowest: e^(x - m) is 0 there, and 0 times a finite distance adds
// nothing to S.
template <typename T>
struct Raw {
    static constexpr int V = 8;
    static constexpr bool kBf = std::is_same<T, __nv_bfloat16>::value;
    static constexpr uint32_t kNone = kBf ? 0xff80ff80u : 0xfc00fc00u;     // -inf
    static constexpr uint32_t kLowest2 = kBf ? 0xfe96fe96u : 0xfbfffbffu;  // -1e38, or fp16's lowest
    static __device__ float lowest() { return unpack2<T>(kLowest2).x; }
    // the largest value, NaN left aside
    static __device__ __forceinline__ void raise(uint32_t (&m)[2], uint4 u) {
        m[0] = max2(max2(m[0], u.x), u.z);
        m[1] = max2(max2(m[1], u.y), u.w);
    }
    static __device__ __forceinline__ float largest(const uint32_t (&m)[2]) {
        const float2 v = unpack2<T>(max2(m[0], m[1]));
        return fmaxf(v.x, v.y);
    }
    static __device__ __forceinline__ float2 pair_of(uint4 u, int i) {   // pair i of 4, raised to kLowest, NaN kept
        const uint32_t w = i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w;
        uint32_t r;
        if (kBf) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(w), "r"(kLowest2));
        else asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(w), "r"(kLowest2));
        return unpack2<T>(r);
    }
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
        uint32_t r;
        if (kBf) asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        else asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ void values(uint4 u, float (&f)[V]) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 a = unpack2<T>(w[i]);
            f[2 * i] = a.x;
            f[2 * i + 1] = a.y;
        }
    }
};
template <>
struct Raw<float> {
    static constexpr int V = 4;
    static constexpr uint32_t kNone = 0xff800000u;
    static __device__ float lowest() { return -1e38f; }
    static __device__ __forceinline__ void raise(uint32_t (&m)[2], uint4 u) {
        const float a = fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), __uint_as_float(m[0]));
        const float b = fmaxf(fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)), __uint_as_float(m[1]));
        m[0] = __float_as_uint(a);
        m[1] = __float_as_uint(b);
    }
    static __device__ __forceinline__ float largest(const uint32_t (&m)[2]) {
        return fmaxf(__uint_as_float(m[0]), __uint_as_float(m[1]));
    }
    static __device__ __forceinline__ float2 pair_of(uint4 u, int i) {
        const float a = __uint_as_float(i == 0 ? u.x : u.z), b = __uint_as_float(i == 0 ? u.y : u.w);
        return make_float2(fmax_nan(a, -1e38f), fmax_nan(b, -1e38f));
    }
    static __device__ void values(uint4 u, float (&f)[V]) {
        f[0] = __uint_as_float(u.x);
        f[1] = __uint_as_float(u.y);
        f[2] = __uint_as_float(u.z);
        f[3] = __uint_as_float(u.w);
    }
};

// A row as vectors: 16-byte vectors from the first aligned element, the
// unaligned head as vector -1, the rest as the last one (`full`).
template <typename T>
struct RowView {
    static constexpr int V = Raw<T>::V;
    const T *x;
    int head, full, vocab;   // head elements, whole vectors, all elements
    __device__ RowView(const T *row, int n) : x(row), vocab(n) {
        head = (int)((16u - ((uint32_t)(uintptr_t)row & 15u)) & 15u) / (int)sizeof(T);
        head = min(head, n);
        full = (n - head) / V;
    }
    // element 0 of vector v and its elements, -1 <= v <= full
    __device__ int first(int v) const { return v < 0 ? 0 : head + v * V; }
    __device__ int count(int v) const { return v < 0 ? head : v < full ? V : vocab - head - full * V; }
    __device__ __forceinline__ uint4 whole(int v) const { return __ldg(reinterpret_cast<const uint4 *>(x + head) + v); }
    // vector v, -inf past its end
    __device__ uint4 any(int v) const {
        if (v >= 0 && v < full) return whole(v);
        union {
            T e[V];
            uint4 u;
        } r;
        const uint32_t none = Raw<T>::kNone;
        r.u = make_uint4(none, none, none, none);
        const int n = count(v), b = first(v);
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i < n) r.e[i] = x[b + i];
        return r.u;
    }
};

// the warp's largest value, NaN left aside
__device__ __forceinline__ float warp_max(float v) {
    float r;
    asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}

// Adds a second part (m2, ...) of a row to the first.  S is kept in log2
// units: the sum of e^(x - m) (x - m) log2(e).
__device__ __forceinline__ void fold(float &m, float &top, float &rest, float &mom, float m2, float top2, float rest2,
                                     float mom2) {
    if (m2 == m) {
        top += top2;
        rest += rest2;
        mom += mom2;
        return;
    }
    const bool up = m2 > m;   // the second part's maximum is the larger: it keeps its top
    const float d = fmax_nan((up ? m - m2 : m2 - m) * kLog2e, kLpFloor), w = exp2_approx(d);
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

// fold() over the lanes' parts (NULL: none) of a power of two of lanes.
__device__ __forceinline__ void fold_lanes(const float *part, int n, float &m, float &top, float &rest, float &mom) {
    m = part ? part[0] : -INFINITY;
    top = part ? part[1] : 0.f;
    rest = part ? part[2] : 0.f;
    mom = part ? part[3] : 0.f;
    for (int o = n / 2; o > 0; o >>= 1)
        fold(m, top, rest, mom, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, top, o),
             __shfl_xor_sync(0xffffffffu, rest, o), __shfl_xor_sync(0xffffffffu, mom, o));
    m = __shfl_sync(0xffffffffu, m, 0);
    top = __shfl_sync(0xffffffffu, top, 0);
    rest = __shfl_sync(0xffffffffu, rest, 0);
    mom = __shfl_sync(0xffffffffu, mom, 0);
}

// The CTA's K best where more than kLpFound logits reach the floor (equal
// logits, sorted rows): each warp holds a sorted list across its lanes and
// goes over its values in the order of their ids, so that equal ones later in
// the row cost a comparison each.
template <typename T, int NTH>
__device__ __noinline__ void list_rows(LpSmem<T, NTH> &sh, const RowView<T> &x, int v0, int v1, int K, float floor) {
    constexpr int V = Raw<T>::V, kBatch = NTH * kLpLoads;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    Key mine = 0;   // lane i: the warp's i-th best
    int b = 0;
    for (int vb = v0; vb < v1; vb += kBatch, b++) {
        const bool hit = (float)sh.batch_max[b % LpSmem<T, NTH>::kSlots][threadIdx.x] >= floor;
        if (!__any_sync(0xffffffffu, hit)) continue;
        for (int u = 0; u < kLpLoads; u++) {
            const int v = vb + u * NTH + threadIdx.x;
            const uint32_t none = Raw<T>::kNone;
            float f[V];
            Raw<T>::values(hit && v < v1 ? x.any(v) : make_uint4(none, none, none, none), f);
            const int id0 = x.first(v), n = hit && v < v1 ? x.count(v) : 0;
#pragma unroll
            for (int i = 0; i < V; i++) {
                bool cand = i < n && f[i] >= floor;
                if (!__any_sync(0xffffffffu, cand)) continue;
                const Key k = make_key(f[i], id0 + i);
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
    sh.lists[warp][lane] = lane < K ? mine : 0;
    __syncthreads();
    if (lane < K && mine != 0) {   // the rank of each key among the warps' lists
        int rank = 0;
        for (int w = 0; w < (NTH / 32); w++) rank += better(sh.lists[w], K, mine);
        if (rank < K) sh.merged[rank] = mine;
    }
}

template <typename T, int NTH>
__global__ void __launch_bounds__(NTH, NTH == kLpMany ? kLpCtas : 1024 / NTH) token_logprobs_kernel(const LogprobParams p, int Z) {
    constexpr int V = Raw<T>::V;
    __shared__ LpSmem<T, NTH> sh;
    __shared__ LpCluster cl;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr bool kAhead = LpSmem<T, NTH>::kAhead;
    static_assert(!kAhead || kLpCtas * (sizeof(sh) + 1024) <= 228 * 1024, "they fit an SM");
    if (kAhead) Z = 1;   // (no code for shares)
    const int row = blockIdx.x / Z, z = blockIdx.x % Z;
    const RowView<T> x(static_cast<const T *>(p.logits) + (long long)row * p.ld, p.vocab);
    // this CTA's vectors, of -1 .. full
    const int nv = x.full + 2;
    const int v0 = (int)((long long)z * nv / Z) - 1, v1 = (int)((long long)(z + 1) * nv / Z) - 1;
    const int K = p.n_top;

    // Z = top + rest: `top` counts the logits equal to m, the others' e^(x - m)
    // add up apart from it, so that a confident row's ln Z and H keep their
    // leading digits (ln Z = log1p(rest)).
    // The maximum is the warp's, so that few batches move it.
    const float lowest = Raw<T>::lowest();
    float m = lowest, top = 0.f, rest = 0.f, mom = 0.f, best = -INFINITY;
    constexpr int kSlots = LpSmem<T, NTH>::kSlots;
    for (int s = 0; s < kSlots; s++) sh.batch_max[s][threadIdx.x] = (T)-INFINITY;
    constexpr int kBatch = NTH * kLpLoads;
    auto load = [&](int vb, uint4 (&u)[kLpLoads]) {
        const int v = vb + threadIdx.x;
        if (vb >= 0 && vb + kBatch <= min(v1, x.full)) {
#pragma unroll
            for (int i = 0; i < kLpLoads; i++) u[i] = x.whole(v + i * NTH);
        } else {
#pragma unroll
            for (int i = 0; i < kLpLoads; i++) {
                const uint32_t none = Raw<T>::kNone;
                u[i] = v + i * NTH < v1 ? x.any(v + i * NTH) : make_uint4(none, none, none, none);
            }
        }
    };
    auto take = [&](const uint4 (&u)[kLpLoads], int b) {   // batch b
        uint32_t mw[2] = {Raw<T>::kNone, Raw<T>::kNone};
#pragma unroll
        for (int i = 0; i < kLpLoads; i++) Raw<T>::raise(mw, u[i]);
        const float bm = Raw<T>::largest(mw);
        best = fmaxf(best, bm);
        T &kept = sh.batch_max[b % kSlots][threadIdx.x];   // (bm is one of the logits: exact in T)
        kept = (T)(b < kSlots ? bm : fmaxf((float)kept, bm));
        const float wm = fmaxf(warp_max(bm), lowest);
        if (wm > m) {
            const float d = fmax_nan((m - wm) * kLog2e, kLpFloor), w = exp2_approx(d);
            rest += top;
            mom = w * fmaf(rest, d, mom);
            rest *= w;
            top = 0.f;
            m = wm;
        }
        // x - m first, then log2(e): in one multiply-add -m log2(e) would be
        // rounded to m's size, and every weight off by as much (fp32 logits
        // near 30000: ln Z by 1e-3)
        const uint64_t l2 = pair(kLog2e, kLog2e), nm = pair(-m, -m);
        uint64_t s2[2] = {0, 0}, t2[2] = {0, 0};
        if (wm < m) {   // (the maximum is in another batch)
#pragma unroll
            for (int i = 0; i < kLpLoads; i++)
#pragma unroll
                for (int j = 0; j < V / 2; j++) {
                    const float2 f = Raw<T>::pair_of(u[i], j);
                    const uint64_t t = mul2(add2(pair(f.x, f.y), nm), l2);
                    float ta, tb;
                    unpair(t, ta, tb);
                    const uint64_t e = pair(exp2_approx(ta), exp2_approx(tb));
                    s2[j & 1] = add2(s2[j & 1], e);
                    t2[j & 1] = fma2(e, t, t2[j & 1]);
                }
        } else {
#pragma unroll
            for (int i = 0; i < kLpLoads; i++)
#pragma unroll
                for (int j = 0; j < V / 2; j++) {
                    const float2 f = Raw<T>::pair_of(u[i], j);
                    const uint64_t t = mul2(add2(pair(f.x, f.y), nm), l2);
                    float ta, tb;
                    unpair(t, ta, tb);
                    const bool a = f.x == m, c = f.y == m;
                    top += (a ? 1.f : 0.f) + (c ? 1.f : 0.f);
                    const uint64_t e = pair(a ? 0.f : exp2_approx(ta), c ? 0.f : exp2_approx(tb));
                    s2[j & 1] = add2(s2[j & 1], e);
                    t2[j & 1] = fma2(e, t, t2[j & 1]);
                }
        }
        float a, c;
        unpair(add2(s2[0], s2[1]), a, c);
        rest += a + c;
        unpair(add2(t2[0], t2[1]), a, c);
        mom += a + c;
    };
    if constexpr (kAhead) {
        constexpr int kBufs = kLpAhead + 1;
        auto fetch = [&](int b) {   // a group of copies even where no batch is left, so that the groups count
            const int vb = v0 + b * kBatch, v = vb + threadIdx.x;
            uint4(*const to)[NTH] = sh.ahead[b % kBufs];
            if (vb >= 0 && vb + kBatch <= min(v1, x.full)) {
#pragma unroll
                for (int i = 0; i < kLpLoads; i++)
                    cp_async16(smem_u32(&to[i][threadIdx.x]), reinterpret_cast<const uint4 *>(x.x + x.head) + v + i * NTH, true);
            } else if (vb < v1) {
                uint4 u[kLpLoads];
                load(vb, u);
#pragma unroll
                for (int i = 0; i < kLpLoads; i++) to[i][threadIdx.x] = u[i];
            }
            cp_async_commit();
        };
#pragma unroll
        for (int b = 0; b < kLpAhead; b++) fetch(b);
        for (int b = 0; v0 + b * kBatch < v1; b++) {
            fetch(b + kLpAhead);
            cp_async_wait<kLpAhead>();
            uint4 u[kLpLoads];
#pragma unroll
            for (int i = 0; i < kLpLoads; i++) u[i] = sh.ahead[b % kBufs][i][threadIdx.x];
            take(u, b);
        }
        cp_async_wait<0>();
    } else {
        for (int vb = v0, b = 0; vb < v1; vb += kBatch, b++) {
            uint4 u[kLpLoads];
            load(vb, u);
            take(u, b);
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
    {
        float g = best;
#pragma unroll
        for (int o = NTH / kLpGroups / 2; o > 0; o >>= 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, o));
        if (lane % (NTH / kLpGroups) == 0) sh.group_max[threadIdx.x / (NTH / kLpGroups)] = g;
    }
    if (threadIdx.x < kTopMax) sh.merged[threadIdx.x] = 0;
    if (threadIdx.x == 0) sh.count = sh.hits = 0;
    __syncthreads();
    if (warp == 0) {
        fold_lanes(lane < (NTH / 32) ? sh.red[lane] : nullptr, (NTH / 32), m, top, rest, mom);
        const float g = warp_max(fmaxf(sh.group_max[lane], sh.group_max[lane + 32]));
        if (lane == 0) {
            sh.stat[0] = m;
            sh.stat[1] = top;
            sh.stat[2] = rest;
            sh.stat[3] = mom;
            sh.stat[4] = g;
        }
    }
    if (K > 0) {
        if (warp == 1 || warp == 2) {   // the K-th largest group maximum: K - 1 others are at least as large
            const int me = lane + 32 * (warp - 1);
            const float g = sh.group_max[me];
            int rank = 0;
#pragma unroll 16
            for (int o = 0; o < kLpGroups; o++) {
                const float h = sh.group_max[o];
                rank += h > g || (h == g && o < me);
            }
            if (rank == K - 1) sh.floor = g;
        }
        __syncthreads();
        const float floor = sh.floor;
        // the batches that reach it: 16 * kLpLoads bytes of one thread each
        const int batches = (v1 - v0 + kBatch - 1) / kBatch;
        if (best >= floor)
            for (int s = 0; s < min(kSlots, batches); s++)
                if ((float)sh.batch_max[s][threadIdx.x] >= floor)
                    for (int b = s; b < batches; b += kSlots) {
                        const int at = atomicAdd(&sh.hits, 1);
                        if (at < kLpFound) sh.hit[at] = b * NTH + threadIdx.x;
                    }
        __syncthreads();
        // a warp per batch, a value per lane
        constexpr int kValues = V * kLpLoads;
        const int hits = sh.hits;
#pragma unroll 4
        for (int h = warp; h < min(hits, kLpFound); h += NTH / 32) {
            const int e = sh.hit[h], v = v0 + e / NTH * kBatch + lane / V * NTH + e % NTH;
            float f = -INFINITY;
            int id = 0;
            if (lane < kValues && v < v1 && lane % V < x.count(v)) {
                id = x.first(v) + lane % V;
                f = (float)x.x[id];
                if (f >= floor) {
                    const int at = atomicAdd(&sh.count, 1);
                    if (at < kLpFound) sh.found[at] = make_key(f, id);
                }
            }
        }
        __syncthreads();
        const int found = sh.count;
        if (found <= kLpFound && hits <= kLpFound) {
            for (int f = threadIdx.x; f < found; f += NTH) {
                const Key k = sh.found[f];
                int rank = 0;
#pragma unroll 8
                for (int o = 0; o < found; o++) rank += sh.found[o] > k;
                if (rank < K) sh.merged[rank] = k;
            }
        } else {
            list_rows<T, NTH>(sh, x, v0, v1, K, floor);
        }
    }
    __syncthreads();

    // the row's (m, top, rest, S) and largest logit
    float gm, gn, gr, gt, gb;
    if (Z > 1) {
        cluster_sync_all();
        for (int e = threadIdx.x; e < Z * 5; e += NTH)
            cl.stat[e / 5][e % 5] = ld_dsmem_f1(mapa_shared(smem_u32(sh.stat + e % 5), e / 5));
        for (int e = threadIdx.x; e < Z * kTopMax && K > 0; e += NTH) {
            const float2 v = ld_dsmem_f2(mapa_shared(smem_u32(sh.merged + e % kTopMax), e / kTopMax));
            cl.lists[e / kTopMax][e % kTopMax] = ((Key)__float_as_uint(v.y) << 32) | __float_as_uint(v.x);
        }
        if (threadIdx.x < kTopMax) cl.rank[threadIdx.x] = 0;
        cluster_sync_all();   // (peers may leave now: their shares have been read)
        fold_lanes(lane < Z ? cl.stat[lane] : nullptr, kLpShares, gm, gn, gr, gt);
        gb = warp_max(lane < Z ? cl.stat[lane][4] : -INFINITY);
    } else {
        gm = sh.stat[0];
        gn = sh.stat[1];
        gr = sh.stat[2];
        gt = sh.stat[3];
        gb = sh.stat[4];
    }
    if ((gb <= lowest || gb > 1e38f) && fabsf(gb) < INFINITY) {
        // every logit is as low as a mask's, and the sums above took the
        // vectors' padding along; or distances overflow, and 0 times an
        // infinite one is NaN: once more, value by value
        gn = gr = gt = 0.f;
        for (int i = threadIdx.x; i < p.vocab; i += NTH) {
            const float d = ((float)x.x[i] - gb) * kLog2e, e = exp2_approx(d);
            if (d == 0.f) gn += 1.f;
            else {
                gr += e;
                if (e != 0.f) gt = fmaf(e, d, gt);
            }
        }
        gn = warp_sum(gn);
        gr = warp_sum(gr);
        gt = warp_sum(gt);
        __syncthreads();
        if (lane == 0) {
            sh.red[warp][0] = gn;
            sh.red[warp][1] = gr;
            sh.red[warp][2] = gt;
        }
        __syncthreads();
        gn = gr = gt = 0.f;
        for (int w = 0; w < (NTH / 32); w++) {
            gn += sh.red[w][0];
            gr += sh.red[w][1];
            gt += sh.red[w][2];
        }
    }
    float lz = gn == 1.f ? log1pf(gr) : logf(gn + gr);
    gt *= 0.69314718055994531f;              // from log2 units
    if (!(fabsf(gb) < INFINITY)) lz = NAN;   // no finite logit, or an infinite one
    if (z == 0 && threadIdx.x == 0) {
        if (p.logprob) {
            const int tok = __ldg(p.tokens + row);
            p.logprob[row] = tok >= 0 && tok < p.vocab ? ((float)x.x[tok] - gb) - lz : NAN;
        }
        if (p.entropy) p.entropy[row] = lz - gt / (gn + gr);
    }
    if (K == 0) return;
    int *ids = p.top_ids + (long long)row * K;
    float *lps = p.top_logprob ? p.top_logprob + (long long)row * K : nullptr;
    auto put = [&](int rank, Key k) {   // NaN logits are no alternatives: key 0 where nothing is left
        ids[rank] = k ? key_id(k) : -1;
        if (lps) lps[rank] = k ? (key_value(k) - gb) - lz : NAN;
    };
    if (Z == 1) {
        if (threadIdx.x < K) put(threadIdx.x, sh.merged[threadIdx.x]);
        return;
    }
    // each share ranks its own list among all: a thread per (key, list)
    for (int e = threadIdx.x; e < Z * kTopMax; e += NTH) {
        const Key k = cl.lists[z][e % kTopMax];
        if (k) atomicAdd(&cl.rank[e % kTopMax], better(cl.lists[e / kTopMax], K, k));
    }
    __syncthreads();
    if (threadIdx.x < K) {
        const Key k = cl.lists[z][threadIdx.x];
        if (k && cl.rank[threadIdx.x] < K) put(cl.rank[threadIdx.x], k);
    }
    if (z == 0 && threadIdx.x < 32) {   // places that nothing fills
        int found = lane < Z ? better(cl.lists[lane], K, 0) : 0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) found += __shfl_xor_sync(0xffffffffu, found, o);
        if (lane < K && lane >= found) put(lane, 0);
    }
}

template <typename T, int NTH>
cudaError_t launch_threads(const LogprobParams &p, int Z, cudaStream_t st) {
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (!(done.load() & bit)) {
        e = cudaFuncSetAttribute(token_logprobs_kernel<T, NTH>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
        done.fetch_or(bit);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(p.n_rows * Z));
    cfg.blockDim = dim3(NTH);
    cfg.stream = st;
    cudaLaunchAttribute a[1];
    a[0].id = cudaLaunchAttributeClusterDimension;
    a[0].val.clusterDim.x = Z;
    a[0].val.clusterDim.y = 1;
    a[0].val.clusterDim.z = 1;
    cfg.attrs = a;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, NTH>, p, Z);
}

template <typename T>
cudaError_t launch_typed(const LogprobParams &p, int Z, int sms, cudaStream_t st) {
    return p.n_rows <= sms ? launch_threads<T, kLpFew>(p, Z, st) : launch_threads<T, kLpMany>(p, 1, st);
}

}  // namespace

cudaError_t launch_token_logprobs(const LogprobParams &p, int sms, cudaStream_t st) {
    // shares of a row: as many as fill the SMs twice, each with a batch of
    // work for its threads, at most a cluster's 16
    const int elem = p.dtype == ELEM_F32 ? 4 : 2;
    const long long batch = (long long)kLpFew * 16 / elem;
    const long long by_work = std::max<long long>(1, p.vocab / batch);
    const long long by_sms = 2ll * sms / p.n_rows;
    const int Z = (int)std::max(1ll, std::min<long long>(16, std::min(by_work, by_sms)));
    switch (p.dtype) {
        case ELEM_F32: return launch_typed<float>(p, Z, sms, st);
        case ELEM_BF16: return launch_typed<__nv_bfloat16>(p, Z, sms, st);
        default: return launch_typed<__half>(p, Z, sms, st);
    }
}

}  // namespace vc
