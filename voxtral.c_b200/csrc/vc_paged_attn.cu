// vc_paged_attn.cu - attention of a few rows per stream over a paged cache in
// 8 bits: one token, a few drafted ones.
//
// Bound by HBM where there are many keys: each is read once, 2 HD bytes, and 4 HD
// operations per query head of its group follow, on the tensor cores (mma.sync
// m16n8k16, fp16 operands, fp32 sums), which leaves them mostly idle at these row
// counts.  e4m3 is exact in fp16, and the orders of dims and keys within an MMA are
// free as long as both operands have the same, so that each lane takes 16
// consecutive bytes of a key at a time:
//   S^T = K Q^T    A = 16 keys, lane (g, t) has dims 16 t .. 16 t + 15 (and 64
//                  more on) of keys g and g + 8; B = packed rows (row x head of
//                  the group), 8 to a column tile
//   O^T += V^T P^T A = V^T, lane (g, t) has dims g HD / 8 .. of keys 2 t, 2 t + 1,
//                  2 t + 8, 2 t + 9, which a byte permutation pairs; B = P^T,
//                  which is S^T transposed in 8 x 8 tiles (movmatrix)
// A lane's S and O columns are the same two packed rows, so that their maximum
// and sum are its own.
//
// A warp takes 32 keys at a time, by itself, through a ring of its own in shared
// memory that asynchronous copies fill two steps ahead (without it, the next keys in
// registers: 64 tokens of 7400 keys on the average 333 us, with it 250).  Its CTA's
// warps and then the CTAs of a cluster, which share the keys of a tile of rows, join
// their sums at the end, in order.
//
// Measured, 32 / 8 heads of 128, inputs that L2 does not hold: 64 tokens over 5 to 16
// thousand keys 246 us, 5.7 TB/s, 0.86 of the copy rate (217 to 234 where a graph replays
// the call over the same few caches); 24 tokens over 4100 keys 40 us, 0.53 (384 CTAs, two
// or three to an SM); 8 streams of 6 tokens over 1 to 3 thousand keys 28 us; one token
// over 8192 keys 14.8 us, of which ~7 are the launch, three dependent reads before the
// first key and the merge, the rest 4 to 5 steps of a warp at ~1.3 us each: reads from
// shared memory, conversions, MMAs and exponentials in turn.
//
// q: bf16 rows are scaled by a power of two into fp16's range (exact but for
// values 2^-29 of the row's largest).  V's scales vs go into P: P = 2^(s - m) vs is
// rounded to fp16, half a step of 2^-11, with m the row's own maximum of s + log2 vs so
// far, less 7 (its P is 2^7, which rounds to itself), which moves only when one exceeds
// it by 15: P fills the type up to 2^15, and what is lost is 2^-32 of the row's largest
// weight times scale, whatever the scales of pages that it does not see.  The weights'
// sum has a base of its own, the row's maximum of s: with one for both, a weight on a
// page of small V (zeros have the scale 2^-100) would be lost to one or the other.
// Sums, maxima and O are fp32.
#include "vc_cluster.h"
#include "vc_paged.cuh"
#include "vc_tc.cuh"

#include <algorithm>
#include <math.h>

namespace vc {

using namespace tc;

namespace {

constexpr int kFwKeys = 32;              // keys of a warp's step
constexpr int fw_ctas(int w, int s) { return w == 8 ? 1 : s == 2 ? 3 : 2; }
constexpr float kFwBelow = 7.f;          // P's maximum less m
constexpr float kFwAbove = 15.f;         // log2 of what P, or a weight, may reach before its base moves
constexpr float kFwWide = 0x1p100f;      // from this factor on P is not taken from the weight, which may have left fp32

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ uint32_t half2_bits(uint32_t e4m3x2) {
    const __half2 h = from_e4m3x2(e4m3x2);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <int N>   // 4 N bytes of shared memory
__device__ __forceinline__ void lds_words(uint32_t (&w)[N], uint32_t addr) {
    if constexpr (N == 4)
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr));
    else
        asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
}
__device__ __forceinline__ float log2_approx(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void cp_async4(uint32_t dst_smem, const void *src, bool ok) {
    const int n = ok ? 4 : 0;
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst_smem), "l"(src), "r"(n) : "memory");
}

// A stage: 32 keys' K, then V, as lines of 128 bytes (HD = 64: two keys a line)
// whose 16-byte chunks are permuted so that the lanes of a load meet no bank
// twice.
template <int HD>
__device__ __forceinline__ int k_chunk(int r, int ch) {
    return HD == 128 ? r * 128 + ((ch ^ ((r & 1) << 2)) << 4) : r * 64 + (ch << 4);
}
template <int HD>
__device__ __forceinline__ int v_chunk(int r, int ch) {
    const int sw = ((r >> 1) & 3) << 1;
    return HD == 128 ? r * 128 + ((ch ^ sw) << 4) : (r >> 1) * 128 + ((((r & 1) * 4 + ch) ^ sw) << 4);
}

template <int HD, int NR, int W, int S>
struct FwSmem {
    static constexpr int kTile = kFwKeys * HD;
    union {
        unsigned char kv[W][S][2][kTile];
        float o[W][8 * NR][HD];
    };
    float scale[W][S][4];   // K's of the two groups of 16 keys, V's
    float mx[W][8 * NR], sum[W][8 * NR];
};

// NR: column tiles of 8 packed rows; W warps, rings of S stages
template <typename T, int HD, int NR, int W, int S>
__global__ void __launch_bounds__(W * 32, fw_ctas(W, S)) paged_few_kernel(const PagedAttnParams p) {
    constexpr int KC = HD / 64;       // 64-dim parts of a key
    constexpr int MT = HD / 16;       // 16-dim tiles of O
    constexpr int VW = HD / 32;       // words that a lane has of a V row
    constexpr int kRows = 8 * NR;
    constexpr int kWarps = W, kThreads = W * 32, kStages = S, kTile = FwSmem<HD, NR, W, S>::kTile;
    extern __shared__ __align__(128) unsigned char fw_smem_raw[];
    FwSmem<HD, NR, W, S> &sh = *reinterpret_cast<FwSmem<HD, NR, W, S> *>(fw_smem_raw);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int z = blockIdx.x % p.shares, Z = p.shares;
    const int m0 = blockIdx.x / p.shares * kRows, kvh = blockIdx.y, stream = blockIdx.z;
    const RowSpan s = paged_span(p.r, p.c, stream);
    const int M = s.n * p.group;
    if (m0 >= M) return;   // the whole cluster leaves
    const int i0 = m0 / p.group, i1 = (min(m0 + kRows, M) - 1) / p.group;
    // positions that some row sees: [0, ns) and [lo, hi), in units of 32
    const int p_min = s.pos + i0, p_max = s.pos + i1, hi = p_max + 1, ns = min(p.n_sink, hi);
    const int lo = p.window > 0 ? max(0, p_min - p.window + 1) : 0;
    const int sink_units = (ns + kFwKeys - 1) / kFwKeys, first = max(lo / kFwKeys, sink_units);
    const int units = sink_units + max(0, (hi + kFwKeys - 1) / kFwKeys - first);
    const int u0 = (int)((long long)z * units / Z), u1 = (int)((long long)(z + 1) * units / Z);
    auto key_of = [&](int u) { return (u < sink_units ? u : first + u - sink_units) * kFwKeys; };

    // a unit's pages, of its two groups of 16 keys
    auto pages_of = [&](int u, int (&pg)[2]) {
        pg[0] = pg[1] = -1;
        if (u >= u1) return;
        const int key = key_of(u);
#pragma unroll
        for (int a = 0; a < 2; a++) {
            const int k = key + 16 * a;
            if (k < hi && (k + 16 > lo || k < ns)) pg[a] = page_at(p.c, stream, k >> p.c.page_shift);
        }
    };
    // a unit's keys and scales on their way to a stage (zeros where there is no page)
    const uint32_t ring = smem_u32(sh.kv[warp]), scales = smem_u32(sh.scale[warp]);
    auto fetch = [&](int u, int stage, const int (&pg)[2]) {
        if (u < u1) {
            constexpr int kCh = HD / 16, kAtOnce = 32 / kCh;   // chunks of a row, rows of a step
            const int key = key_of(u), r0 = lane / kCh, ch = lane % kCh;
            const uint32_t k_to = ring + stage * (2 * kTile), v_to = k_to + kTile;
#pragma unroll
            for (int a = 0; a < 2; a++) {
                const bool ok = pg[a] >= 0;
                const long long from = ok ? page_base(p.c, p.layer, pg[a], kvh) + ((key + 16 * a) & (p.c.page - 1)) * p.c.slot_stride +
                                                r0 * p.c.slot_stride + ch * 16
                                          : 0;
#pragma unroll
                for (int i = 0; i < 16; i += kAtOnce) {
                    const long long off = from + (ok ? i * p.c.slot_stride : 0);
                    cp_async16(k_to + k_chunk<HD>(16 * a + i + r0, ch), p.c.k + off, ok);
                    cp_async16(v_to + v_chunk<HD>(16 * a + i + r0, ch), p.c.v + off, ok);
                }
            }
            if (lane < 4) {
                const int of = lane & 1 ? pg[1] : pg[0];
                const float *const from = lane < 2 ? p.c.k_scale : p.c.v_scale;
                cp_async4(scales + stage * 16 + lane * 4, from + (of >= 0 ? scale_at(p.c, p.layer, of, kvh) : 0), of >= 0);
            }
        }
        cp_async_commit();
    };
    int pg[2] = {-1, -1};
    uint32_t have = 0u;   // two bits a unit, the newest lowest: its groups' pages are there
    auto note = [&]() { have = have << 2 | (pg[1] >= 0 ? 2u : 0u) | (pg[0] >= 0 ? 1u : 0u); };
#pragma unroll
    for (int i = 0; i < kStages - 1; i++) {
        pages_of(u0 + warp + i * kWarps, pg);
        fetch(u0 + warp + i * kWarps, i, pg);
        note();
    }
    pages_of(u0 + warp + (kStages - 1) * kWarps, pg);
    // q as B operands: lane (g, t) has row g's dims in the order of K's
    uint32_t qf[NR][KC * 4][2];
    float cf[NR][2];          // score factor of the lane's rows 2 t, 2 t + 1, in log2
    int at[NR][2];            // their positions; -1: no row
#pragma unroll
    for (int n = 0; n < NR; n++) {
        const int m = m0 + n * 8 + g;
        float x[KC][16], big = 0.f;
        if (m < M) {
            const T *q = static_cast<const T *>(p.q) + ((long long)(s.r0 + m / p.group) * p.n_heads + kvh * p.group + m % p.group) * HD;
#pragma unroll
            for (int c = 0; c < KC; c++)
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const float4 v = load4<T>(q + c * 64 + t * 16 + e);
                    x[c][e] = v.x, x[c][e + 1] = v.y, x[c][e + 2] = v.z, x[c][e + 3] = v.w;
                }
        } else {
#pragma unroll
            for (int c = 0; c < KC; c++)
#pragma unroll
                for (int e = 0; e < 16; e++) x[c][e] = 0.f;
        }
        float up = 1.f;       // a power of two that takes the row's largest to [2^14, 2^15)
        if constexpr (sizeof(T) == 2 && !std::is_same<T, __half>::value) {
#pragma unroll
            for (int c = 0; c < KC; c++)
#pragma unroll
                for (int e = 0; e < 16; e++) big = fmaxf(big, fabsf(x[c][e]) < INFINITY ? fabsf(x[c][e]) : 0.f);
            big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
            big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
            const int e = (int)(__float_as_uint(big) >> 23) - 127;
            up = big > 0.f ? __uint_as_float((uint32_t)(min(14 - e, 126) + 127) << 23) : 1.f;
        }
#pragma unroll
        for (int c = 0; c < KC; c++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                qf[n][c * 4 + e][0] = pack2<__half>(x[c][4 * e] * up, x[c][4 * e + 1] * up);
                qf[n][c * 4 + e][1] = pack2<__half>(x[c][4 * e + 2] * up, x[c][4 * e + 3] * up);
            }
        const float f = p.scale_log2 / up;
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int mm = m0 + n * 8 + 2 * t + e;
            cf[n][e] = __shfl_sync(0xffffffffu, f, (2 * t + e) * 4);
            at[n][e] = mm < M ? s.pos + mm / p.group : -1;
        }
    }

    float o[NR][MT][4], l[NR][2];
    float lb[NR][2], pb[NR][2];   // bases of the sums (a whole number) and of P; -inf: nothing yet
    float up[NR][2];              // 2^(lb - pb); 0: nothing yet
#pragma unroll
    for (int n = 0; n < NR; n++) {
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[n][mt][e] = 0.f;
        lb[n][0] = lb[n][1] = pb[n][0] = pb[n][1] = -INFINITY;
        l[n][0] = l[n][1] = up[n][0] = up[n][1] = 0.f;
    }

    // 16 dims x 16 keys of V^T as an A operand
    auto v_tile = [&](const uint32_t (&w)[4][VW], int mt, uint32_t (&a)[4]) {
        const uint32_t sel = (mt & 1) ? 0x7362u : 0x5140u;
        const uint32_t x = __byte_perm(w[0][mt / 2], w[1][mt / 2], sel), y = __byte_perm(w[2][mt / 2], w[3][mt / 2], sel);
        a[0] = half2_bits(x & 0xffffu);
        a[1] = half2_bits(x >> 16);
        a[2] = half2_bits(y & 0xffffu);
        a[3] = half2_bits(y >> 16);
    };

    int stage = 0;
    for (int u = u0 + warp; u < u1; u += kWarps) {
        cp_async_wait<kStages - 2>();
        __syncwarp();   // this unit is there for all lanes, and all have done with the one before
        fetch(u + (kStages - 1) * kWarps, stage == 0 ? kStages - 1 : stage - 1, pg);
        note();
        pages_of(u + kStages * kWarps, pg);
        const uint32_t k_at = ring + stage * (2 * kTile), v_at = k_at + kTile;
        const uint32_t there = have >> (2 * (kStages - 1));
        const float4 sc = *reinterpret_cast<const float4 *>(sh.scale[warp][stage]);
        const float k_now[2] = {sc.x, sc.y}, v_now[2] = {sc.z, sc.w};
        const float v_log[2] = {log2_approx(sc.z), log2_approx(sc.w)};
        stage = stage + 1 == kStages ? 0 : stage + 1;
        const int key = key_of(u);
        const bool whole = (there & 3u) == 3u && key + kFwKeys - 1 <= p_min &&
                           (p.window <= 0 || key > p_max - p.window || key + kFwKeys <= p.n_sink);
        // scores
        float x[NR][2][4];
#pragma unroll
        for (int n = 0; n < NR; n++)
#pragma unroll
            for (int a = 0; a < 2; a++)
#pragma unroll
                for (int e = 0; e < 4; e++) x[n][a][e] = 0.f;
#pragma unroll
        for (int a = 0; a < 2; a++)
#pragma unroll
            for (int c = 0; c < KC; c++) {
                uint32_t w0[4], w1[4];
                lds_words<4>(w0, k_at + k_chunk<HD>(16 * a + g, c * 4 + t));
                lds_words<4>(w1, k_at + k_chunk<HD>(16 * a + g + 8, c * 4 + t));
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    uint32_t f[4];
                    f[0] = half2_bits(w0[e] & 0xffffu);
                    f[1] = half2_bits(w1[e] & 0xffffu);
                    f[2] = half2_bits(w0[e] >> 16);
                    f[3] = half2_bits(w1[e] >> 16);
#pragma unroll
                    for (int n = 0; n < NR; n++) mma_f16(x[n][a], f, qf[n][c * 4 + e][0], qf[n][c * 4 + e][1]);
                }
            }
        bool over = false;
        uint32_t vis = 0xffffffffu;   // bit 4 (2 n + a) + e: the lane's row sees its key
#pragma unroll
        for (int n = 0; n < NR; n++)
#pragma unroll
            for (int a = 0; a < 2; a++) {
                const float most[2] = {fminf(lb[n][0] + kFwAbove, pb[n][0] + kFwAbove - v_log[a]),
                                       fminf(lb[n][1] + kFwAbove, pb[n][1] + kFwAbove - v_log[a])};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float &v = x[n][a][e];
                    v *= cf[n][e & 1] * k_now[a];
                    if (!whole) {
                        const int j = key + 16 * a + g + (e >> 1) * 8, i = at[n][e & 1];
                        const bool see = ((there >> a) & 1u) && j <= i && (p.window <= 0 || j > i - p.window || j < p.n_sink);
                        v = see ? v : -INFINITY;
                        if (!see) vis &= ~(1u << (8 * n + 4 * a + e));
                    }
                    over |= v > most[e & 1];
                }
            }
        if (__any_sync(0xffffffffu, over)) {
#pragma unroll
            for (int n = 0; n < NR; n++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const float x0 = fmaxf(x[n][0][e], x[n][0][e + 2]), x1 = fmaxf(x[n][1][e], x[n][1][e + 2]);
                    float top = fmaxf(x0, x1), p_top = fmaxf(x0 + v_log[0], x1 + v_log[1]);
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) {
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                        p_top = fmaxf(p_top, __shfl_xor_sync(0xffffffffu, p_top, d));
                    }
                    if (top > lb[n][e] + kFwAbove) {
                        const float base = ceilf(top);
                        l[n][e] *= exp2f(lb[n][e] - base);
                        lb[n][e] = base;
                    }
                    if (p_top > pb[n][e] + kFwAbove) {
                        const float base = p_top - kFwBelow, f = exp2f(pb[n][e] - base);
                        pb[n][e] = base;
#pragma unroll
                        for (int mt = 0; mt < MT; mt++) {
                            o[n][mt][e] *= f;
                            o[n][mt][e + 2] *= f;
                        }
                    }
                    up[n][e] = pb[n][e] == -INFINITY ? 0.f : exp2f(lb[n][e] - pb[n][e]);
                }
        }
        uint32_t pf[NR][2][2];
#pragma unroll
        for (int n = 0; n < NR; n++) {
            const float base[2] = {lb[n][0] == -INFINITY ? 0.f : lb[n][0], lb[n][1] == -INFINITY ? 0.f : lb[n][1]};
#pragma unroll
            for (int a = 0; a < 2; a++) {
                const float by[2] = {v_now[a] * up[n][0], v_now[a] * up[n][1]};
                float w[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    w[e] = exp2_approx(x[n][a][e] - base[e & 1]);
                    l[n][e & 1] += w[e];
                    w[e] *= by[e & 1];
                }
                if (by[0] > kFwWide || by[1] > kFwWide) {
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (by[e & 1] > kFwWide) w[e] = exp2_approx(x[n][a][e] + (v_log[a] - pb[n][e & 1]));
                }
                pf[n][a][0] = transpose8(pack2<__half>(w[0], w[1]));
                pf[n][a][1] = transpose8(pack2<__half>(w[2], w[3]));
            }
        }
        uint32_t vw[2][4][VW];
#pragma unroll
        for (int a = 0; a < 2; a++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int row = 16 * a + 2 * t + (r & 1) + (r >> 1) * 8;
                lds_words<VW>(vw[a][r], v_at + (HD == 128 ? v_chunk<HD>(row, g) : v_chunk<HD>(row, g >> 1) + (g & 1) * 8));
            }
        bool nan = false;
        if (!whole) {
            // zero times a masked key's NaN would be NaN: zeros in its place, and
            // NaN for the rows that do see it
            uint32_t bad[2][4][VW];
#pragma unroll
            for (int a = 0; a < 2; a++)
#pragma unroll
                for (int r = 0; r < 4; r++)
#pragma unroll
                    for (int e = 0; e < VW; e++) {
                        bad[a][r][e] = __vcmpeq4(vw[a][r][e] & 0x7f7f7f7fu, 0x7f7f7f7fu);
                        vw[a][r][e] &= ~bad[a][r][e];
                        nan |= bad[a][r][e] != 0u;
                    }
            if (__any_sync(0xffffffffu, nan)) {
#pragma unroll
                for (int n = 0; n < NR; n++)
#pragma unroll
                    for (int a = 0; a < 2; a++) {
                        const uint32_t b = vis >> (8 * n + 4 * a);
                        const uint32_t s0 = transpose8(pack2<__half>(b & 1u ? 1.f : 0.f, b & 2u ? 1.f : 0.f));
                        const uint32_t s1 = transpose8(pack2<__half>(b & 4u ? 1.f : 0.f, b & 8u ? 1.f : 0.f));
                        uint32_t one[4][VW];
#pragma unroll
                        for (int r = 0; r < 4; r++)
#pragma unroll
                            for (int e = 0; e < VW; e++) one[r][e] = bad[a][r][e] & 0x38383838u;   // 1.0
#pragma unroll
                        for (int mt = 0; mt < MT; mt++) {
                            uint32_t f[4];
                            float d[4] = {0.f, 0.f, 0.f, 0.f};
                            v_tile(one, mt, f);
                            mma_f16(d, f, s0, s1);
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                if (d[e] > 0.f) o[n][mt][e] = NAN;
                        }
                    }
            }
        }
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int a = 0; a < 2; a++) {
                uint32_t f[4];
                v_tile(vw[a], mt, f);
#pragma unroll
                for (int n = 0; n < NR; n++) mma_f16(o[n][mt], f, pf[n][a][0], pf[n][a][1]);
            }
    }
    cp_async_wait<0>();
    __syncthreads();   // the ring becomes the warps' sums

    // the warp's share: its sum over the lanes as a number of [1, 2) times a power of
    // two, which is its base, and O in the same units, so that no merge overflows
#pragma unroll
    for (int n = 0; n < NR; n++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            float sum = l[n][e];
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            const int r = n * 8 + 2 * t + e, bits = sum > 0.f && sum < INFINITY ? (int)(__float_as_uint(sum) >> 23) - 127 : 0;
            const float down = __uint_as_float((uint32_t)(127 - bits) << 23), f = pb[n][e] == -INFINITY ? 0.f : exp2f(pb[n][e] - lb[n][e]);
            if (g == 0) {
                sh.mx[warp][r] = lb[n][e] + (float)bits;
                sh.sum[warp][r] = sum * down;
            }
            float *const to = sh.o[warp][r] + g * (HD / 8);
#pragma unroll
            for (int mt = 0; mt < MT; mt += 2)
                *reinterpret_cast<float4 *>(to + 2 * mt) = make_float4(o[n][mt][e] * down * f, o[n][mt][e + 2] * down * f,
                                                                       o[n][mt + 1][e] * down * f, o[n][mt + 1][e + 2] * down * f);
        }
    __syncthreads();
    // the CTA's: into its first warp's place
    const int rows = min(kRows, M - m0);
    for (int e = threadIdx.x; e < kRows * (HD / 4); e += kThreads) {
        const int r = e / (HD / 4), d = e % (HD / 4) * 4;
        float top = sh.mx[0][r];
#pragma unroll
        for (int w = 1; w < kWarps; w++) top = fmaxf(top, sh.mx[w][r]);
        const float base = top == -INFINITY ? 0.f : top;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; w++) {
            const float f = exp2_approx(sh.mx[w][r] - base);
            const float4 v = *reinterpret_cast<const float4 *>(sh.o[w][r] + d);
            a.x = fmaf(f, v.x, a.x), a.y = fmaf(f, v.y, a.y), a.z = fmaf(f, v.z, a.z), a.w = fmaf(f, v.w, a.w);
        }
        *reinterpret_cast<float4 *>(sh.o[0][r] + d) = a;
    }
    __syncthreads();
    if (threadIdx.x < kRows) {
        const int r = threadIdx.x;
        float top = sh.mx[0][r], sum = 0.f;
#pragma unroll
        for (int w = 1; w < kWarps; w++) top = fmaxf(top, sh.mx[w][r]);
        const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int w = 0; w < kWarps; w++) sum = fmaf(exp2_approx(sh.mx[w][r] - base), sh.sum[w][r], sum);
        sh.mx[0][r] = top;
        sh.sum[0][r] = sum;
    }
    if (Z > 1) cluster_sync_all();
    else __syncthreads();
    const uint32_t o_s = smem_u32(sh.o[0]), m_s = smem_u32(sh.mx[0]), l_s = smem_u32(sh.sum[0]);
    for (int e = z * kThreads + threadIdx.x; e < rows * (HD / 4); e += Z * kThreads) {
        const int r = e / (HD / 4), d = e % (HD / 4) * 4, m = m0 + r;
        float top = -INFINITY, sum = 0.f;
        for (int c = 0; c < Z; c++) top = fmaxf(top, ld_dsmem_f1(mapa_shared(m_s + 4 * r, c)));
        const float base = top == -INFINITY ? 0.f : top;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int c = 0; c < Z; c++) {
            const float f = exp2_approx(ld_dsmem_f1(mapa_shared(m_s + 4 * r, c)) - base);
            const float4 v = ld_dsmem_f4(mapa_shared(o_s + 4 * (r * HD + d), c));
            sum = fmaf(f, ld_dsmem_f1(mapa_shared(l_s + 4 * r, c)), sum);
            a.x = fmaf(f, v.x, a.x), a.y = fmaf(f, v.y, a.y), a.z = fmaf(f, v.z, a.z), a.w = fmaf(f, v.w, a.w);
        }
        const float il = sum == 0.f ? 0.f : 1.0f / sum;
        const long long line = (long long)(s.r0 + m / p.group) * p.n_heads + kvh * p.group + m % p.group;
        store4<T>(static_cast<T *>(p.out) + line * HD + d, make_float4(a.x * il, a.y * il, a.z * il, a.w * il));
        if (p.lse && d == 0) p.lse[line] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.69314718055994531f;
    }
    if (Z > 1) cluster_sync_all();   // no CTA leaves while a peer still reads its share
}

// A shape's launch: its cluster size and what that costs.
struct FwPlan {
    double cost = 1e30;
    int shares = 0;
};

// Microseconds: fitted to the times of 40 calls (1 to 64 streams, 1 to 16 rows, 100
// to 16000 positions, 5 head layouts) in every shape and with 1 to 8 shares; the
// least by the model is within 2% of the least measured on the average, 15% at most.
//   a CTA's start and end, the merge of shares, and per share; a further wave of CTAs
constexpr double kFwFixed = 3.9, kFwMerge = 0.9, kFwShare = 0.23, kFwWave = 4.4, kFwEight = 1.1;   // kFwEight: of 8 warps
//   a step of 32 keys: what a warp by itself takes, and what the SM does for each,
//   for heads of 128 and 8 packed rows; and of 64, 16 rows, rings of two stages
constexpr double kFwStep = 1.07, kFwStepSm = 0.155;
constexpr double kFwStep64 = 1.5, kFwStepSm64 = 0.32, kFwStep16 = 2.1, kFwStepSm16 = 1.85, kFwStepTwo = 1.9;
constexpr double kFwRagged = 0.7;   // how far a started wave counts whole

template <typename T, int HD, int NR, int W, int S>
cudaError_t plan_few(const PagedAttnParams &p, int sms, FwPlan *out) {
    auto kernel = paged_few_kernel<T, HD, NR, W, S>;
    static ClusterKernel ck;
    int dev = 0;
    constexpr size_t kSmem = sizeof(FwSmem<HD, NR, W, S>);
    static_assert(kSmem <= (228 / fw_ctas(W, S) - 1) * 1024, "they fit an SM");
    cudaError_t e = cluster_prepare(ck, kernel, kSmem, &dev);
    if (e != cudaSuccess) return e;
    const long long M = (long long)p.r.max_rows * p.group, tiles = (M + 8 * NR - 1) / (8 * NR);
    long long keys = (long long)p.c.table_stride * p.c.page;   // that the table has room for: the lengths are on the device
    if (p.window > 0) keys = std::min(keys, (long long)p.window + p.n_sink + (8 * NR - 1) / p.group + 2);
    const long long units = (keys + kFwKeys - 1) / kFwKeys, clusters = tiles * p.c.n_kv_heads * p.c.n_streams;
    const double alone = kFwStep * (HD == 64 ? kFwStep64 : 1.0) * (NR == 2 ? kFwStep16 : 1.0) * (S == 2 ? kFwStepTwo : 1.0);
    const double each = kFwStepSm * (HD == 64 ? kFwStepSm64 : 1.0) * (NR == 2 ? kFwStepSm16 : 1.0);
    for (int Z = 1; Z <= 8 && Z <= units; Z++) {
        int at_once = 0;   // of what fits an SM (444, 296 and 148 CTAs by shape, without a cluster)
        if ((e = cluster_active(ck, kernel, dev, W * 32, kSmem, Z, &at_once)) != cudaSuccess) return e;
        if (at_once < 1) continue;
        const double fill = (double)clusters / at_once, most = (double)at_once * Z / sms;   // CTAs on an SM
        const double ctas = fill < 1.0 ? std::min(most, ceil((double)clusters * Z / sms)) : most;
        const double steps = (double)((units + (long long)Z * W - 1) / ((long long)Z * W)), waves = std::max(1.0, fill);
        const double t = kFwFixed + (W == 8 ? kFwEight : 0.0) + (Z > 1 ? kFwMerge : 0.0) + kFwShare * Z + kFwWave * (ceil(waves) - 1.0) +
                         steps * std::max(alone, ctas * W * each) * ((1.0 - kFwRagged) * waves + kFwRagged * ceil(waves));
        if (t < out->cost) {
            out->cost = t;
            out->shares = Z;
        }
    }
    return out->shares ? cudaSuccess : cudaErrorInvalidConfiguration;
}

template <typename T, int HD, int NR, int W, int S>
cudaError_t launch_few(PagedAttnParams p, const FwPlan &plan, cudaStream_t st, RowsPlan *only) {
    if (only) {
        *only = {8 * NR, fw_ctas(W, S), plan.shares};
        return cudaSuccess;
    }
    const long long M = (long long)p.r.max_rows * p.group, tiles = (M + 8 * NR - 1) / (8 * NR);
    p.shares = plan.shares;
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg = cluster_config(dim3((unsigned)(p.shares * tiles), p.c.n_kv_heads, p.c.n_streams), W * 32,
                                                  sizeof(FwSmem<HD, NR, W, S>), p.shares, &attr, st);
    return cudaLaunchKernelEx(&cfg, paged_few_kernel<T, HD, NR, W, S>, p);
}

// Up to this many packed rows of a stream the few-rows kernel may be faster
// (2 streams of 64 over 3016 keys 21 us; 24), beyond it tiles of 8 and 16 read the
// keys too often.
constexpr long long kFwMost = 128;

// The shapes, by their modelled times: 4 warps, two CTAs to an SM (three with heads
// of 64); 8 warps, one, where there are few CTAs (one token over 8192 keys 15.9 ->
// 14.7 us); for heads of 128 also rings of two stages, three CTAs, where there are
// many short ones (48 streams of 1000 keys 33 -> 26), and tiles of 16 rows, which
// read the keys once for more than 8 (8 streams of 32 rows over 3008 keys 32); or
// the many-rows kernel.
template <typename T, int HD>
cudaError_t launch_dim(const PagedAttnParams &p, int sms, cudaStream_t st, RowsPlan *only) {
    const long long M = (long long)p.r.max_rows * p.group;
    if (M > kFwMost) return launch_paged_attn_tc(p, st, only, nullptr);
    FwPlan two, one, three, wide;
    double many = 1e30;
    cudaError_t e;
    if ((e = plan_few<T, HD, 1, 4, 3>(p, sms, &two)) != cudaSuccess || (e = plan_few<T, HD, 1, 8, 3>(p, sms, &one)) != cudaSuccess) return e;
    if constexpr (HD == 128) {
        if ((e = plan_few<T, HD, 1, 4, 2>(p, sms, &three)) != cudaSuccess) return e;
        if (M > 8 && (e = plan_few<T, HD, 2, 4, 3>(p, sms, &wide)) != cudaSuccess) return e;
    }
    if (M > 8 && (e = launch_paged_attn_tc(p, st, nullptr, &many)) != cudaSuccess) return e;
    const double best = std::min({two.cost, one.cost, three.cost, wide.cost, many});
    if (many == best) return launch_paged_attn_tc(p, st, only, nullptr);
    if constexpr (HD == 128) {
        if (three.cost == best) return launch_few<T, HD, 1, 4, 2>(p, three, st, only);
        if (wide.cost == best) return launch_few<T, HD, 2, 4, 3>(p, wide, st, only);
    }
    if (one.cost == best) return launch_few<T, HD, 1, 8, 3>(p, one, st, only);
    return launch_few<T, HD, 1, 4, 3>(p, two, st, only);
}

template <typename T>
cudaError_t attn_typed(const PagedAttnParams &p, int sms, cudaStream_t st, RowsPlan *only) {
    return p.c.head_dim == 64 ? launch_dim<T, 64>(p, sms, st, only) : launch_dim<T, 128>(p, sms, st, only);
}

}  // namespace

cudaError_t launch_paged_attn(const PagedAttnParams &p, int sms, cudaStream_t st, RowsPlan *only) {
    return p.q_type == ELEM_BF16 ? attn_typed<__nv_bfloat16>(p, sms, st, only) : attn_typed<__half>(p, sms, st, only);
}

}  // namespace vc
