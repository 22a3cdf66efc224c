// vc_paged_attn_tc.cu - attention of many rows per stream over a paged cache in
// 8 bits, on the tcgen05 tensor cores: chunks and whole prompts.
//
// A CTA takes NT (1 or 2) tiles of 128 packed query rows (m = row * group +
// head, TMEM lane = packed row) of one (stream, KV head) and a share of the
// blocks of 64 or 128 keys that they see; the shares are a cluster.
//   4 warps per tile softmax, thread = packed row, 64 keys a step: P = 2^(s - m)
//                    of S (TMEM), rounded to fp16, over the S columns it came
//                    from; before that they load their rows of Q
//   4 warps          K and V: 16 bytes of a key to a thread, e4m3 to fp16 (exact),
//                    into the MMAs' swizzled layout, the next block's loads under
//                    way meanwhile
//   1 warp per tile  issues its MMAs by steps of 64 keys, M 128: S_t = Q_t K^T (K
//                    HD) and O_t += P_t V (N HD; A from TMEM, V an MN-major operand)
// Two tiles share each K and V block, so that its conversion (about a quarter
// of the CTA's instructions) is paid once per 256 rows.  A tile has two S ranges
// in turn: S(u + 2) goes over P(u) as soon as O has it, so that S(u + 1) waits for
// the softmax and not the softmax for it (one range of 128 keys, whose MMAs read
// Q half as often, took 527 us for the prompt chunks, this 465).
//
// Measured: prompt chunks of 1024 and 997 rows of 32 / 8 heads of 128 over 15035 and
// 8008 keys, bf16: 447 us, 0.50 of the bf16 rate - the MMA pipe is 66% busy (an S of
// 64 keys takes 48 cycles per 16 dims to read Q and K where 32 are mathematics), the
// exponential unit 46%, issue 51%, and each waits for the others; a prompt of 2000 rows
// 72 us; an encoder chunk of 1500 rows of 32 heads of 64, window 750: 59 us.
//
// All operands are fp16, whatever q's type: bf16 rows of Q are scaled by a power
// of two into its range (exact but for values 2^-29 of the row's largest), K's
// scales multiply the scores, V's the values, relative to the largest that the
// CTA sees: exact down to 2^-15 of it, where e4m3's least number is fp16's.  The
// weights are rounded to fp16, half a step of 2^-11; m is the running maximum less 7
// and moves only when a score exceeds it by 15, so that P fills the type up to 2^15
// and what is lost is 2^-32 of the row's largest weight per key.  Sums, maxima and O
// are fp32.
//
// Scales farther apart, or outside 2^-60 .. 2^60 (a page of zeros has 2^-100): a row
// goes by the scales that it sees, which may be the small ones.  A CTA that meets such
// leaves V as it is and puts its scale into the weights' exponents, with a base for P,
// the row's largest s + log2 vs, and one for the weights' sum, its largest s.  That is
// two 2^x for each score: the prompt chunks take 930 us so, the encoder chunk 131.
// One loop for both cases, with the sums of P brought to weights by groups of 16
// keys, cost the ordinary case 20% (spills, and MMA operands that left their uniform
// registers).
//
// Zero times a masked key's NaN would be NaN: in blocks that some row does not
// see whole, the converting threads put zeros in the place of NaN in V and set a
// flag, and the rows that do see them get NaN at the end.
#include "vc_attn_tc.cuh"
#include "vc_cluster.h"
#include "vc_paged.cuh"

#include <algorithm>

namespace vc {

using namespace tc;

namespace {

constexpr int kPtHalf = 64;             // keys per softmax step
constexpr int kPtConv = 128;            // threads that convert K and V
constexpr int kPtStages = 2;
constexpr int pt_keys(int nt) { return nt == 1 ? 64 : 128; }
constexpr int pt_ctas(int nt) { return nt == 1 ? 2 : 1; }
constexpr int pt_threads(int nt) { return nt * kAtRows + kPtConv + nt * 32; }
constexpr uint64_t kPtWaitNs = 2000000000ull, kPtBlockNs = 10000ull;   // a CTA's waits end after this, per block as well
constexpr float kPtBelow = 7.f;         // the maximum less m
constexpr float kPtAbove = 15.f;        // log2 of what a weight may reach before m moves
constexpr int kPtOneCta = 120 * 1024;   // more than half an SM's shared memory: one CTA per SM

template <int HD, int NT>
struct PtSmem {
    static constexpr int kKeys = pt_keys(NT);
    // Q, K and V tiles are HD / 64 sub-tiles of [rows or keys][128 bytes]
    static constexpr int kTile = kKeys * HD * 2, kSubTile = kKeys * 128, kQTile = kAtRows * HD * 2, kQSub = kAtRows * 128;
    static constexpr int kO = NT * kAtRows * HD * 4;   // bytes of O in fp32, over K and V at the end
    unsigned char q[NT][kQTile];
    union {
        unsigned char kv[2][kPtStages][kTile];         // K, V
        unsigned char o[kO];
    };
    float mx[NT * kAtRows], sum[NT * kAtRows], factor[NT * kAtRows];
    uint64_t q_full[NT], k_full[kPtStages], k_empty[kPtStages], v_full[kPtStages], v_empty[kPtStages];
    uint64_t s_full[NT][2], p_full[NT][2], o_part[NT], o_done[NT];   // [2]: by S range
    uint32_t tmem;
    int v_top, v_least;   // V's largest scale and its least but 0, as the bits of floats >= 0
    int bad;      // a masked block holds NaN in V
    int failed;   // some warp's wait ran out: the CTA's rows are void
    uint64_t stall;   // nothing arrives here
};

__device__ __forceinline__ float max3(float a, float b, float c) {   // a NaN is passed over
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// The weights of 64 keys of a row: w = 2^(s f - base) as pairs of fp16, ls their
// sum before rounding; the largest s f - base as the result.  f: the row's factor
// times K's scale, by groups of 16 keys in the warp's lanes.  The next 16 scores
// are on their way from TMEM while 16 are worked on.  (2^x on the FMA pipe for
// some of the pairs, which the exponential unit's 8 cycles a warp suggest, costs
// more issue slots than it saves: 3 of 8 pairs 601 against 531 us for the prompt
// chunks of 15035 and 8008 keys.)
template <bool MASKED>
__device__ __forceinline__ float weigh64(uint32_t ts, float sl2, float ks, int g0, float base, const uint32_t (&vis)[2], uint32_t (&w)[32],
                                          float &ls) {
    float mx = -INFINITY;
    uint64_t rs[2] = {0, 0};
    const uint64_t nb = pair(-base, -base);
    uint32_t ra[16], rb[16];
    tmem_ld16_async(ts, ra);
#pragma unroll
    for (int c = 0; c < 64; c += 16) {
        uint32_t(&cur)[16] = (c & 16) ? rb : ra;
        const float f = sl2 * __shfl_sync(0xffffffffu, ks, g0 + c / 16);
        const uint64_t sl = pair(f, f);
        tmem_ld_wait(cur);
        if (c + 16 < 64) tmem_ld16_async(ts + c + 16, (c & 16) ? ra : rb);
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
            float xa, xb;
            unpair(fma2(pair(__uint_as_float(cur[j]), __uint_as_float(cur[j + 1])), sl, nb), xa, xb);
            if (MASKED) {
                xa = vis[c / 32] & (1u << ((c & 16) + j)) ? xa : -INFINITY;
                xb = vis[c / 32] & (2u << ((c & 16) + j)) ? xb : -INFINITY;
            }
            mx = max3(mx, xa, xb);
            xa = exp2_approx(xa);
            xb = exp2_approx(xb);
            rs[(j >> 1) & 1] = add2(rs[(j >> 1) & 1], pair(xa, xb));
            w[(c + j) >> 1] = pack2<__half>(xa, xb);
        }
    }
    float a, b;
    unpair(add2(rs[0], rs[1]), a, b);
    ls = a + b;
    return mx;
}

// The same where V's scales stand far apart: P 2^(s f + log2 vs - p_base), weights 2^(s f - l_base), both bases the row's
// own.  lv: log2 vs, as ks.
struct Tops {
    float l, p;   // the largest s f, the largest s f + log2 vs
};
__device__ __forceinline__ Tops weigh64_far(uint32_t ts, float sl2, float ks, float lv, int g0, float l_base, float p_base,
                                             const uint32_t (&vis)[2], uint32_t (&w)[32], float &ls) {
    Tops top = {-INFINITY, -INFINITY};
    ls = 0.f;
#pragma unroll
    for (int c = 0; c < 64; c += 16) {
        uint32_t r[16];
        tmem_ld16_async(ts + c, r);
        const float f = sl2 * __shfl_sync(0xffffffffu, ks, g0 + c / 16), v = __shfl_sync(0xffffffffu, lv, g0 + c / 16);
        float most = -INFINITY;
        tmem_ld_wait(r);
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
            const float xa = vis[c / 32] & (1u << ((c & 16) + j)) ? __uint_as_float(r[j]) * f : -INFINITY;
            const float xb = vis[c / 32] & (2u << ((c & 16) + j)) ? __uint_as_float(r[j + 1]) * f : -INFINITY;
            most = max3(most, xa, xb);
            ls += exp2_approx(xa - l_base) + exp2_approx(xb - l_base);
            w[(c + j) >> 1] = pack2<__half>(exp2_approx(xa + (v - p_base)), exp2_approx(xb + (v - p_base)));
        }
        top.l = fmaxf(top.l, most);
        top.p = fmaxf(top.p, most + v);
    }
    return top;
}

// The softmax of a warp's 32 rows over a CTA's keys where V's scales stand far apart:
// the steps, waits and TMEM of the kernel's own loop.
struct FarArgs {
    const int *table;                     // the stream's
    const float *k_scale, *v_scale;       // of page 0, by n_kv_heads
    int n_pages, page_shift, n_kv_heads;
    int b0, nb, sink_blocks, first;       // the CTA's blocks
    int lo, hi, ns;                       // positions that its rows see
    int at, e1, s2;                       // the row's, [0, e1) and [s2, at]
    int gap, on, end;                     // steps that the tile leaves out: [gap, on), [end, ..)
    float sl2;
    uint32_t s_tmem, o_tmem;              // S ranges and O of the warp's lanes
    int t;
    uint64_t deadline;
};
struct FarResult {
    float l, base, unit;   // the weights' sum, in [1, 2), and its base; O's unit for it
    uint32_t turns;        // steps taken
    bool ok;
};
template <int HD, int NT>
__device__ __forceinline__ FarResult weigh_far(PtSmem<HD, NT> &sh, const FarArgs &a) {
    constexpr int kKeys = pt_keys(NT), kSteps = kKeys / kPtHalf, kGroups = kKeys / 16;
    const int lane = threadIdx.x & 31;
    FarResult r = {0.f, -INFINITY, 0.f, 0u, true};
    float p_base = -INFINITY;
    uint32_t phase = 0u;
    for (int b = 0; b < a.nb; b++) {
        const int key = (a.b0 + b < a.sink_blocks ? a.b0 + b : a.first + a.b0 + b - a.sink_blocks) * kKeys, mine = key + 16 * lane;
        const int g = lane < kGroups && mine < a.hi && (mine + 16 > a.lo || mine < a.ns) ? __ldg(a.table + (mine >> a.page_shift)) : -1;
        const bool page = g >= 0 && g < a.n_pages;
        const uint32_t there = __ballot_sync(0xffffffffu, page);
        const float ks = page ? __ldg(a.k_scale + (long long)g * a.n_kv_heads) : 0.f;
        const float lv = log2f(page ? __ldg(a.v_scale + (long long)g * a.n_kv_heads) : 0.f);   // (exact for powers of two; 0: -inf)
#pragma unroll 1
        for (int h = 0; h < kSteps; h++) {
            const int c0 = key + h * kPtHalf, u = b * kSteps + h;
            if ((u >= a.gap && u < a.on) || u >= a.end) continue;
            const uint32_t ts = a.s_tmem + (u & 1) * kPtHalf, pages = (there >> (4 * h)) & 15u;
            if (!warp_wait(&sh.s_full[a.t][u & 1], (phase >> (u & 1)) & 1u, a.deadline)) r.ok = false;
            phase ^= 1u << (u & 1);
            tc_fence_after();
            uint32_t vis[2], w[32];
#pragma unroll
            for (int e = 0; e < 2; e++)
                vis[e] = (range_bits(c0 + 32 * e, 0, a.e1) | range_bits(c0 + 32 * e, a.s2, a.at + 1)) &
                         ((pages >> (2 * e) & 1u ? 0xffffu : 0u) | (pages >> (2 * e) & 2u ? 0xffff0000u : 0u));
            float factor = 1.f, ls;
            bool moved = false;
#pragma unroll 1
            for (;;) {
                const Tops top = weigh64_far(ts, a.sl2, ks, lv, 4 * h, r.base == -INFINITY ? 0.f : r.base,
                                             p_base == -INFINITY ? 0.f : p_base, vis, w, ls);
                const bool sum = top.l > r.base + kPtAbove, move = top.p > p_base + kPtAbove;   // (-inf: nothing yet)
                if (moved || !__any_sync(0xffffffffu, sum || move)) break;
                moved = true;
                if (sum) {
                    const float base = ceilf(top.l);
                    r.l *= exp2f(r.base - base);
                    r.base = base;
                }
                if (move) {
                    const float base = top.p - kPtBelow;
                    factor = exp2f(p_base - base);
                    p_base = base;
                }
            }
            r.l += ls;
            tmem_st32_async(ts, w);   // over S
            if (moved && r.turns > 0) {
                // O must hold the P before these: the step before this one may be under way
                if (!warp_wait(&sh.o_part[a.t], (r.turns - 1) & 1u, a.deadline)) r.ok = false;
                tc_fence_after();
#pragma unroll 1
                for (int c = 0; c < HD; c += 32) {
                    float o[32];
                    tmem_ld32(a.o_tmem + c, o);
#pragma unroll
                    for (int j = 0; j < 32; j++) o[j] *= factor;
                    tmem_st32(a.o_tmem + c, o);
                }
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.p_full[a.t][u & 1]);
            r.turns++;
        }
    }
    // to a sum in [1, 2), and O with it, so that no product leaves fp32
    const int up = r.l > 0.f && r.l < INFINITY ? (int)(__float_as_uint(r.l) >> 23) - 127 : 0;
    const float down = __uint_as_float((uint32_t)(127 - up) << 23);
    r.unit = p_base == -INFINITY ? 0.f : exp2f(p_base - r.base);
    r.l *= down;
    r.base += (float)up;
    if (r.turns > 0) {
        if (!warp_wait(&sh.o_done[a.t], 0u, a.deadline)) r.ok = false;
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < HD; c += 32) {
            float o[32];
            tmem_ld32(a.o_tmem + c, o);
#pragma unroll
            for (int j = 0; j < 32; j++) o[j] *= down;
            tmem_st32(a.o_tmem + c, o);
        }
    }
    return r;
}

// As a call, so that its registers are not the kernel's.  That suits one tile (8 streams
// of 32 rows over 3008 keys, which never come here, 43.7 us, without the call 45.0; encoder
// chunk 58.8, 60.0), two tiles not (whole prompts 89.7, 87.5): what lives across the call
// weighs on a CTA's start and end.
template <int HD, int NT>
__device__ __noinline__ FarResult weigh_far_call(PtSmem<HD, NT> &sh, const FarArgs a) {
    return weigh_far<HD, NT>(sh, a);
}

// The stream that reaches n-th farthest (of up to 32; of more simply the n-th): a
// warp's lanes each have one.  Prompt chunks over 15035 and 8008 keys: 456 us, with
// the streams in turn 575.
__device__ __forceinline__ int nth_longest(const PagedAttnParams &p, int n, int lane) {
    const int streams = p.c.n_streams;
    if (streams > 32) return n;
    int end = -1, rank = 0;
    if (lane < streams) {
        const RowSpan s = paged_span(p.r, p.c, lane);
        end = s.n > 0 ? s.pos + s.n : 0;
    }
    for (int i = 0; i < streams; i++) {
        const int other = __shfl_sync(0xffffffffu, end, i);
        rank += other > end || (other == end && i < lane);
    }
    return __ffs(__ballot_sync(0xffffffffu, lane < streams && rank == n)) - 1;
}

template <typename T, int HD, int NT>
__global__ void __launch_bounds__(pt_threads(NT), pt_ctas(NT)) paged_many_kernel(const PagedAttnParams p) {
    using Sm = PtSmem<HD, NT>;
    constexpr int kSub = HD / 64;            // 64-dim sub-tiles of a tile
    constexpr int kWarpConv = NT * 4, kWarpMma = kWarpConv + kPtConv / 32;
    constexpr int kThreads = pt_threads(NT), kKeys = Sm::kKeys, kSteps = kKeys / kPtHalf, kGroups = kKeys / 16;
    // Steps that a tile's rows do not see are left out, and masks are applied by
    // warp: for heads of 64, an encoder's, whose tiles are long (a row per
    // position) and windows short: its chunk 69 -> 62 us.  The registers that this
    // takes cost heads of 128, where a group's heads share positions, more than it
    // gives (prompt chunks 454 -> 490 us).
    constexpr bool kSkip = HD == 64;
    constexpr uint32_t kTmemCols = NT == 2 ? 512 : 256;
    constexpr uint32_t kOCol = NT * 2 * kPtHalf;   // S ranges first, two a tile, then O tiles
    extern __shared__ __align__(1024) unsigned char pt_smem_raw[];
    Sm &sh = *reinterpret_cast<Sm *>(pt_smem_raw);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // CTAs in order: the streams that reach farthest, their later tiles first - in a
    // prompt those see the most - so that what starts last ends soon
    const int Z = p.shares, z = blockIdx.x % Z;
    const unsigned nth = blockIdx.x / Z, of = nth / p.c.n_kv_heads;
    const int kvh = nth % p.c.n_kv_heads, m0 = (p.tiles - 1 - (int)(of % p.tiles)) * (NT * kAtRows);
    const int stream = nth_longest(p, of / p.tiles, lane);
    const RowSpan s = paged_span(p.r, p.c, stream);
    const int M = s.n * p.group;
    if (m0 >= M) return;   // the whole cluster leaves
    const int i0 = m0 / p.group, i1 = (min(m0 + NT * kAtRows, M) - 1) / p.group;
    // positions that some row sees: [0, ns) and [lo, hi)
    const int p_min = s.pos + i0, p_max = s.pos + i1, hi = p_max + 1, ns = min(p.n_sink, hi);
    const int lo = p.window > 0 ? max(0, p_min - p.window + 1) : 0;
    const int sink_blocks = (ns + kKeys - 1) / kKeys, first = max(lo / kKeys, sink_blocks);
    const int blocks = sink_blocks + max(0, (hi + kKeys - 1) / kKeys - first);
    const int b0 = (int)((long long)z * blocks / Z), nb = (int)((long long)(z + 1) * blocks / Z) - b0;
    const int tiles = M - m0 > kAtRows ? NT : 1;   // tiles with rows
    const int head0 = kvh * p.group;
    auto key_of = [&](int b) { return (b0 + b < sink_blocks ? b0 + b : first + b0 + b - sink_blocks) * kKeys; };
    // every row sees the block's positions
    auto whole = [&](int key) {
        return key + kKeys - 1 <= p_min && (p.window <= 0 || key > p_max - p.window || key + kKeys <= p.n_sink);
    };
    // the table's entry for 16 positions, -1: no row sees them; whether it is a
    // page is asked where it is used, blocks later, so that nothing waits for it here
    const int *const table = p.c.table + (long long)stream * p.c.table_stride;
    auto entry_of = [&](int key) { return key < hi && (key + 16 > lo || key < ns) ? __ldg(table + (key >> p.c.page_shift)) : -1; };
    auto is_page = [&](int g) { return g >= 0 && g < p.c.n_pages; };
    // Steps of 64 keys: half u % kSteps of block u / kSteps.  A tile leaves out
    // those that none of its rows sees: [gap, on) between the sinks and the window,
    // and from `end` on.
    const int steps = nb * kSteps;
    struct Steps {
        int gap, on, end;
        __device__ bool left_out(int u) const { return (u >= gap && u < on) || u >= end; }
    };
    auto steps_below = [&](int key) {   // steps whose first key is less
        const int c = (max(key, 0) + kPtHalf - 1) / kPtHalf;
        const int all = min(c, sink_blocks * kSteps) + max(0, min(c, first * kSteps + (blocks - sink_blocks) * kSteps) - first * kSteps);
        return min(max(all - b0 * kSteps, 0), steps);
    };
    auto steps_of = [&](int t) {
        const int a = s.pos + (m0 + t * kAtRows) / p.group, b = s.pos + (min(m0 + (t + 1) * kAtRows, M) - 1) / p.group;
        Steps st = {0, 0, steps_below(b + 1)};
        if (p.window > 0) {
            st.gap = steps_below(p.n_sink);
            st.on = max(st.gap, steps_below(a - p.window + 1 - (kPtHalf - 1)));
        }
        return st;
    };
    bool ok = true;
    // V's scales do not fit fp16 beside one another, or their products fp32 (once they have been looked through)
    auto far_apart = [&] {
        const float top = __int_as_float(*(volatile int *)&sh.v_top), least = __int_as_float(*(volatile int *)&sh.v_least);
        return top > 0.f && (least < top * 0x1p-15f || top > 0x1p60f || top < 0x1p-60f);
    };

    if (threadIdx.x == 0) {
        for (int i = 0; i < kPtStages; i++) {
            mbar_init(&sh.k_full[i], kPtConv / 32);
            mbar_init(&sh.v_full[i], kPtConv / 32);
            mbar_init(&sh.k_empty[i], tiles);
            mbar_init(&sh.v_empty[i], tiles);
        }
        for (int t = 0; t < NT; t++) {
            const int warps = max(1, min(4, (M - m0 - t * kAtRows + 31) / 32));   // of the tile, with rows
            mbar_init(&sh.q_full[t], warps);
            mbar_init(&sh.p_full[t][0], warps);
            mbar_init(&sh.p_full[t][1], warps);
            mbar_init(&sh.s_full[t][0], 1);
            mbar_init(&sh.s_full[t][1], 1);
            mbar_init(&sh.o_part[t], 1);
            mbar_init(&sh.o_done[t], 1);
        }
        mbar_init(&sh.stall, 1);
        sh.v_top = sh.bad = sh.failed = 0;
        sh.v_least = 0x7f800000;   // infinity
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kWarpMma) {
        tmem_alloc(&sh.tmem, kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    const uint64_t deadline = globaltimer() + kPtWaitNs + (uint64_t)nb * kPtBlockNs;   // (TMEM may have been another kernel's)

    if (warp >= kWarpConv && warp < kWarpMma) {
        // ---- K and V ----
        constexpr int kRowsAtOnce = kPtConv * 16 / HD, kLoads = kKeys / kRowsAtOnce;
        // a thread's 16 dims of a row, so that the lanes of a store meet no bank twice
        const int tid = threadIdx.x - kWarpConv * 32;
        const int r0 = HD == 128 ? ((tid >> 4) << 1 | ((tid >> 2) & 1)) : tid >> 2, sub = HD == 128 ? (tid >> 3) & 1 : 0, ch = tid & 3;
        const long long mine = (r0 & 15) * p.c.slot_stride + sub * 64 + ch * 16;
        uint4 k_raw[kLoads], v_raw[kLoads];
        // lane g has the place of a block's positions 16 g .. and V's scale of
        // their page; the threads that load them ask for it
        struct Place {
            long long off;   // -1: no page
            float vs;
        };
        const long long base = page_base(p.c, p.layer, 0, kvh), scale0 = scale_at(p.c, p.layer, 0, kvh);
        auto entry = [&](int b) { return b < nb && lane < kGroups ? entry_of(key_of(b) + 16 * lane) : -1; };
        auto place = [&](int b, int g) {
            Place at = {-1, 0.f};
            if (is_page(g)) {
                at.off = base + (long long)g * p.c.page_stride + ((key_of(b) + 16 * lane) & (p.c.page - 1)) * p.c.slot_stride;
                at.vs = __ldg(p.c.v_scale + scale0 + (long long)g * p.c.n_kv_heads);
            }
            return at;
        };
        auto group = [&](int i) { return HD == 128 ? i : 2 * i + (r0 >> 4); };   // of the thread's load i
        auto load = [&](const unsigned char *pool, const Place &at, uint4 (&raw)[kLoads]) {
#pragma unroll
            for (int i = 0; i < kLoads; i++) {
                raw[i] = make_uint4(0u, 0u, 0u, 0u);
                const long long off = __shfl_sync(0xffffffffu, at.off, group(i));
                if (off >= 0) raw[i] = __ldg(reinterpret_cast<const uint4 *>(pool + off + mine));
            }
        };
        auto put = [&](unsigned char *tile, int r, const uint4 &u, __half2 by, bool scaled) {
            const uint32_t in[4] = {u.x, u.y, u.z, u.w};
            uint32_t out[8];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                __half2 a = from_e4m3x2(in[e] & 0xffffu), b = from_e4m3x2(in[e] >> 16);
                if (scaled) {
                    a = __hmul2(a, by);
                    b = __hmul2(b, by);
                }
                out[2 * e] = *reinterpret_cast<const uint32_t *>(&a);
                out[2 * e + 1] = *reinterpret_cast<const uint32_t *>(&b);
            }
            unsigned char *const row = tile + sub * Sm::kSubTile + r * 128;
            *reinterpret_cast<uint4 *>(row + (((2 * ch) ^ (r & 7)) << 4)) = make_uint4(out[0], out[1], out[2], out[3]);
            *reinterpret_cast<uint4 *>(row + (((2 * ch + 1) ^ (r & 7)) << 4)) = make_uint4(out[4], out[5], out[6], out[7]);
        };
        Place here = place(0, entry(0));
        load(p.c.k, here, k_raw);
        load(p.c.v, here, v_raw);
        int next = entry(1);
        {   // the largest scale of V and the least
            const int step = min(p.c.page, kKeys), n = nb * (kKeys / step);
            float top = 0.f, least = INFINITY;
            for (int i = tid; i < n; i += kPtConv) {
                int key = key_of(i / (kKeys / step)) + i % (kKeys / step) * step;
                // a page's first positions may be among those that nobody sees
                const bool seen = key < hi && (key + step > lo || key < ns);
                const int g = seen ? page_at(p.c, stream, key >> p.c.page_shift) : -1;
                const float v = g >= 0 ? __ldg(p.c.v_scale + scale_at(p.c, p.layer, g, kvh)) : 0.f;
                top = fmaxf(top, v);
                least = fminf(least, v > 0.f ? v : INFINITY);
            }
            const int most = __reduce_max_sync(0xffffffffu, __float_as_int(top)), few = __reduce_min_sync(0xffffffffu, __float_as_int(least));
            if (lane == 0) {
                atomicMax(&sh.v_top, most);
                atomicMin(&sh.v_least, few);
            }
            asm volatile("bar.sync 1, %0;" ::"n"(kPtConv) : "memory");
            asm volatile("bar.arrive 2, %0;" ::"n"(kPtConv + NT * kAtRows) : "memory");
        }
        const float v_top = __int_as_float(*(volatile int *)&sh.v_top), inv_top = v_top > 0.f ? 1.0f / v_top : 0.f;
        const bool apart = far_apart();
        for (int b = 0; b < nb; b++) {
            const int st = b % kPtStages;
            const uint32_t back = (b / kPtStages + 1) & 1u;
            const int key = key_of(b);
            if (b >= kPtStages && !warp_wait(&sh.k_empty[st], back, deadline)) {
                ok = false;
                break;
            }
#pragma unroll
            for (int i = 0; i < kLoads; i++) put(sh.kv[0][st], i * kRowsAtOnce + r0, k_raw[i], __half2(), false);
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.k_full[st]);
            const Place then = place(b + 1, next);
            load(p.c.k, then, k_raw);
            if (b >= kPtStages && !warp_wait(&sh.v_empty[st], back, deadline)) {
                ok = false;
                break;
            }
            if (!whole(key)) {
                bool found = false;
#pragma unroll
                for (int i = 0; i < kLoads; i++) {
                    uint4 &u = v_raw[i];
                    const uint4 n = make_uint4(__vcmpeq4(u.x & 0x7f7f7f7fu, 0x7f7f7f7fu), __vcmpeq4(u.y & 0x7f7f7f7fu, 0x7f7f7f7fu),
                                               __vcmpeq4(u.z & 0x7f7f7f7fu, 0x7f7f7f7fu), __vcmpeq4(u.w & 0x7f7f7f7fu, 0x7f7f7f7fu));
                    const int j = key + i * kRowsAtOnce + r0;   // (what nobody sees, a page's unwritten end, needs no flag)
                    found |= (n.x | n.y | n.z | n.w) != 0u && j < hi && (j >= lo || j < ns);
                    u = make_uint4(u.x & ~n.x, u.y & ~n.y, u.z & ~n.z, u.w & ~n.w);
                }
                if (found) atomicExch(&sh.bad, 1);
            }
#pragma unroll
            for (int i = 0; i < kLoads; i++)
                put(sh.kv[1][st], i * kRowsAtOnce + r0, v_raw[i],
                    __float2half2_rn(apart ? 1.0f : __shfl_sync(0xffffffffu, here.vs, group(i)) * inv_top), true);
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.v_full[st]);
            load(p.c.v, then, v_raw);
            here = then;
            next = entry(b + 2);
        }
    } else if (warp >= kWarpMma) {
        // ---- the MMAs of tile t ----
        const int t = warp - kWarpMma;
        if (nb > 0 && t < tiles) {
            const uint32_t lead = lane == 0, tm = __shfl_sync(0xffffffffu, tmem, 0);
            constexpr uint32_t id_s = at_idesc<__half>(kPtHalf, false), id_o = at_idesc<__half>(HD, true);
            // Step u has S range u % 2.  Operands depend on u alone, which counts,
            // and what is left out is issued by no lane, not branched around: where
            // the compiler cannot see that all lanes have the same, each MMA costs
            // moves to uniform registers (60 us of 450 for the prompt chunks).
            const Steps st = steps_of(t);
            auto issue_s = [&](int u, uint32_t lead) {
                const int b = u / kSteps, h = u % kSteps;
                const uint64_t a0 = smem_desc_sw128(sh.q[t]), k0 = smem_desc_sw128(sh.kv[0][b % kPtStages]) + h * (kPtHalf * 128 / 16);
#pragma unroll
                for (int d = 0; d < kSub; d++)
#pragma unroll
                    for (int k = 0; k < 4; k++)   // 16 dims: +32 bytes
                        warp_mma(tm + (t * 2 + (u & 1)) * kPtHalf, a0 + d * (Sm::kQSub / 16) + 2 * k, k0 + d * (Sm::kSubTile / 16) + 2 * k,
                                 id_s, (d | k) != 0 ? 1u : 0u, lead);
                warp_commit(&sh.s_full[t][u & 1], lead);
            };
            auto issue_o = [&](int u, bool more, uint32_t lead) {   // O += P V
                const int b = u / kSteps, h = u % kSteps;
                const uint64_t v0 = at_desc_mn(sh.kv[1][b % kPtStages], Sm::kSubTile) + h * (kPtHalf * 128 / 16);
#pragma unroll
                for (int k = 0; k < kPtHalf / 16; k++)   // 16 keys: 8 columns of P, 2048 bytes of V
                    warp_mma_ta(tm + kOCol + t * HD, tm + (t * 2 + (u & 1)) * kPtHalf + 8 * k, v0 + k * (2048 / 16), id_o,
                                more || k != 0 ? 1u : 0u, lead);
                warp_commit(&sh.o_part[t], lead);
            };
            uint32_t phase = 0u;   // bit r: of p_full[t][r]
            bool more = false;     // O holds something
            ok = warp_wait(&sh.q_full[t], 0u, deadline);
            for (int u = -2; u < steps && ok; u++) {
                const int b = u / kSteps, s2 = u + 2, bs = s2 / kSteps;
                if (u >= 0) {
                    if (u % kSteps == 0) ok = warp_wait(&sh.v_full[b % kPtStages], (b / kPtStages) & 1u, deadline);
                    const bool take = !kSkip || !st.left_out(u);
                    if (take) {
                        ok = ok && warp_wait(&sh.p_full[t][u & 1], kSkip ? (phase >> (u & 1)) & 1u : (u >> 1) & 1u, deadline);
                        phase ^= 1u << (u & 1);
                    }
                    if (!ok) break;
                    tc_fence_after();
                    issue_o(u, kSkip ? more : u > 0, take ? lead : 0u);
                    more |= take;
                    if (u % kSteps == kSteps - 1) warp_commit(&sh.v_empty[b % kPtStages], lead);
                }
                if (ok && s2 < steps) {   // S of the second step on, over P(u) and behind the MMAs that read it
                    if (s2 % kSteps == 0) ok = warp_wait(&sh.k_full[bs % kPtStages], (bs / kPtStages) & 1u, deadline);
                    if (!ok) break;
                    tc_fence_after();
                    issue_s(s2, kSkip && st.left_out(s2) ? 0u : lead);
                    if (s2 % kSteps == kSteps - 1) warp_commit(&sh.k_empty[bs % kPtStages], lead);
                }
            }
            warp_commit(&sh.o_done[t], lead);
        }
        if (p.stall_ns && t == 0) ok = warp_wait(&sh.stall, 0u, globaltimer() + p.stall_ns) && ok;
    } else {
        // ---- softmax: thread = packed row ----
        const int t = warp / 4, q = warp % 4, ml = t * kAtRows + 32 * q + lane, m = m0 + ml;
        const bool here = m0 + t * kAtRows + 32 * q < M;   // the warp has rows
        if (!here) asm volatile("bar.arrive 2, %0;" ::"n"(kPtConv + NT * kAtRows) : "memory");
        if (here) {
            const int i = min(m, M - 1) / p.group, at = s.pos + i;
            const long long row = (long long)(s.r0 + i) * p.n_heads + head0 + min(m, M - 1) % p.group;
            {   // the warp's 32 rows of Q as fp16: HD / 8 lanes a row, zeros past M; all on their way at once
                constexpr int kCh = HD / 8, kAtOnce = 32 / kCh, kIts = 32 / kAtOnce;
                const int ch = lane % kCh;
                unsigned char *const to = sh.q[t] + (ch >> 3) * Sm::kQSub;
                uint4 raw[kIts];
#pragma unroll
                for (int it = 0; it < kIts; it++) {
                    const int r = it * kAtOnce + lane / kCh;
                    const long long from = __shfl_sync(0xffffffffu, row, r);
                    raw[it] = make_uint4(0u, 0u, 0u, 0u);
                    if (m0 + t * kAtRows + 32 * q + r < M)
                        raw[it] = *reinterpret_cast<const uint4 *>(static_cast<const T *>(p.q) + from * HD + ch * 8);
                }
#pragma unroll
                for (int it = 0; it < kIts; it++) {
                    const int rt = 32 * q + it * kAtOnce + lane / kCh;
                    uint4 u = raw[it];
                    float up = 1.f;   // a power of two that takes the row's largest to [2^14, 2^15)
                    if constexpr (!std::is_same<T, __half>::value) {
                        const uint32_t in[4] = {u.x, u.y, u.z, u.w};
                        float v[8], big = 0.f;
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const float2 f = unpack2<T>(in[e]);
                            v[2 * e] = f.x;
                            v[2 * e + 1] = f.y;
                        }
#pragma unroll
                        for (int e = 0; e < 8; e++) big = fmaxf(big, fabsf(v[e]) < INFINITY ? fabsf(v[e]) : 0.f);
#pragma unroll
                        for (int o = kCh / 2; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
                        const int e = (int)(__float_as_uint(big) >> 23) - 127;
                        up = big > 0.f ? __uint_as_float((uint32_t)(min(14 - e, 126) + 127) << 23) : 1.f;
                        u = make_uint4(pack2<__half>(v[0] * up, v[1] * up), pack2<__half>(v[2] * up, v[3] * up),
                                       pack2<__half>(v[4] * up, v[5] * up), pack2<__half>(v[6] * up, v[7] * up));
                    }
                    *reinterpret_cast<uint4 *>(to + rt * 128 + (((ch & 7) ^ (rt & 7)) << 4)) = u;
                    if (ch == 0) sh.factor[t * kAtRows + rt] = p.scale_log2 / up;
                }
            }
            // positions that the row sees: [0, e1) and [s2, at]
            const int e1 = min(ns, at + 1), s2 = p.window > 0 ? max(0, at - p.window + 1) : 0;
            const uint32_t tl = tmem + ((uint32_t)(32 * q) << 16);
            const uint32_t to = tl + kOCol + t * HD;
            float mr = -INFINITY, l = 0.f;
            float sv[32];
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.q_full[t]);
            const float sl2 = sh.factor[ml];
            // lane g: table entry and K's scale of a block's positions 16 g ..
            auto entry = [&](int b) { return b < nb && lane < kGroups ? entry_of(key_of(b) + 16 * lane) : -1; };
            auto scale = [&](int g) { return is_page(g) ? __ldg(p.c.k_scale + scale_at(p.c, p.layer, g, kvh)) : 0.f; };
            int page = entry(0), page_next = entry(1);
            float ks = scale(page);
            const Steps st = kSkip ? steps_of(t) : Steps{};
            const int w_min = __shfl_sync(0xffffffffu, at, 0), w_max = __shfl_sync(0xffffffffu, at, 31);
            uint32_t phase = 0u, turns = 0u;   // bit r: of s_full[t][r]; steps taken
            float unit;                        // of O
            asm volatile("bar.sync 2, %0;" ::"n"(kPtConv + NT * kAtRows) : "memory");   // V's scales have been looked through
            if (far_apart()) {
                const long long scale0 = scale_at(p.c, p.layer, 0, kvh);
                const FarArgs args = {table, p.c.k_scale + scale0, p.c.v_scale + scale0, p.c.n_pages, p.c.page_shift, p.c.n_kv_heads, b0, nb,
                                      sink_blocks, first, lo, hi, ns, at, e1, s2, st.gap, st.on, kSkip ? st.end : INT_MAX, sl2,
                                      tl + t * 2 * kPtHalf, to, t, deadline};
                FarResult r;
                if constexpr (NT == 1) r = weigh_far_call<HD, NT>(sh, args);
                else r = weigh_far<HD, NT>(sh, args);
                l = r.l;
                mr = r.base;
                unit = r.unit;
                turns = r.turns;
                ok = r.ok;
            } else {
                unit = __int_as_float(*(volatile int *)&sh.v_top);
                for (int b = 0; b < nb; b++) {
                    const int key = key_of(b);
                    const uint32_t there = __ballot_sync(0xffffffffu, is_page(page));
                    const bool all = !kSkip && whole(key) && there == (1u << kGroups) - 1;   // the CTA's rows see the whole block
                    const float ks_now = ks;
                    page = page_next;
                    ks = scale(page);
                    page_next = entry(b + 2);
#pragma unroll 1
                    for (int h = 0; h < kSteps; h++) {
                        const int c0 = key + h * kPtHalf;
                        const int u = b * kSteps + h;
                        if (kSkip && st.left_out(u)) continue;
                        const uint32_t ts = tl + (t * 2 + (u & 1)) * kPtHalf, pages = (there >> (4 * h)) & 15u;
                        const bool full = !kSkip ? all
                                                 : c0 + kPtHalf - 1 <= w_min && pages == 15u &&
                                                       (p.window <= 0 || c0 > w_max - p.window || c0 + kPtHalf <= p.n_sink);
                        if (!warp_wait(&sh.s_full[t][u & 1], kSkip ? (phase >> (u & 1)) & 1u : (u >> 1) & 1u, deadline)) ok = false;
                        phase ^= 1u << (u & 1);
                        tc_fence_after();
                        uint32_t vis[2] = {0u, 0u};
                        if (!full)
#pragma unroll
                            for (int e = 0; e < 2; e++)
                                vis[e] = (range_bits(c0 + 32 * e, 0, e1) | range_bits(c0 + 32 * e, s2, at + 1)) &
                                         ((pages >> (2 * e) & 1u ? 0xffffu : 0u) | (pages >> (2 * e) & 2u ? 0xffff0000u : 0u));
                        // P against m so far; a row whose keys exceed it by 2^15 takes
                        // theirs, and the warp goes over them again (S is intact until P
                        // is stored)
                        uint32_t w[32];
                        float base = mr == -INFINITY ? 0.f : mr, factor = 1.f, ls = 0.f;
                        float over;   // the largest less base
                        bool moved = false;
#pragma unroll 1
                        for (;;) {    // (one copy of its code)
                            over = full ? weigh64<false>(ts, sl2, ks_now, 4 * h, base, vis, w, ls)
                                        : weigh64<true>(ts, sl2, ks_now, 4 * h, base, vis, w, ls);
                            const bool move = mr == -INFINITY ? over > -INFINITY : over > kPtAbove;
                            if (moved || !__any_sync(0xffffffffu, move)) break;
                            moved = true;
                            if (move) {
                                const float mn = base + over - kPtBelow;
                                factor = mr == -INFINITY ? 0.f : exp2_approx(mr - mn);
                                mr = base = mn;
                                l *= factor;
                            }
                        }
                        l += ls;
                        tmem_st32_async(ts, w);       // over S
                        if (moved && (kSkip ? turns : u) > 0) {
                            // O must hold the weights before these: the step before
                            // this one may be under way
                            if (!warp_wait(&sh.o_part[t], ((kSkip ? turns : u) - 1) & 1u, deadline)) ok = false;
                            tc_fence_after();
#pragma unroll
                            for (int c = 0; c < HD; c += 32) {
                                tmem_ld32(to + c, sv);
#pragma unroll
                                for (int j = 0; j < 32; j++) sv[j] *= factor;
                                tmem_st32(to + c, sv);
                            }
                        }
                        tmem_wait_st();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sh.p_full[t][u & 1]);
                        turns++;
                    }
                }
            }
            // shares go over K and V, which the other tile's MMAs may still read
            for (int e = Z > 1 ? 0 : t; e < (Z > 1 ? tiles : t + 1); e++)
                if (nb > 0 && !warp_wait(&sh.o_done[e], 0u, deadline)) ok = false;
            tc_fence_after();
            const float il = l == 0.f ? 0.f : unit / l;   // no weight at all: zeros (O is tiny, not NaN)
            const bool bad = *(volatile int *)&sh.bad != 0;
#pragma unroll
            for (int c = 0; c < HD; c += 32) {
                if ((kSkip ? turns : steps) > 0) tmem_ld32(to + c, sv);
                else {
#pragma unroll
                    for (int j = 0; j < 32; j++) sv[j] = 0.f;
                }
                if (bad)   // the NaN of V that this row sees in masked blocks
                    for (int b = 0; b < nb; b++) {
                        const int key = key_of(b);
                        if (whole(key)) continue;
                        for (int j = key; j < key + kKeys; j++) {
                            if (j >= at + 1 || (j >= e1 && j < s2)) continue;
                            const int pg = page_at(p.c, stream, j >> p.c.page_shift);
                            if (pg < 0) continue;
                            const unsigned char *v = p.c.v + page_base(p.c, p.layer, pg, kvh) + (j & (p.c.page - 1)) * p.c.slot_stride + c;
                            for (int d = 0; d < 32; d++)
                                if ((v[d] & 0x7fu) == 0x7fu)
#pragma unroll
                                    for (int e = 0; e < 32; e++) sv[e] = e == d ? NAN : sv[e];
                        }
                    }
                if (Z > 1) {
                    // this share's sums, 16-byte chunks swizzled by the row
                    float *o = reinterpret_cast<float *>(sh.o) + ml * HD;
#pragma unroll
                    for (int j = 0; j < 32; j += 4)
                        *reinterpret_cast<float4 *>(o + ((((c + j) >> 2) ^ (ml & 7)) << 2)) =
                            make_float4(sv[j] * unit, sv[j + 1] * unit, sv[j + 2] * unit, sv[j + 3] * unit);
                } else if (ok && m < M) {
                    T *dst = static_cast<T *>(p.out) + row * HD + c;
#pragma unroll
                    for (int j = 0; j < 32; j += 8)
                        *reinterpret_cast<uint4 *>(dst + j) =
                            make_uint4(pack2<T>(sv[j] * il, sv[j + 1] * il), pack2<T>(sv[j + 2] * il, sv[j + 3] * il),
                                       pack2<T>(sv[j + 4] * il, sv[j + 5] * il), pack2<T>(sv[j + 6] * il, sv[j + 7] * il));
                }
            }
            if (Z > 1) {
                sh.mx[ml] = mr;
                sh.sum[ml] = l;
            } else if (ok && m < M && p.lse) {
                p.lse[row] = l == 0.f ? -INFINITY : (mr + log2f(l)) * 0.69314718055994531f;
            }
        }
    }
    if (!ok) {
        sh.failed = 1;
        if (p.err) atomicExch_system(p.err, 1u);
        const uint64_t grace = globaltimer() + 10000000ull;   // let copies and MMAs in flight land
        while (globaltimer() < grace) {
        }
    }
    // TMEM goes back before the cluster meets: no CTA holds it while it waits
    // for a peer that may itself wait for TMEM
    tc_fence_before();
    __syncthreads();
    if (warp == kWarpMma) {
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
    if (sh.failed) {   // whatever was written or is to be merged: NaN, so that no void row passes for a result
        const int rows = min(NT * kAtRows, M - m0);
        for (int ml = threadIdx.x; ml < rows; ml += kThreads) {
            const int m = m0 + ml;
            const long long row = (long long)(s.r0 + m / p.group) * p.n_heads + head0 + m % p.group;
            sh.mx[ml] = sh.sum[ml] = NAN;
            if (Z > 1) continue;
            for (int d = 0; d < HD; d += 8)
                *reinterpret_cast<uint4 *>(static_cast<T *>(p.out) + row * HD + d) =
                    make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);   // NaN in either type
            if (p.lse) p.lse[row] = NAN;
        }
    }
    if (Z > 1) {
        cluster_sync_all();
        const uint32_t o_s = smem_u32(sh.o), m_s = smem_u32(sh.mx), l_s = smem_u32(sh.sum);
        const int rows = min(NT * kAtRows, M - m0);
        for (int e = z * kThreads + threadIdx.x; e < rows * (HD / 4); e += Z * kThreads) {
            const int ml = e / (HD / 4), d4 = e % (HD / 4), m = m0 + ml;
            float gm = -INFINITY;
            for (int r = 0; r < Z; r++) gm = fmaxf(gm, ld_dsmem_f1(mapa_shared(m_s + 4 * ml, r)));
            float gl = 0.f;
            float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int r = 0; r < Z; r++) {
                const float mr = ld_dsmem_f1(mapa_shared(m_s + 4 * ml, r));
                const float w = mr == -INFINITY ? 0.f : exp2_approx(mr - gm);
                const float l = ld_dsmem_f1(mapa_shared(l_s + 4 * ml, r));
                const float4 v = ld_dsmem_f4(mapa_shared(o_s + 4 * (ml * HD + ((d4 ^ (ml & 7)) << 2)), r));
                if (mr == -INFINITY && l == 0.f) continue;   // this share saw no key of the row
                gl = fmaf(w, l, gl);
                a.x = fmaf(w, v.x, a.x);
                a.y = fmaf(w, v.y, a.y);
                a.z = fmaf(w, v.z, a.z);
                a.w = fmaf(w, v.w, a.w);
            }
            const float il = gl == 0.f ? 0.f : 1.0f / gl;
            const long long row = (long long)(s.r0 + m / p.group) * p.n_heads + head0 + m % p.group;
            store4<T>(static_cast<T *>(p.out) + row * HD + 4 * d4, make_float4(a.x * il, a.y * il, a.z * il, a.w * il));
            if (p.lse && d4 == 0) p.lse[row] = gl == 0.f ? -INFINITY : (gm + log2f(gl)) * 0.69314718055994531f;
        }
        cluster_sync_all();   // no CTA leaves while a peer still reads its share
    }
}

template <int HD, int NT>
constexpr size_t pt_smem() {
    return std::max<size_t>(sizeof(PtSmem<HD, NT>), NT == 2 ? kPtOneCta : 0);
}

// A shape's launch: its cluster size and what that costs.
struct PtPlan {
    double cost = 1e30;
    int shares = 0;
};

// Microseconds, measured: a CTA's start and end; the merge of shares; a block of
// keys, of 128 for two tiles, of 64 for a tile alone on its SM and beside another.
constexpr double kPtFixed = 11, kPtMerge = 6, kPtTwo = 2.5, kPtAlone = 1.15, kPtBeside = 1.75;

// Shares by the least time.  With one CTA to an SM equal CTAs end together, so a
// started wave is a whole one; with two, waves run into each other and their blocks
// count in proportion.  The keys are those that the table has room for: the
// lengths are on the device.
// 8 streams of 64 packed rows over 3016 keys: 1 share 72 us, 2 48, 4 39, 8 53; of 256
// over 2064: two tiles, 1 share 64, 2 51, 4 68, one tile 56, 54, 67.  Encoder chunk
// (192 two-tile CTAs): 64, one tile 58.  300 rows of 12 heads, 2 streams, 3300 keys:
// one tile, 2 shares 52, 3 51, 4 62.
template <typename T, int HD, int NT>
cudaError_t plan_many(const PagedAttnParams &p, PtPlan *out) {
    auto kernel = paged_many_kernel<T, HD, NT>;
    constexpr size_t kSmem = pt_smem<HD, NT>();
    static_assert(kSmem <= (228 / pt_ctas(NT) - 1) * 1024, "they fit an SM");
    static ClusterKernel ck;
    int dev = 0;
    cudaError_t e = cluster_prepare(ck, kernel, kSmem, &dev);
    if (e != cudaSuccess) return e;
    const long long M = (long long)p.r.max_rows * p.group, tiles = (M + NT * kAtRows - 1) / (NT * kAtRows);
    long long keys = (long long)p.c.table_stride * p.c.page;
    if (p.window > 0) keys = std::min(keys, (long long)p.window + p.n_sink + (NT * kAtRows - 1) / p.group + 2);
    const long long blocks = (keys + pt_keys(NT) - 1) / pt_keys(NT), clusters = tiles * p.c.n_kv_heads * p.c.n_streams;
    for (int Z = 1; Z <= kMaxCluster && Z <= blocks; Z++) {
        // for this kernel the device's answer is one CTA to an SM (148 without a
        // cluster), while two one-tile CTAs do run side by side: 148 of them over 2900
        // keys take 67 us, 296 88, 368 139
        int at_once = 0;
        if ((e = cluster_active(ck, kernel, dev, pt_threads(NT), kSmem, Z, &at_once)) != cudaSuccess) return e;
        if (at_once < 1) continue;
        const double fill = (double)clusters / (at_once * pt_ctas(NT)), waves = std::max(1.0, ceil(fill));
        const double part = (double)((blocks + Z - 1) / Z);
        const double work = NT == 2 ? part * waves * kPtTwo : part * (fill <= 0.5 ? kPtAlone : std::max(1.0, fill) * kPtBeside);
        const double t = work + waves * kPtFixed + (Z > 1 ? kPtMerge : 0.0);
        if (t < out->cost) {
            out->cost = t;
            out->shares = Z;
        }
    }
    return out->shares ? cudaSuccess : cudaErrorInvalidConfiguration;
}

template <typename T, int HD, int NT>
cudaError_t launch_many(PagedAttnParams p, const PtPlan &plan, cudaStream_t st, RowsPlan *only) {
    if (only) {
        *only = {NT * kAtRows, pt_ctas(NT), plan.shares};
        return cudaSuccess;
    }
    const long long M = (long long)p.r.max_rows * p.group, tiles = (M + NT * kAtRows - 1) / (NT * kAtRows);
    p.shares = plan.shares;
    cudaLaunchAttribute attr;
    const long long ctas = p.shares * tiles * p.c.n_kv_heads * p.c.n_streams;
    if (ctas > INT_MAX) return cudaErrorInvalidConfiguration;   // (2^31 CTAs would take hours)
    p.tiles = (int)tiles;
    const cudaLaunchConfig_t cfg = cluster_config(dim3((unsigned)ctas), pt_threads(NT), pt_smem<HD, NT>(), p.shares, &attr, st);
    return cudaLaunchKernelEx(&cfg, paged_many_kernel<T, HD, NT>, p);
}

template <typename T, int HD>
cudaError_t launch_dim(const PagedAttnParams &p, cudaStream_t st, RowsPlan *only, double *cost) {
    PtPlan one, two;
    cudaError_t e = plan_many<T, HD, 1>(p, &one);
    if (e != cudaSuccess) return e;
    if ((long long)p.r.max_rows * p.group > kAtRows && (e = plan_many<T, HD, 2>(p, &two)) != cudaSuccess) return e;
    if (cost) {
        *cost = std::min(one.cost, two.cost);
        return cudaSuccess;
    }
    return two.cost < one.cost ? launch_many<T, HD, 2>(p, two, st, only) : launch_many<T, HD, 1>(p, one, st, only);
}
template <typename T>
cudaError_t launch_typed(const PagedAttnParams &p, cudaStream_t st, RowsPlan *only, double *cost) {
    return p.c.head_dim == 64 ? launch_dim<T, 64>(p, st, only, cost) : launch_dim<T, 128>(p, st, only, cost);
}

}  // namespace

cudaError_t launch_paged_attn_tc(const PagedAttnParams &p, cudaStream_t st, RowsPlan *only, double *cost) {
    return p.q_type == ELEM_BF16 ? launch_typed<__nv_bfloat16>(p, st, only, cost) : launch_typed<__half>(p, st, only, cost);
}

}  // namespace vc
