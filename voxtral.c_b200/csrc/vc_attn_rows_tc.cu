// vc_attn_rows_tc.cu - attention of a call's rows over a 16-bit cache slab on
// the tcgen05 tensor cores: windows, sinks and trees as in vc_attn_rows.cu.
//
// A CTA takes NT (1 or 2) tiles of 128 packed query rows (m = row * group +
// head, TMEM lane = packed row) of one (stream, KV head) and a share of the
// blocks of 64 or 128 keys that they see; the shares are a cluster.
//   4 warps per tile softmax, thread = packed row, 64 keys a step: P = 2^(s - m)
//                    of S (TMEM), rounded to the cache's type, over the S
//                    columns it came from; before that they load their rows of Q
//   3 warps          loads: K (one warp) and V blocks two or more deep, by TMA where a
//                    block's slots follow one another, by 16-byte cp.async into
//                    the same swizzled layout where they do not (ring wrap,
//                    sinks, the last block: zeros past the end)
//   1 warp           issues the MMAs, M 128: S_t = Q_t K^T (K HD) and, by
//                    steps of 64 keys, O_t += P_t V (N HD; A from TMEM, V an
//                    MN-major operand)
// Two tiles: S_t(b + 1) overwrites P_t(b), so it is issued behind the MMAs that
// read it; the tiles alternate - one's softmax runs under the other's MMAs -
// and share each K and V block.
//
// The running maximum m moves only when a step exceeds it by more than 2^8,
// and only then O is rescaled.  Rounding P to 16 bits is one half step of the
// type per weight, as the output's own rounding; the sums l take the unrounded
// weights.  In fp16 the steps below 2^-14 are fixed ones of 2^-24: P = 2^(s - m)
// would lose a key whose weight is 2^-25 of the largest, and a hundred thousand
// of them are a visible part of l.  There m is the maximum less 7, so that P
// fills the type up to 2^15 and what is lost is 2^-32 of the largest weight per
// key: half a step of the output only from 2^21 keys on.
//
// Zero times a masked key's NaN or infinity would be NaN: in blocks that some
// row does not see whole, the loading threads look for non-finite V values,
// put zeros in their place and set a flag, and the rows that do see them add
// them at the end.
#include "vc_cluster.h"
#include "vc_rows.cuh"
#include "vc_tc.cuh"

#include <algorithm>
#include <atomic>
#include <type_traits>
#include <math.h>

namespace vc {

using namespace tc;

namespace {

constexpr int kAtHalf = 64;             // keys per softmax step
constexpr int kAtRows = 128;            // packed rows per MMA tile = TMEM lanes
// Shapes: NT tiles of RT rows that exist (the MMA's other rows are whatever
// lies behind Q in shared memory; nobody reads their lanes).
//   <2, 128>  heads of 128, many rows over long contexts: bound by the
//             latency of the softmax chain (~5450 cycles a block; the MMAs'
//             reads of shared memory are ~1540, the exponentials ~1280).
//             128-key blocks (an MMA of N
//             64 takes as long as one of N 128, reading its A tile), one CTA
//             per SM.  2021 rows of 32 heads over 4100 keys, bf16: 195 to
//             200 us, 0.41 of the bf16 rate (two S ranges of 64 keys: 229)
//   <1, 128>  heads of 128: 64-key blocks with two S ranges, so that S(b + 1)
//             is ready when the softmax is done with S(b); two CTAs per SM.
//             Heads of 64, any number of rows (at_three): one S range, 128 TMEM
//             columns, three CTAs per SM, whose chains S - softmax - P - P.V
//             fill each other's gaps.  1500 rows of 32 heads, window 750: 51 us
//             (<2, 128> took 72: 192 CTAs in two waves; vc_enc_attn_tc.cu, whose
//             P goes through shared memory, so that S(b + 1) need not wait for
//             it, takes 31 over its own ring)
//   <1, 32>   up to 32 rows, a token's or a few tokens' heads, bound by HBM: Q
//             is small, 96 KB of keys in flight per CTA, two CTAs per SM.  24
//             tokens of 32 / 8 heads over 4100 keys: 57 us, 4.7 TB/s, 0.73 of
//             the copy rate (<1, 128> as long); 4 tokens of 8 streams over 512
//             keys 13.0 us (<1, 128>: 14.5), of one over 4096 15.7 (16.6)
constexpr int at_keys(int nt) { return nt == 1 ? 64 : 128; }
constexpr bool at_three(int hd, int nt, int rt) { return hd == 64 && nt == 1 && rt == 128; }
constexpr int at_stages(int hd, int nt, int rt) { return at_three(hd, nt, rt) ? 3 : nt == 2 ? 2 : (rt == 32 ? 3 : 2) * (128 / hd); }
constexpr int at_ctas(int hd, int nt, int rt) { return at_three(hd, nt, rt) ? 3 : nt == 1 ? 2 : 1; }
// RT / 32 softmax warps per tile, a K and two V loaders, an MMA warp
constexpr int at_threads(int nt, int rt) { return (nt * rt / 32 + 4) * 32; }
constexpr uint64_t kAtWaitNs = 2000000000ull, kAtBlockNs = 10000ull;   // a CTA's waits end after this, per block as well
constexpr float kAtRescale = 8.0f;      // log2 of what a step may exceed the maximum by before it moves
template <typename T>
constexpr float kAtAbove = std::is_same<T, __half>::value ? 7.0f : 0.0f;   // the maximum less m
constexpr int kAtOneCta = 120 * 1024;   // more than half an SM's shared memory: one CTA per SM
constexpr double kAtFixed = 8;          // block times of a CTA's start and merge (6 to 8 us)
constexpr double kAtMerge = 4;          // more for the merge of 128 rows' shares (64 KB of sums to a CTA)
constexpr double kAtAlone = 0.6;        // a block's time on an SM of its own, of that beside another CTA

template <int HD, int NT, int RT>
struct AtSmem {
    static constexpr int kKeys = at_keys(NT), kStages = at_stages(HD, NT, RT);
    // Q, K and V tiles are HD / 64 sub-tiles of [rows or keys][128 bytes]
    static constexpr int kTile = kKeys * HD * 2, kSubTile = kKeys * 128, kQTile = RT * HD * 2, kQSub = RT * 128;
    static constexpr int kO = NT * RT * HD * 4;   // bytes of O in fp32, over K and V at the end
    unsigned char q[NT][kQTile];
    union {
        unsigned char kv[2][kStages][kTile];      // K, V
        unsigned char o[kO];
    };
    uint32_t anc[NT * RT][kTreeMax / 32];
    float mx[NT * RT], sum[NT * RT];
    short parent[kTreeMax];
    uint64_t q_full, v_land[kStages], k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages], s_full[2], p_full[NT][2], o_part[NT], o_done;   // s_full: by tile, or (one tile) by S range
    uint32_t tmem;
    int bad;      // a masked block holds non-finite V values
    int failed;   // some warp's wait ran out: the CTA's rows are void
    uint64_t stall;   // nothing arrives here
};

template <typename T>
__host__ __device__ constexpr uint32_t at_idesc(int N, bool b_mn) {
    return (1u << 4) | (sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u) |
           (b_mn ? (1u << 16) : 0u) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(kAtRows >> 4) << 24);
}

// MN-major operand, 128-byte swizzle: 64-element atoms along N `atom` bytes
// apart (a sub-tile), 8-key groups 1024 bytes apart.
__device__ __forceinline__ uint64_t at_desc_mn(const void *p, int atom) {
    const uint64_t addr = smem_u32(p);
    return ((addr >> 4) & 0x3FFFull) | ((uint64_t)(atom >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) |
           (2ull << 61);
}

// A bounded wait of a whole warp: the same answer in every lane.
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, uint64_t deadline) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, deadline));
}

// The MMA warp's instructions: all 32 lanes reach them and `lead` is set in
// one, so that the warp never diverges and its operands stay in uniform
// registers (issued from a branch of one lane each MMA took ~75 cycles).
// D[tmem] (+)= A[smem] . B[smem]
__device__ __forceinline__ void warp_mma(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                         uint32_t accumulate, uint32_t lead) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(lead)
        : "memory");
}
// D[tmem] (+)= A[tmem] . B[smem]: A holds two 16-bit values per column
__device__ __forceinline__ void warp_mma_ta(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                            uint32_t accumulate, uint32_t lead) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(lead)
        : "memory");
}
__device__ __forceinline__ void warp_commit(uint64_t *bar, uint32_t lead) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
        "r"(lead)
        : "memory");
}

// Columns of this thread's TMEM lane: a store is complete after tmem_wait_st,
// a load after tmem_ld_wait, which names the values so that no use moves ahead
// of it.
__device__ __forceinline__ void tmem_st32_async(uint32_t taddr, const uint32_t *v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
        "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
        "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
        : "memory");
}
__device__ __forceinline__ void tmem_ld16_async(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// bits i with a <= c0 + i < b
__device__ __forceinline__ uint32_t range_bits(int c0, int a, int b) {
    const int s = max(a - c0, 0), e = min(b - c0, 32);
    if (s >= e) return 0u;
    return (0xffffffffu >> (32 - (e - s))) << s;
}

// A packed row's visible keys in the walk's order: [0, e1), [s2, e2), and the
// ancestor bits from index `node` on.
struct RowKeys {
    int e1, s2, e2, node;
    __device__ uint32_t bits(int c0, const uint32_t *anc) const {
        uint32_t w = range_bits(c0, 0, e1) | range_bits(c0, s2, e2);
        if (anc) {
            const int o = c0 - node;   // bit o + i of the ancestor mask for column i
            const int word = o >> 5, sh = o & 31;
            const uint32_t a = word >= 0 && word < kTreeMax / 32 ? anc[word] : 0u;
            const uint32_t b = word + 1 >= 0 && word + 1 < kTreeMax / 32 ? anc[word + 1] : 0u;
            w |= __funnelshift_r(a, b, sh);
        }
        return w;
    }
};

// 2^x of two values on the FMA pipe: x = n + f, n the nearest whole number
// (left in the low bits by adding 1.5 * 2^23), 2^f by its minimax polynomial
// of degree 4 on [-1/2, 1/2] (Remez: relative error 2.6e-6, of either sign),
// n added to the exponent.  Below -126 the result stays near 2^-126.
__device__ __forceinline__ void exp2_poly2(float &a, float &b) {
    const uint64_t x = pair(fmax_nan(a, -126.f), fmax_nan(b, -126.f));
    const uint64_t t = add2(x, pair(12582912.f, 12582912.f));
    const uint64_t f = fma2(add2(t, pair(-12582912.f, -12582912.f)), pair(-1.f, -1.f), x);
    uint64_t r = fma2(f, pair(0.00957010201463f, 0.00957010201463f), pair(0.0559178603063f, 0.0559178603063f));
    r = fma2(f, r, pair(0.24024744825f, 0.24024744825f));
    r = fma2(f, r, pair(0.693121814743f, 0.693121814743f));
    r = fma2(f, r, pair(0.999999261447f, 0.999999261447f));
    float ta, tb;
    unpair(t, ta, tb);
    unpair(r, a, b);
    a = __int_as_float(__float_as_int(a) + (__float_as_int(ta) << 23));
    b = __int_as_float(__float_as_int(b) + (__float_as_int(tb) << 23));
}

// Half a block of a row: w = 2^(s sl2 - base) as pairs of T, ls their sum
// before rounding; the largest s sl2 - base as the result (NaN if one is).
// The next 16 scores are on their way from TMEM while 16 are worked on.  The
// exponential unit takes 8 cycles per warp, so in blocks without a mask
// kAtPoly of 8 pairs go through the FMA pipe instead (2021 rows over 4100 keys
// 196 -> 191 us).
constexpr int kAtPoly = 3;
template <typename T, bool MASKED>
__device__ __forceinline__ float weigh_half(uint32_t ts, float sl2, float base, const RowKeys &keys, int c0,
                                            const uint32_t *anc, uint32_t (&w)[kAtHalf / 2], float &ls) {
    float mx[2] = {-INFINITY, -INFINITY};
    uint64_t rs[2] = {0, 0};
    const uint64_t sl = pair(sl2, sl2), nb = pair(-base, -base);
    uint32_t ra[16], rb[16], vis = 0xffffffffu;
    tmem_ld16_async(ts, ra);
#pragma unroll
    for (int c = 0; c < kAtHalf; c += 16) {
        uint32_t(&cur)[16] = (c & 16) ? rb : ra;
        tmem_ld_wait(cur);
        if (c + 16 < kAtHalf) tmem_ld16_async(ts + c + 16, (c & 16) ? ra : rb);
        if (MASKED) vis = (c & 16) ? vis >> 16 : keys.bits(c0 + c, anc);
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
            float xa, xb;
            unpair(fma2(pair(__uint_as_float(cur[j]), __uint_as_float(cur[j + 1])), sl, nb), xa, xb);
            if (MASKED) {
                xa = (vis >> j) & 1u ? xa : -INFINITY;
                xb = (vis >> (j + 1)) & 1u ? xb : -INFINITY;
            }
            mx[0] = fmax_nan(mx[0], xa);
            mx[1] = fmax_nan(mx[1], xb);
            if (!MASKED && (j >> 1) % 8 < kAtPoly) {
                exp2_poly2(xa, xb);
            } else {
                xa = exp2_approx(xa);
                xb = exp2_approx(xb);
            }
            rs[(j >> 1) & 1] = add2(rs[(j >> 1) & 1], pair(xa, xb));
            w[(c + j) >> 1] = pack2<T>(xa, xb);
        }
    }
    float a, b;
    unpair(add2(rs[0], rs[1]), a, b);
    ls = a + b;
    return fmax_nan(mx[0], mx[1]);
}
template <typename T>
__device__ __forceinline__ float weigh(uint32_t ts, float sl2, float base, bool full, const RowKeys &keys, int c0,
                                       const uint32_t *anc, uint32_t (&w)[kAtHalf / 2], float &ls) {
    return full ? weigh_half<T, false>(ts, sl2, base, keys, c0, anc, w, ls)
                : weigh_half<T, true>(ts, sl2, base, keys, c0, anc, w, ls);
}

template <typename T>
__device__ __forceinline__ uint32_t nonfinite2(uint32_t u) {   // 0xffff in each half that is inf or NaN
    constexpr uint32_t e = std::is_same<T, __nv_bfloat16>::value ? 0x7f807f80u : 0x7c007c00u;
    return __vcmpeq2(u & e, e);
}

template <typename T, int HD, int NT, int RT>
__global__ void __launch_bounds__(at_threads(NT, RT), at_ctas(HD, NT, RT)) attn_rows_tc_kernel(const __grid_constant__ CUtensorMap tm_k,
                                                                   const __grid_constant__ CUtensorMap tm_v,
                                                                   const RowsAttnParams p) {
    using Sm = AtSmem<HD, NT, RT>;
    constexpr int kSub = HD / 64;            // 64-dim sub-tiles of a tile
    constexpr int kSoft = RT / 32;           // softmax warps of a tile
    constexpr int kThreads = at_threads(NT, RT), kWarpK = kSoft * NT, kWarpV2 = kWarpK + 2, kWarpMma = kWarpK + 3;
    constexpr int kStages = Sm::kStages;
    constexpr int kKeys = Sm::kKeys, kSteps = kKeys / kAtHalf;
    constexpr bool kTwoS = NT == 1 && !at_three(HD, NT, RT);          // two S ranges
    constexpr uint32_t kTmemCols = at_three(HD, NT, RT) ? 128 : NT == 2 ? 512 : 256;
    extern __shared__ __align__(1024) unsigned char at_smem_raw[];
    Sm &sh = *reinterpret_cast<Sm *>(at_smem_raw);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int z = blockIdx.x % p.shares, Z = p.shares;
    const int m0 = blockIdx.x / p.shares * (NT * RT), kvh = blockIdx.y, stream = blockIdx.z;
    const RowSpan s = row_span(p.r, stream);
    const int M = s.n * p.group;
    if (m0 >= M) return;   // the whole cluster leaves
    const bool tree = p.r.parent != nullptr;
    const int i0 = m0 / p.group, i1 = (min(m0 + NT * RT, M) - 1) / p.group + 1;
    const KeyRange kr = key_range(p.c, s, i0, i1, p.window, tree);
    const int total = kr.total(), blocks = (total + kKeys - 1) / kKeys;
    const int b0 = (int)((long long)z * blocks / Z), nb = (int)((long long)(z + 1) * blocks / Z) - b0;
    const int tiles = M - m0 > RT ? NT : 1;   // tiles with rows
    const int head0 = kvh * p.group;
    bool ok = true;

    // keys that every row of the CTA sees, in the walk's order: [core_s, core_e)
    // (and [0, ns) when core_s = ns, contiguous with it)
    const int up_min = tree ? s.pos - 1 : s.pos + i0;
    int core_s = kr.ns + (p.window > 0 ? max(0, min(s.pos + i1 - p.window - kr.lo, kr.nm)) : 0), core_e = kr.ns + max(0, min(up_min - kr.lo + 1, kr.nm));
    if (up_min < kr.ns - 1) core_e = 0;
    else if (core_s == kr.ns) core_s = 0;
    auto whole = [&](int b) { return b * kKeys >= core_s && (b + 1) * kKeys <= core_e; };

    if (threadIdx.x == 0) {
        mbar_init(&sh.q_full, min(NT * kSoft, (M - m0 + 31) / 32));   // the warps with rows
        for (int i = 0; i < kStages; i++) {
            mbar_init(&sh.v_land[i], 1);
            mbar_init(&sh.k_full[i], 1);
            mbar_init(&sh.v_full[i], 2);   // one arrival per V warp
            mbar_init(&sh.k_empty[i], 1);
            mbar_init(&sh.v_empty[i], 1);
        }
        for (int t = 0; t < NT; t++) {
            mbar_init(&sh.o_part[t], 1);
            // one arrival per warp with rows
            const int warps = max(1, min(kSoft, (M - m0 - t * RT + 31) / 32));
            mbar_init(&sh.p_full[t][0], warps);
            mbar_init(&sh.p_full[t][1], warps);
        }
        mbar_init(&sh.s_full[0], 1);
        mbar_init(&sh.s_full[1], 1);
        mbar_init(&sh.o_done, 1);
        mbar_init(&sh.stall, 1);
        sh.bad = sh.failed = 0;
        if (p.maps) {
            prefetch_tensormap(&tm_k);
            prefetch_tensormap(&tm_v);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kWarpMma) {
        tmem_alloc(&sh.tmem, kTmemCols);
        tmem_relinquish();
    }
    if (tree) load_parents(sh.parent, p.r, s, threadIdx.x, kThreads);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    const uint64_t deadline = globaltimer() + kAtWaitNs + (uint64_t)nb * kAtBlockNs;   // (TMEM may have been another kernel's)
    constexpr uint32_t kOCol = kTwoS ? 2 * kKeys : NT * kKeys;   // S ranges first, then O tiles

    if (warp >= kWarpK && warp <= kWarpV2) {
        // ---- loads: one warp K, two V ----
        constexpr int kCh = HD / 8;                   // 16-byte chunks per row
        const bool is_v = warp != kWarpK;
        // chunk ch of row r: sub-tile ch / 8, swizzled by the row
        auto at = [&](int r, int ch) { return (ch >> 3) * Sm::kSubTile + r * 128 + (((ch & 7) ^ (r & 7)) << 4); };
        const long long base = p.layer_off + (long long)stream * p.c.stream_stride + (long long)kvh * p.c.head_stride;
        const char *src = (is_v ? p.c.v : p.c.k) + base * 2;
        const long long slot_bytes = p.c.slot_stride * 2;
        const int lo_slot = cache_slot(p.c, kr.lo);
        unsigned char(*const bufs)[Sm::kTile] = sh.kv[is_v];
        uint64_t *const full = is_v ? sh.v_full : sh.k_full, *const empty = is_v ? sh.v_empty : sh.k_empty;
        // this warp's chunks of a block that it copies or looks through itself
        const int first = (warp == kWarpV2 ? 32 : 0) + lane, step = is_v ? 64 : 32;
        enum { kNone, kLook, kCopied };
        int pending = kNone, pending_b = 0;
        uint32_t land = 0;   // bit i: the phase that v_land[i] completes next
        auto settle = [&]() {   // publish the pending block once it has landed
            if (pending == kNone) return;
            if (pending == kLook) {
                const int i = pending_b % kStages;
                if (!mbar_wait(&sh.v_land[i], (land >> i) & 1u, deadline)) ok = false;
                land ^= 1u << i;
            } else {
                cp_async_wait<0>();
            }
            if (is_v && !whole(b0 + pending_b)) {
                unsigned char *v = bufs[pending_b % kStages];
                bool found = false;
                // after TMA any thread may look at any chunk; after copies, at its own
#pragma unroll 8
                for (int e = first; e < kKeys * kCh; e += step) {
                    uint4 *c = reinterpret_cast<uint4 *>(v + at(e / kCh, e % kCh));
                    const uint4 u = *c;
                    const uint4 n = make_uint4(nonfinite2<T>(u.x), nonfinite2<T>(u.y), nonfinite2<T>(u.z), nonfinite2<T>(u.w));
                    if (n.x | n.y | n.z | n.w) {
                        *c = make_uint4(u.x & ~n.x, u.y & ~n.y, u.z & ~n.z, u.w & ~n.w);
                        found = true;
                    }
                }
                if (found) atomicExch(&sh.bad, 1);
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[pending_b % kStages]);
            pending = kNone;
        };
        for (int b = 0; b < nb; b++) {
            if (b >= kStages &&
                !__all_sync(0xffffffffu, mbar_wait(&empty[b % kStages], (b / kStages + 1) & 1u, deadline))) {
                ok = false;
                break;
            }
            unsigned char *buf = bufs[b % kStages];
            const int idx0 = (b0 + b) * kKeys;
            int slot0 = lo_slot + (idx0 - kr.ns);   // of index idx0, past the sinks
            if (slot0 >= p.c.cap) slot0 -= p.c.ring;
            const bool look = is_v && !whole(b0 + b);
            if (p.maps && idx0 >= kr.ns && idx0 + kKeys <= total && slot0 + kKeys <= p.c.cap) {   // slots in a row
                uint64_t *bar = look ? &sh.v_land[b % kStages] : &full[b % kStages];
                if (warp != kWarpV2 && lane == 0) {
                    mbar_expect_tx(bar, Sm::kTile);
#pragma unroll
                    for (int h = 0; h < kSub; h++)
                        tma_load_4d(buf + h * Sm::kSubTile, is_v ? &tm_v : &tm_k, h * 64, kvh, slot0, stream, bar);
                } else if (warp == kWarpV2 && lane == 0 && !look) {
                    mbar_arrive(bar);
                }
                settle();
                if (look) pending = kLook;
            } else {
                const uint32_t dst = smem_u32(buf);
#pragma unroll 4
                for (int e = first; e < kKeys * kCh; e += step) {
                    const int r = e / kCh, ch = e % kCh, idx = idx0 + r;
                    int slot = idx;
                    if (idx >= kr.ns) {
                        slot = lo_slot + (idx - kr.ns);
                        if (slot >= p.c.cap) slot -= p.c.ring;
                    }
                    cp_async16(dst + at(r, ch), src + (idx < total ? slot * slot_bytes + ch * 16 : 0), idx < total);
                }
                cp_async_commit();
                settle();
                pending = kCopied;
            }
            pending_b = b;
        }
        settle();
    } else if (warp == kWarpMma) {
        // ---- MMAs ----
        if (nb > 0) {
            const uint32_t lead = lane == 0, tm = __shfl_sync(0xffffffffu, tmem, 0);
            constexpr uint32_t id_s = at_idesc<T>(kKeys, false), id_o = at_idesc<T>(HD, true);
            auto issue_s = [&](int t, int b) {   // S range t of two tiles, b % 2 of one
                const uint64_t a0 = smem_desc_sw128(sh.q[t]), k0 = smem_desc_sw128(sh.kv[0][b % kStages]);
                const int r = kTwoS ? b & 1 : t;
#pragma unroll
                for (int h = 0; h < kSub; h++)
#pragma unroll
                    for (int k = 0; k < 4; k++)   // 16 dims: +32 bytes
                        warp_mma(tm + r * kKeys, a0 + h * (Sm::kQSub / 16) + 2 * k, k0 + h * (Sm::kSubTile / 16) + 2 * k,
                                 id_s, (h | k) != 0 ? 1u : 0u, lead);
                warp_commit(&sh.s_full[r], lead);
            };
            auto issue_o = [&](int t, int b, int h) {   // 64 keys of O += P V
                const uint64_t v0 = at_desc_mn(sh.kv[1][b % kStages], Sm::kSubTile);
                const int r = kTwoS ? b & 1 : t;
#pragma unroll
                for (int k = 0; k < kAtHalf / 16; k++)   // 16 keys: 8 columns of P, 2048 bytes of V
                    warp_mma_ta(tm + kOCol + t * HD, tm + r * kKeys + h * kAtHalf + 8 * k, v0 + (h * 8192 + k * 2048) / 16,
                                id_o, (b | h | k) != 0 ? 1u : 0u, lead);
                if (kTwoS || h + 1 < kSteps) warp_commit(&sh.o_part[t], lead);
            };
            ok = warp_wait(&sh.q_full, 0u, deadline) && warp_wait(&sh.k_full[0], 0u, deadline);
            if (ok) {
                tc_fence_after();
                for (int t = 0; t < tiles; t++) issue_s(t, 0);
                warp_commit(&sh.k_empty[0], lead);
            }
            for (int b = 0; b < nb && ok; b++) {
                if constexpr (kTwoS) {
                    if (b + 1 < nb) {   // over P(b - 1), behind the MMAs that read it
                        ok = warp_wait(&sh.k_full[(b + 1) % kStages], ((b + 1) / kStages) & 1u, deadline);
                        if (!ok) break;
                        tc_fence_after();
                        issue_s(0, b + 1);
                        warp_commit(&sh.k_empty[(b + 1) % kStages], lead);
                    }
                    ok = warp_wait(&sh.v_full[b % kStages], (b / kStages) & 1u, deadline) &&
                         warp_wait(&sh.p_full[0][b & 1], (b >> 1) & 1u, deadline);
                    if (!ok) break;
                    tc_fence_after();
                    issue_o(0, b, 0);
                    warp_commit(&sh.v_empty[b % kStages], lead);
                } else {
                    // K(b + 1) too, before P is there: a poll takes ~300 cycles once
                    // MMAs read shared memory (8 trees of 64 rows 107.8 -> 106.2 us)
                    ok = warp_wait(&sh.v_full[b % kStages], (b / kStages) & 1u, deadline) &&
                         (b + 1 == nb || warp_wait(&sh.k_full[(b + 1) % kStages], ((b + 1) / kStages) & 1u, deadline));
                    for (int t = 0; t < tiles && ok; t++) {
#pragma unroll
                        for (int h = 0; h < kSteps; h++) {
                            if (ok) ok = warp_wait(&sh.p_full[t][h], b & 1u, deadline);
                            if (!ok) break;
                            tc_fence_after();
                            issue_o(t, b, h);
                        }
                        if (!ok) break;
                        if (b + 1 < nb) issue_s(t, b + 1);   // over P(b), behind the MMAs that read it
                        if (t == tiles - 1) {
                            warp_commit(&sh.v_empty[b % kStages], lead);
                            if (b + 1 < nb) warp_commit(&sh.k_empty[(b + 1) % kStages], lead);
                        }
                    }
                }
            }
            warp_commit(&sh.o_done, lead);
        }
        if (p.stall_ns) ok = warp_wait(&sh.stall, 0u, globaltimer() + p.stall_ns) && ok;
    } else {
        // ---- softmax: thread = packed row ----
        const int t = warp / kSoft, q = warp % kSoft, ml = t * RT + 32 * q + lane, m = m0 + ml;
        const bool here = m0 + t * RT + 32 * q < M;   // the warp has rows
        if (here) {
            const int i = min(m, M - 1) / p.group;
            {   // the warp's 32 rows of Q: HD / 8 lanes a row, zeros past M
                constexpr int kCh = HD / 8, kAtOnce = 32 / kCh;
                const int ch = lane % kCh;
                const uint32_t dst = smem_u32(sh.q[t]) + (ch >> 3) * Sm::kQSub;
                const long long row = (long long)(s.r0 + i) * p.n_heads + head0 + min(m, M - 1) % p.group;
#pragma unroll 8
                for (int it = 0; it < 32 / kAtOnce; it++) {
                    const int r = it * kAtOnce + lane / kCh, rt = 32 * q + r;
                    const long long from = __shfl_sync(0xffffffffu, row, r);
                    cp_async16(dst + rt * 128 + (((ch & 7) ^ (rt & 7)) << 4),
                               static_cast<const T *>(p.q) + from * HD + ch * 8, m0 + t * RT + rt < M);
                }
                cp_async_commit();
            }
            int pl = s.pos + i;
            const uint32_t *anc = nullptr;
            if (tree) {
                uint32_t *bits = sh.anc[ml];
#pragma unroll
                for (int w = 0; w < kTreeMax / 32; w++) bits[w] = 0u;
                const int depth = ancestor_bits(bits, sh.parent, i);
                window_bits(bits, sh.parent, i, depth, s.pos, p.c.n_sink, p.window);
                pl = s.pos + depth;
                anc = bits;
            }
            const int up = tree ? s.pos - 1 : pl;
            RowKeys keys;
            keys.e1 = min(kr.ns, up + 1);
            keys.s2 = kr.ns + (p.window > 0 ? max(0, pl - p.window + 1 - kr.lo) : 0);
            keys.e2 = kr.ns + min(max(0, up - kr.lo + 1), kr.nm);
            keys.node = s.pos < kr.ns ? s.pos : kr.ns + s.pos - kr.lo;
            const uint32_t tl = tmem + ((uint32_t)(32 * q) << 16);
            const uint32_t to = tl + kOCol + t * HD;
            const float sl2 = p.scale_log2;
            float mr = -INFINITY, l = 0.f;
            float sv[32];
            cp_async_wait<0>();
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.q_full);
            for (int b = 0; b < nb; b++) {
                const int r = kTwoS ? b & 1 : t;   // the S range
                if (!__all_sync(0xffffffffu, mbar_wait(&sh.s_full[r], (kTwoS ? b >> 1 : b) & 1u, deadline))) ok = false;
                tc_fence_after();
                const bool full = whole(b0 + b);
#pragma unroll 1
                for (int h = 0; h < kSteps; h++) {
                    const uint32_t ts = tl + r * kKeys + h * kAtHalf;
                    const int c0 = (b0 + b) * kKeys + h * kAtHalf;
                    // P against m so far; a row whose keys exceed the maximum
                    // by more than 2^8 takes theirs, and the warp goes over
                    // them again (S is intact until P is stored)
                    uint32_t w[kAtHalf / 2];
                    float base = mr == -INFINITY ? 0.f : mr, factor = 1.f, ls = 0.f;
                    float over;   // the largest less base
                    bool moved = false;
#pragma unroll 1
                    for (;;) {    // (one copy of its code)
                        over = weigh<T>(ts, sl2, base, full, keys, c0, anc, w, ls);
                        const bool move = mr == -INFINITY ? over > -INFINITY : over > kAtRescale + kAtAbove<T>;
                        if (moved || !__any_sync(0xffffffffu, move)) break;
                        moved = true;
                        if (move) {
                            const float mn = base + over - kAtAbove<T>;
                            factor = mr == -INFINITY ? 0.f : exp2_approx(mr - mn);
                            mr = base = mn;
                            l *= factor;
                        }
                    }
                    if (mr > -INFINITY) l += ls;
                    if (over != over) l = over;   // a NaN score: the row is NaN
                    tmem_st32_async(ts, w);       // over S
                    if (moved && b + h > 0) {
                        // O must hold the weights before these.  Two S ranges:
                        // S(b) is behind the MMAs of block b - 2, those of b - 1
                        // may be under way; else S(b) is behind block b - 1's,
                        // and the second step waits for the first's.
                        if (kTwoS || h == 1)
                            if (!__all_sync(0xffffffffu, mbar_wait(&sh.o_part[t], (kTwoS ? b - 1 : b) & 1u, deadline)))
                                ok = false;
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
                    if (lane == 0) mbar_arrive(&sh.p_full[t][kTwoS ? r : h]);
                }
            }
            if (nb > 0 && !__all_sync(0xffffffffu, mbar_wait(&sh.o_done, 0u, deadline))) ok = false;
            tc_fence_after();
            const float il = l == 0.f ? 0.f : 1.0f / l;   // no weight at all: zeros (O is tiny, not NaN)
            const bool bad = *(volatile int *)&sh.bad != 0;
            const long long row = (long long)(s.r0 + i) * p.n_heads + head0 + min(m, M - 1) % p.group;
#pragma unroll
            for (int c = 0; c < HD; c += 32) {
                if (nb > 0) tmem_ld32(to + c, sv);
                else {
#pragma unroll
                    for (int j = 0; j < 32; j++) sv[j] = 0.f;
                }
                if (bad) {
                    // the non-finite V values that this row sees in masked blocks
                    const long long base = p.layer_off + (long long)stream * p.c.stream_stride +
                                           (long long)kvh * p.c.head_stride + c;
                    const int lo_slot = cache_slot(p.c, kr.lo);
                    for (int idx = b0 * kKeys; idx < min(total, (b0 + nb) * kKeys); idx++) {
                        if (whole(idx / kKeys) || !((keys.bits(idx & ~31, anc) >> (idx & 31)) & 1u)) continue;
                        int slot = idx;
                        if (idx >= kr.ns) {
                            slot = lo_slot + (idx - kr.ns);
                            if (slot >= p.c.cap) slot -= p.c.ring;
                        }
                        const T *v = reinterpret_cast<const T *>(p.c.v) + base + slot * p.c.slot_stride;
#pragma unroll
                        for (int j = 0; j < 32; j++) {
                            const float x = (float)v[j];
                            if (!(fabsf(x) < INFINITY)) sv[j] += x;
                        }
                    }
                }
                if (Z > 1) {
                    // this share's sums, 16-byte chunks swizzled by the row
                    float *o = reinterpret_cast<float *>(sh.o) + ml * HD;
#pragma unroll
                    for (int j = 0; j < 32; j += 4)
                        *reinterpret_cast<float4 *>(o + ((((c + j) >> 2) ^ (ml & 7)) << 2)) =
                            make_float4(sv[j], sv[j + 1], sv[j + 2], sv[j + 3]);
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
        const int rows = min(NT * RT, M - m0);
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
        const int rows = min(NT * RT, M - m0);
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

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                  const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
    static const EncodeTiledFn fn = [] {
        void *q = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &q, cudaEnableDefault, &r) != cudaSuccess ||
            r != cudaDriverEntryPointSuccess)
            q = nullptr;
        return (EncodeTiledFn)q;
    }();
    return fn;
}

// One layer's K or V as [stream][slot][head][dim], boxes of `keys` slots x 64
// dims of one head, 128-byte swizzle.
bool cache_map(CUtensorMap *m, char *base, const CacheView &c, int keys) {
    EncodeTiledFn fn = encode_fn();
    const long long most = 1ll << 40;   // bytes of a stride
    if (!fn || c.cap < keys || c.head_stride * 2 >= most || c.slot_stride * 2 >= most || c.stream_stride * 2 >= most)
        return false;
    const cuuint64_t dims[4] = {(cuuint64_t)c.head_dim, (cuuint64_t)c.n_kv_heads, (cuuint64_t)c.cap, (cuuint64_t)c.n_streams};
    const cuuint64_t strides[3] = {(cuuint64_t)c.head_stride * 2, (cuuint64_t)c.slot_stride * 2,
                                   (cuuint64_t)c.stream_stride * 2};
    const cuuint32_t box[4] = {64, 1, (cuuint32_t)keys, 1}, estr[4] = {1, 1, 1, 1};
    return fn(m, c.dtype == ELEM_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, base, dims,
              strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// A shape's launch: its cluster size and what that costs.
struct Plan {
    double cost = 1e30;
    int shares = 0;
};

template <int HD, int NT, int RT>
constexpr size_t at_smem() {
    return std::max<size_t>(sizeof(AtSmem<HD, NT, RT>), NT == 2 ? kAtOneCta : 0);
}

template <typename T, int HD, int NT, int RT>
cudaError_t plan_tiles(const RowsAttnParams &p, Plan *out) {
    constexpr int kKeys = at_keys(NT);
    constexpr int kPer = at_ctas(HD, NT, RT);
    constexpr size_t kSmem = at_smem<HD, NT, RT>();
    static_assert(kSmem <= (228 / at_ctas(HD, NT, RT) - 1) * 1024, "they fit an SM");
    auto kernel = attn_rows_tc_kernel<T, HD, NT, RT>;
    static ClusterKernel ck;
    int dev = 0;
    cudaError_t e = cluster_prepare(ck, kernel, kSmem, &dev);
    if (e != cudaSuccess) return e;
    const long long M = (long long)p.r.max_rows * p.group;
    const long long tiles = (M + NT * RT - 1) / (NT * RT);
    const long long clusters = tiles * p.c.n_kv_heads * p.c.n_streams, blocks = (most_keys(p, NT * RT) + kKeys - 1) / kKeys;
    // Shares: the least time in units of a block, with kAtFixed for each wave's
    // starts and merges.  With several CTAs to an SM waves run into each other,
    // so their blocks count in proportion; with one, equal CTAs end together and
    // a started wave is a whole one (4 streams of 400 rows of 32 / 8 heads over
    // 4100 keys, 200 two-tile CTAs: 177 us, 400 of one tile 150; 12 / 12 heads, 16 streams of
    // 800 rows over 5200 keys 598 / 499).  In one wave a CTA
    // alone on its SM is faster than one beside others.  (The device counts
    // these clusters for one CTA to an SM.)
    // 24 x 8 tiles of 65 blocks: 1 share 70 us, 2 58, 4 66; 8 x 8 tiles: 2
    // shares 39, 4 33; 128 tiles of 128 rows, 9 blocks: 1 share 17, 2 25.
    for (int Z = 1; Z <= kMaxCluster && Z <= blocks; Z++) {
        int at_once = 0;
        if ((e = cluster_active(ck, kernel, dev, at_threads(NT, RT), kSmem, Z, &at_once)) != cudaSuccess) return e;
        if (at_once < 1) continue;
        at_once *= kPer;
        const double fill = (double)clusters / at_once, part = (double)blocks / Z;
        const double waves = kPer == 1 ? std::max(1.0, ceil(fill)) : fill > 1.0 ? fill : fill * kPer <= 1.0 ? kAtAlone : 1.0;
        const double t = part * waves + std::max(1.0, ceil(fill)) * kAtFixed + (Z > 1 && RT == kAtRows ? kAtMerge : 0.0);
        if (t < out->cost) {
            out->cost = t;
            out->shares = Z;
        }
    }
    return out->shares ? cudaSuccess : cudaErrorInvalidConfiguration;
}

template <typename T, int HD, int NT, int RT>
cudaError_t launch_tiles(RowsAttnParams p, const Plan &plan, cudaStream_t st, RowsPlan *only) {
    if (only) {
        *only = {NT * RT, at_ctas(HD, NT, RT), plan.shares};
        return cudaSuccess;
    }
    constexpr int kKeys = at_keys(NT);
    const long long M = (long long)p.r.max_rows * p.group;
    const long long tiles = (M + NT * RT - 1) / (NT * RT);
    p.shares = plan.shares;
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg = cluster_config(dim3((unsigned)(p.shares * tiles), p.c.n_kv_heads, p.c.n_streams),
                                                  at_threads(NT, RT), at_smem<HD, NT, RT>(), p.shares, &attr, st);
    CUtensorMap mk = {}, mv = {};
    p.maps = cache_map(&mk, p.c.k + p.layer_off * 2, p.c, kKeys) && cache_map(&mv, p.c.v + p.layer_off * 2, p.c, kKeys);
    return cudaLaunchKernelEx(&cfg, attn_rows_tc_kernel<T, HD, NT, RT>, mk, mv, p);
}

// A block of 128 keys of <2, 128>, of one of 64 of <1, 128>: measured, <1, 128>
// against <2, 128> with 32 / 8 heads of 128: 256 packed rows of 8 streams over
// 512 keys 17 / 27 us, over 4096 keys 66 / 64, of one stream 25 / 29; 1024 rows
// of 8 streams over 4096 keys 195 / 186.
constexpr double kAtTwoTiles = 1.55;

template <typename T, int HD>
cudaError_t launch_typed(const RowsAttnParams &p, cudaStream_t st, RowsPlan *only) {
    const long long M = (long long)p.r.max_rows * p.group;
    Plan one, two;
    cudaError_t e;
    if (M <= 32) {
        if ((e = plan_tiles<T, HD, 1, 32>(p, &one)) != cudaSuccess) return e;
        return launch_tiles<T, HD, 1, 32>(p, one, st, only);
    }
    if ((e = plan_tiles<T, HD, 1, 128>(p, &one)) != cudaSuccess) return e;
    if constexpr (HD == 128)
        if (M > kAtRows) {
            if ((e = plan_tiles<T, HD, 2, 128>(p, &two)) != cudaSuccess) return e;
            if (two.cost * kAtTwoTiles < one.cost) return launch_tiles<T, HD, 2, 128>(p, two, st, only);
        }
    return launch_tiles<T, HD, 1, 128>(p, one, st, only);
}
template <typename T>
cudaError_t launch_dim(const RowsAttnParams &p, cudaStream_t st, RowsPlan *only) {
    return p.c.head_dim == 64 ? launch_typed<T, 64>(p, st, only) : launch_typed<T, 128>(p, st, only);
}

}  // namespace

cudaError_t launch_attn_rows_tc(const RowsAttnParams &p, cudaStream_t st, RowsPlan *only) {
    return p.c.dtype == ELEM_BF16 ? launch_dim<__nv_bfloat16>(p, st, only) : launch_dim<__half>(p, st, only);
}

}  // namespace vc
