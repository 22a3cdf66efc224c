// vc_attn_rows_tc.cu - attention of a call's rows over a 16-bit cache slab on
// the tcgen05 tensor cores: windows, sinks and trees as in vc_attn_rows.cu.
//
// A CTA takes NT (1 or 2) tiles of 128 packed query rows (m = row * group +
// head, TMEM lane = packed row) of one (stream, KV head) and a share of the
// 128-key blocks that they see; the shares of a tile pair are a cluster.
//   warps 0-3, 4-7   softmax of tile 0 and 1, thread = packed row: the block's
//                    maximum over S (TMEM), then P = 2^(s - m), rounded to
//                    the cache's type, over S in TMEM
//   warps 8-11       loads: Q once, then two warps K and two V blocks by
//                    16-byte cp.async into the 128-byte-swizzled operand
//                    layout, two blocks deep, each row from its own slot
//                    (ring wrap, sinks and any stride need no descriptor;
//                    rows past the end are zeros)
//   warp 12          one thread issues the MMAs, M 128:
//                    S_t = Q_t K^T (N 128, K HD) and O_t += P_t V (N HD,
//                    K 128; A from TMEM, V an MN-major operand)
// Per block and tile 2 x 128 x 128 x HD multiply-adds meet 128 x 128
// exponentials: at HD 128 the tensor pipe and the exponential unit are both
// full at the same time, so two tiles alternate - one's softmax runs under the
// other's MMAs - and share each K and V block.
//
// S_t(b + 1) overwrites P_t(b), so it is issued behind O_t += P_t(b) V(b); its
// completion therefore also says that O_t may be rescaled.  The running
// maximum moves only when a block exceeds it by more than 2^8 (P <= 256 in
// either type), and only then O is rescaled.  Rounding P to 16 bits is one
// half step of the type per weight, as the output's own rounding; the sums l
// take the unrounded weights.
//
// Zero times a masked key's NaN or infinity would be NaN: in blocks that some
// row does not see whole, the loading threads look for non-finite V values,
// put zeros in their place and set a flag, and the rows that do see them add
// them at the end.
#include "vc_rows.cuh"
#include "vc_tc.cuh"

#include <algorithm>
#include <atomic>
#include <type_traits>

namespace vc {

using namespace tc;

namespace {

constexpr int kAtKeys = 128;            // keys per block
constexpr int kAtRows = 128;            // packed rows per tile = TMEM lanes
constexpr int kAtLoaders = 64;          // threads that load K, and as many that load V
constexpr int kAtThreads = 13 * 32;
constexpr uint64_t kAtWaitNs = 2000000000ull;
constexpr float kAtRescale = 8.0f;      // log2 of the largest P before the maximum moves
constexpr int kAtOneCta = 120 * 1024;   // more than half an SM's shared memory: one CTA per SM

template <int HD, int NT>
struct AtSmem {
    static constexpr int kTile = 128 * HD * 2;   // bytes of a Q, K or V tile: HD / 64 sub-tiles of [128][128 bytes]
    unsigned char kv[4][kTile];                  // K stages 0, 1, V stages 0, 1; at the end O [NT * 128][HD] fp32
    unsigned char q[NT][kTile];
    uint32_t anc[NT * kAtRows][kTreeMax / 32];
    float mx[NT * kAtRows], sum[NT * kAtRows];
    short parent[kTreeMax];
    uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[NT], p_full[NT], o_done;
    uint32_t tmem;
    int bad;      // a masked block holds non-finite V values
};

template <typename T>
__host__ __device__ constexpr uint32_t at_idesc(int N, bool b_mn) {
    return (1u << 4) | (sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u) |
           (b_mn ? (1u << 16) : 0u) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(kAtRows >> 4) << 24);
}

// MN-major operand, 128-byte swizzle: 64-element atoms along N 16384 bytes
// apart (a sub-tile of 128 keys), 8-key groups 1024 bytes apart.
__device__ __forceinline__ uint64_t at_desc_mn(const void *p) {
    const uint64_t addr = smem_u32(p);
    return ((addr >> 4) & 0x3FFFull) | ((uint64_t)(16384 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) |
           (2ull << 61);
}

// D[tmem] (+)= A[tmem] . B[smem]: A holds two 16-bit values per column.
__device__ __forceinline__ void tc_mma_f16_ta(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                              uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// 16 columns of this thread's TMEM lane
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
            taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
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

template <typename T>
__device__ __forceinline__ uint32_t nonfinite2(uint32_t u) {   // 0xffff in each half that is inf or NaN
    constexpr uint32_t e = std::is_same<T, __nv_bfloat16>::value ? 0x7f807f80u : 0x7c007c00u;
    return __vcmpeq2(u & e, e);
}

template <typename T, int HD, int NT>
__global__ void __launch_bounds__(kAtThreads, 1) attn_rows_tc_kernel(const RowsAttnParams p) {
    using Sm = AtSmem<HD, NT>;
    constexpr int kSub = HD / 64;            // 64-dim sub-tiles of a tile
    constexpr uint32_t kTmemCols = NT == 2 ? 512 : 256;
    extern __shared__ __align__(1024) unsigned char at_smem_raw[];
    Sm &sh = *reinterpret_cast<Sm *>(at_smem_raw);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int z = blockIdx.x % p.shares, Z = p.shares;
    const int m0 = blockIdx.x / p.shares * (NT * kAtRows), kvh = blockIdx.y, stream = blockIdx.z;
    const RowSpan s = row_span(p.r, stream);
    const int M = s.n * p.group;
    if (m0 >= M) return;   // the whole cluster leaves
    const bool tree = p.r.parent != nullptr;
    const int i0 = m0 / p.group, i1 = (min(m0 + NT * kAtRows, M) - 1) / p.group + 1;
    const KeyRange kr = key_range(p.c, s, i0, i1, p.window, tree);
    const int total = kr.total(), blocks = (total + kAtKeys - 1) / kAtKeys;
    const int b0 = (int)((long long)z * blocks / Z), nb = (int)((long long)(z + 1) * blocks / Z) - b0;
    const int tiles = M - m0 > kAtRows ? NT : 1;   // tiles with rows
    const int head0 = kvh * p.group;
    const uint64_t deadline = globaltimer() + kAtWaitNs;
    bool ok = true;

    // keys that every row of the CTA sees, in the walk's order: [core_s, core_e)
    // (and [0, ns) when core_s = ns, contiguous with it)
    const int up_min = tree ? s.pos - 1 : s.pos + i0;
    int core_s = kr.ns + (p.window > 0 ? max(0, min(s.pos + i1 - p.window - kr.lo, kr.nm)) : 0), core_e = kr.ns + max(0, min(up_min - kr.lo + 1, kr.nm));
    if (up_min < kr.ns - 1) core_e = 0;
    else if (core_s == kr.ns) core_s = 0;
    auto whole = [&](int b) { return b * kAtKeys >= core_s && (b + 1) * kAtKeys <= core_e; };

    if (threadIdx.x == 0) {
        mbar_init(&sh.q_full, 2 * kAtLoaders);
        for (int i = 0; i < 2; i++) {
            mbar_init(&sh.k_full[i], kAtLoaders);
            mbar_init(&sh.v_full[i], kAtLoaders);
            mbar_init(&sh.k_empty[i], 1);
            mbar_init(&sh.v_empty[i], 1);
        }
        for (int t = 0; t < NT; t++) {
            mbar_init(&sh.s_full[t], 1);
            // one arrival per warp with rows
            mbar_init(&sh.p_full[t], max(1, min(4, (M - m0 - t * kAtRows + 31) / 32)));
        }
        mbar_init(&sh.o_done, 1);
        sh.bad = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 12) {
        tmem_alloc(&sh.tmem, kTmemCols);
        tmem_relinquish();
    }
    if (tree) load_parents(sh.parent, p.r, s, threadIdx.x, kAtThreads);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    constexpr uint32_t kOCol = NT * kAtKeys;   // S tiles first, then O tiles

    if (warp >= 8 && warp < 12) {
        // ---- loads: warps 8, 9 K, warps 10, 11 V, all of them Q ----
        const int tid = threadIdx.x & (kAtLoaders - 1);
        const bool is_v = warp >= 10;
        constexpr int kCh = HD / 8;                   // 16-byte chunks per row
        constexpr int kRowsAtOnce = kAtLoaders / kCh;
        const int ch = tid % kCh, jr = tid / kCh;
        // chunk ch of row r: sub-tile ch / 8, swizzled by the row
        auto at = [&](int r) { return (ch >> 3) * 16384 + r * 128 + (((ch & 7) ^ (r & 7)) << 4); };
        for (int t = 0; t < tiles; t++) {
            const uint32_t dst = smem_u32(sh.q[t]);
#pragma unroll
            for (int it = 0; it < kAtRows / 2 / kRowsAtOnce; it++) {
                const int r = (2 * it + is_v) * kRowsAtOnce + jr, m = m0 + t * kAtRows + r;
                const T *src = static_cast<const T *>(p.q);
                if (m < M) src += ((long long)(s.r0 + m / p.group) * p.n_heads + head0 + m % p.group) * HD + ch * 8;
                cp_async16(dst + at(r), src, m < M);
            }
        }
        cp_async_commit();
        const long long base = p.layer_off + (long long)stream * p.c.stream_stride + (long long)kvh * p.c.head_stride;
        const char *src = (is_v ? p.c.v : p.c.k) + base * 2 + ch * 16;
        const long long slot_bytes = p.c.slot_stride * 2;
        const int lo_slot = cache_slot(p.c, kr.lo);
        unsigned char *const bufs = sh.kv[is_v ? 2 : 0];
        uint64_t *const full = is_v ? sh.v_full : sh.k_full, *const empty = is_v ? sh.v_empty : sh.k_empty;
        auto publish = [&](int b) {   // block b (of this share) has landed
            if (is_v && !whole(b0 + b)) {
                unsigned char *v = bufs + (b & 1) * Sm::kTile;
                bool found = false;
#pragma unroll 4
                for (int it = 0; it < kAtKeys / kRowsAtOnce; it++) {
                    uint4 *c = reinterpret_cast<uint4 *>(v + at(it * kRowsAtOnce + jr));
                    uint4 u = *c;
                    const uint4 n = make_uint4(nonfinite2<T>(u.x), nonfinite2<T>(u.y), nonfinite2<T>(u.z), nonfinite2<T>(u.w));
                    if (n.x | n.y | n.z | n.w) {
                        *c = make_uint4(u.x & ~n.x, u.y & ~n.y, u.z & ~n.z, u.w & ~n.w);
                        found = true;
                    }
                }
                if (found) atomicExch(&sh.bad, 1);
            }
            fence_async_smem();
            if (b == 0) mbar_arrive(&sh.q_full);   // Q was ahead of it
            mbar_arrive(&full[b & 1]);
        };
        for (int b = 0; b < nb; b++) {
            if (b >= 2 && !mbar_wait(&empty[b & 1], ((b >> 1) + 1) & 1u, deadline)) {
                ok = false;
                break;
            }
            const uint32_t dst = smem_u32(bufs + (b & 1) * Sm::kTile);
            const int idx0 = (b0 + b) * kAtKeys;
            int slot0 = lo_slot + (idx0 - kr.ns);   // of index idx0, past the sinks
            if (slot0 >= p.c.cap) slot0 -= p.c.ring;
            if (idx0 >= kr.ns && idx0 + kAtKeys <= total && slot0 + kAtKeys <= p.c.cap) {
                const char *a = src + (slot0 + jr) * slot_bytes;   // 128 slots in a row
                const long long step = kRowsAtOnce * slot_bytes;
#pragma unroll 8
                for (int it = 0; it < kAtKeys / kRowsAtOnce; it++) {
                    cp_async16(dst + at(it * kRowsAtOnce + jr), a, true);
                    a += step;
                }
            } else {
#pragma unroll 4
                for (int it = 0; it < kAtKeys / kRowsAtOnce; it++) {
                    const int r = it * kRowsAtOnce + jr, idx = idx0 + r;
                    int slot = idx;
                    if (idx >= kr.ns) {
                        slot = lo_slot + (idx - kr.ns);
                        if (slot >= p.c.cap) slot -= p.c.ring;
                    }
                    cp_async16(dst + at(r), src + (idx < total ? slot * slot_bytes : 0), idx < total);
                }
            }
            cp_async_commit();
            if (b >= 1) {
                cp_async_wait<1>();
                publish(b - 1);
            }
        }
        cp_async_wait<0>();
        if (ok && nb > 0) publish(nb - 1);
    } else if (warp == 12) {
        // ---- MMAs ----
        if (lane == 0 && nb > 0) {
            constexpr uint32_t id_s = at_idesc<T>(kAtKeys, false), id_o = at_idesc<T>(HD, true);
            auto issue_s = [&](int t, int b) {
                const uint64_t a0 = smem_desc_sw128(sh.q[t]), k0 = smem_desc_sw128(sh.kv[b & 1]);
#pragma unroll
                for (int h = 0; h < kSub; h++)
#pragma unroll
                    for (int k = 0; k < 4; k++)   // 16 dims: +32 bytes
                        tc_mma_f16(tmem + t * kAtKeys, a0 + h * 1024 + 2 * k, k0 + h * 1024 + 2 * k, id_s,
                                   (h | k) != 0 ? 1u : 0u);
                tc_commit(&sh.s_full[t]);
            };
            ok = mbar_wait(&sh.q_full, 0u, deadline) && mbar_wait(&sh.k_full[0], 0u, deadline);
            if (ok) {
                tc_fence_after();
                for (int t = 0; t < tiles; t++) issue_s(t, 0);
                tc_commit(&sh.k_empty[0]);
            }
            for (int b = 0; b < nb && ok; b++) {
                for (int t = 0; t < tiles && ok; t++) {
                    ok = mbar_wait(&sh.p_full[t], b & 1u, deadline) &&
                         (t > 0 || mbar_wait(&sh.v_full[b & 1], (b >> 1) & 1u, deadline));
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll
                    for (int k = 0; k < kAtKeys / 16; k++)   // 16 keys: 8 columns of P, 2048 bytes of V
                        tc_mma_f16_ta(tmem + kOCol + t * HD, tmem + t * kAtKeys + 8 * k,
                                      at_desc_mn(sh.kv[2 + (b & 1)] + k * 2048), id_o, (b | k) != 0 ? 1u : 0u);
                    if (t == tiles - 1) tc_commit(&sh.v_empty[b & 1]);
                    if (b + 1 < nb) {
                        if (t == 0) {
                            ok = mbar_wait(&sh.k_full[(b + 1) & 1], ((b + 1) >> 1) & 1u, deadline);
                            if (!ok) break;
                            tc_fence_after();
                        }
                        issue_s(t, b + 1);
                        if (t == tiles - 1) tc_commit(&sh.k_empty[(b + 1) & 1]);
                    }
                }
            }
            tc_commit(&sh.o_done);
        }
    } else {
        // ---- softmax: thread = packed row ----
        const int t = warp >> 2, q = warp & 3, ml = t * kAtRows + 32 * q + lane, m = m0 + ml;
        const bool here = t < NT && m0 + t * kAtRows + 32 * q < M;   // the warp has rows
        if (here) {
            const int i = min(m, M - 1) / p.group;
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
            const uint32_t ts = tl + t * kAtKeys, to = tl + kOCol + t * HD;
            const float sl2 = p.scale_log2;
            const bool neg = sl2 < 0.f;
            const float hidden = neg ? INFINITY : -INFINITY;   // a masked key's score
            float mr = -INFINITY, l = 0.f;
            float sv[32];
            for (int b = 0; b < nb; b++) {
                if (!__all_sync(0xffffffffu, mbar_wait(&sh.s_full[t], b & 1u, deadline))) ok = false;
                tc_fence_after();
                const int c0 = (b0 + b) * kAtKeys;
                const bool full = whole(b0 + b);
                float mx[4] = {hidden, hidden, hidden, hidden};
#pragma unroll
                for (int c = 0; c < kAtKeys; c += 32) {
                    tmem_ld32(ts + c, sv);
                    if (!full) {
                        const uint32_t vis = keys.bits(c0 + c, anc);
#pragma unroll
                        for (int j = 0; j < 32; j++) sv[j] = (vis >> j) & 1u ? sv[j] : hidden;
                    }
                    if (neg) {
#pragma unroll
                        for (int j = 0; j < 32; j++) mx[j & 3] = fminf(mx[j & 3], sv[j]);
                    } else {
#pragma unroll
                        for (int j = 0; j < 32; j++) mx[j & 3] = fmaxf(mx[j & 3], sv[j]);
                    }
                }
                const float mb = sl2 * (neg ? fminf(fminf(mx[0], mx[1]), fminf(mx[2], mx[3]))
                                            : fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])));
                const bool move = mb > mr + kAtRescale;
                float factor = 1.f;
                if (move) {
                    factor = mr == -INFINITY ? 0.f : exp2_approx(mr - mb);
                    mr = mb;
                    l *= factor;
                }
                const float base = mr == -INFINITY ? 0.f : mr;
                float rs[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < kAtKeys; c += 32) {
                    tmem_ld32(ts + c, sv);
                    if (!full) {
                        const uint32_t vis = keys.bits(c0 + c, anc);
#pragma unroll
                        for (int j = 0; j < 32; j++) sv[j] = (vis >> j) & 1u ? sv[j] : hidden;
                    }
                    uint32_t h[16];
#pragma unroll
                    for (int j = 0; j < 32; j += 2) {
                        const float ea = exp2_approx(fmaf(sv[j], sl2, -base));
                        const float eb = exp2_approx(fmaf(sv[j + 1], sl2, -base));
                        rs[(j >> 1) & 3] += ea + eb;
                        h[j >> 1] = pack2<T>(ea, eb);
                    }
                    tmem_st16(ts + c / 2, h);   // over S columns that were read already
                }
                l += (rs[0] + rs[1]) + (rs[2] + rs[3]);
                // O_t += P_t(b - 1) V(b - 1) is complete (S_t(b) was behind it)
                if (b > 0 && __any_sync(0xffffffffu, move)) {
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
                if (lane == 0) mbar_arrive(&sh.p_full[t]);
            }
            if (nb > 0 && !__all_sync(0xffffffffu, mbar_wait(&sh.o_done, 0u, deadline))) ok = false;
            tc_fence_after();
            const float il = l == 0.f ? 0.f : 1.0f / l;   // no weight at all: zeros
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
                    for (int idx = b0 * kAtKeys; idx < min(total, (b0 + nb) * kAtKeys); idx++) {
                        if (whole(idx / kAtKeys) || !((keys.bits(idx & ~31, anc) >> (idx & 31)) & 1u)) continue;
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
                    float *o = reinterpret_cast<float *>(sh.kv[0]) + ml * HD;
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
        if (p.err) atomicExch_system(p.err, 1u);
        const uint64_t grace = globaltimer() + 10000000ull;   // let copies and MMAs in flight land
        while (globaltimer() < grace) {
        }
    }
    // TMEM goes back before the cluster meets: no CTA holds it while it waits
    // for a peer that may itself wait for TMEM
    tc_fence_before();
    __syncthreads();
    if (warp == 12) {
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
    if (Z > 1) {
        cluster_sync_all();
        const uint32_t o_s = smem_u32(sh.kv[0]), m_s = smem_u32(sh.mx), l_s = smem_u32(sh.sum);
        const int rows = min(NT * kAtRows, M - m0);
        for (int e = z * kAtThreads + threadIdx.x; e < rows * (HD / 4); e += Z * kAtThreads) {
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

template <typename T, int HD, int NT>
cudaError_t launch_tiles(RowsAttnParams p, int sms, cudaStream_t st) {
    constexpr size_t kSmem = std::max<size_t>(sizeof(AtSmem<HD, NT>), NT == 2 ? kAtOneCta : 0);
    static_assert(kSmem <= 227 * 1024, "fits an SM");
    auto kernel = attn_rows_tc_kernel<T, HD, NT>;
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (!(done.load() & bit)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
        done.fetch_or(bit);
    }
    const long long M = (long long)p.r.max_rows * p.group;
    const long long tiles = (M + NT * kAtRows - 1) / (NT * kAtRows);
    const long long keys =
        p.window > 0 ? std::min<long long>(p.c.cap, (long long)p.window + p.r.max_rows + p.c.n_sink) : p.c.cap;
    const long long ctas = tiles * p.c.n_kv_heads * p.c.n_streams;
    const long long by_sms = std::max<long long>(1, sms / ctas), by_keys = (keys + kAtKeys - 1) / kAtKeys;
    p.shares = (int)std::max<long long>(1, std::min<long long>(16, std::min(by_sms, by_keys)));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(p.shares * tiles), p.c.n_kv_heads, p.c.n_streams);
    cfg.blockDim = dim3(kAtThreads);
    cfg.dynamicSmemBytes = kSmem;
    cfg.stream = st;
    cudaLaunchAttribute a[1];
    a[0].id = cudaLaunchAttributeClusterDimension;
    a[0].val.clusterDim.x = p.shares;
    a[0].val.clusterDim.y = 1;
    a[0].val.clusterDim.z = 1;
    cfg.attrs = a;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <typename T>
cudaError_t launch_typed(const RowsAttnParams &p, int sms, cudaStream_t st) {
    const bool two = (long long)p.r.max_rows * p.group > kAtRows;
    if (p.c.head_dim == 64) return two ? launch_tiles<T, 64, 2>(p, sms, st) : launch_tiles<T, 64, 1>(p, sms, st);
    return two ? launch_tiles<T, 128, 2>(p, sms, st) : launch_tiles<T, 128, 1>(p, sms, st);
}

}  // namespace

cudaError_t launch_attn_rows_tc(const RowsAttnParams &p, int sms, cudaStream_t st) {
    return p.c.dtype == ELEM_BF16 ? launch_typed<__nv_bfloat16>(p, sms, st) : launch_typed<__half>(p, sms, st);
}

}  // namespace vc
