// vc_attn_rows.cu - attention of a call's rows over a cache slab, with a
// sliding window, sinks that stay visible, and trees of drafted rows: the fp32
// kernels, on the CUDA cores (16-bit slabs: vc_attn_rows_tc.cu).
//
// o = sum_j 2^(s_j - m) v_j / l, s = scale * log2(e) * q.k, over the keys that
// the row sees (vc_rows.cuh), in one pass with a running maximum m and sum l.
// A masked key adds nothing, whatever its K and V hold.
//
// A CTA takes a tile of RB query rows of one (stream, KV head) - row i and
// query head g of the group are packed as m = i * group + g, so a KV head's
// keys are read once for its whole group - and a share of the keys that the
// tile sees.  The shares of a tile are the CTAs of one cluster; they merge
// through distributed shared memory, in rank order, so there is no workspace,
// no ticket and no second launch, and a result does not depend on timing.
#include "vc_cluster.h"
#include "vc_rows.cuh"
#include "vc_tc.cuh"

#include <algorithm>
#include <atomic>
#include <type_traits>

namespace vc {

using namespace tc;

namespace {

// What a tile's rows see, and where they are (shared memory).
template <int RB>
struct ArRows {
    int up[RB], low[RB];
    uint32_t anc[RB][kTreeMax / 32];
    short parent[kTreeMax];
};

template <int RB>
__device__ __forceinline__ void setup_rows(ArRows<RB> &rows, const RowsAttnParams &p, const RowSpan &s, int m0, int M) {
    const bool tree = p.r.parent != nullptr;
    if (tree) {
        load_parents(rows.parent, p.r, s, threadIdx.x, blockDim.x);
        __syncthreads();
    }
    for (int m = threadIdx.x; m < RB; m += blockDim.x) {
        const int i = min(m0 + m, M - 1) / p.group;   // rows past the tile repeat the last one
        int at = s.pos + i;
        if (tree) {
#pragma unroll
            for (int w = 0; w < kTreeMax / 32; w++) rows.anc[m][w] = 0u;
            const int depth = ancestor_bits(rows.anc[m], rows.parent, i);
            window_bits(rows.anc[m], rows.parent, i, depth, s.pos, p.c.n_sink, p.window);
            at = s.pos + depth;
        }
        rows.up[m] = tree ? s.pos - 1 : at;
        rows.low[m] = p.window > 0 ? at - p.window + 1 : INT_MIN;
    }
}

template <int RB>
__device__ __forceinline__ bool row_sees(const ArRows<RB> &rows, int m, int j, int pos, int n_sink, bool tree) {
    if (j <= rows.up[m]) return j < n_sink || j >= rows.low[m];
    const int a = j - pos;
    return tree && ((rows.anc[m][a >> 5] >> (a & 31)) & 1u);
}

// The tile's query rows, scaled, into shared memory: `row` floats apart, and 4
// floats more between the `parts` of a row; zeros past M.
template <int HD, int RB>
__device__ __forceinline__ void load_queries(float *q, int row, int parts, const RowsAttnParams &p, const RowSpan &s,
                                             int head0, int m0, int M) {
    for (int e = threadIdx.x; e < RB * HD / 4; e += blockDim.x) {
        const int m = e / (HD / 4), d = e % (HD / 4) * 4;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (m0 + m < M) {
            const int i = (m0 + m) / p.group, g = (m0 + m) % p.group;
            v = load4<float>(static_cast<const float *>(p.q) + ((long long)(s.r0 + i) * p.n_heads + head0 + g) * HD + d);
            v = make_float4(v.x * p.scale_log2, v.y * p.scale_log2, v.z * p.scale_log2, v.w * p.scale_log2);
        }
        *reinterpret_cast<float4 *>(q + m * row + d + d / (HD / parts) * 4) = v;
    }
}

// o += P V of a warp's tile, whose lanes hold which of the R rows see their two
// keys (vis); weigh(j, v, rows) adds key j's to some rows.  A masked key's
// weight is 0, but 0 times a NaN or an infinity is NaN: where a tile has masked
// keys and the sums come out NaN, they are taken back and such keys skipped.
template <int HD, int KEYS, int R, typename Weigh>
__device__ __forceinline__ void add_values(uint64_t (&o)[R][2], const unsigned char *vt, const uint32_t (&vis)[2], int sub,
                                           int d4, Weigh weigh) {
    constexpr int kPvKeys = 128 / HD;   // keys that the lanes take at once
    constexpr uint32_t kAll = (1u << R) - 1u;
    const bool masked = __any_sync(0xffffffffu, (vis[0] & vis[1]) != kAll);
    uint64_t before[R][2];
    if (masked) {
#pragma unroll
        for (int r = 0; r < R; r++) {
            before[r][0] = o[r][0];
            before[r][1] = o[r][1];
        }
    }
#pragma unroll 4
    for (int x = 0; x < KEYS / kPvKeys; x++) {
        const int j = x * kPvKeys + sub;
        weigh(j, *reinterpret_cast<const ulonglong2 *>(vt + (j * HD + d4) * 4), kAll);
    }
    if (!masked) return;
    bool nan = false;
#pragma unroll
    for (int r = 0; r < R; r++) {
        float a, b, c, d;
        unpair(o[r][0], a, b);
        unpair(o[r][1], c, d);
        nan |= a != a || b != b || c != c || d != d;
    }
    if (!__any_sync(0xffffffffu, nan)) return;
#pragma unroll
    for (int r = 0; r < R; r++) {
        o[r][0] = before[r][0];
        o[r][1] = before[r][1];
    }
#pragma unroll 1
    for (int x = 0; x < KEYS / kPvKeys; x++) {
        const int j = x * kPvKeys + sub;
        const uint32_t v0 = __shfl_sync(0xffffffffu, vis[0], j % (KEYS / 2)), v1 = __shfl_sync(0xffffffffu, vis[1], j % (KEYS / 2));
        weigh(j, *reinterpret_cast<const ulonglong2 *>(vt + (j * HD + d4) * 4), j < KEYS / 2 ? v0 : v1);
    }
}

// The shares of a tile merge by pushing: rank z owns a Z-th of the tile's sums
// (groups of 4 dims), every CTA writes its part of them, and its rows' maxima
// and sums, into the owners' shared memory, and after one cluster barrier each
// owner finds all parts in its own.
template <int HD, int RB>
struct ArMerge {
    static constexpr int kGroups = RB * HD / 4;
    float4 part[kGroups + kMaxCluster];       // [rank][group of this owner]
    float2 ml[kMaxCluster][RB];               // the ranks' maxima and sums
};

// Called once by every thread before merge_store, early: the peers have started.
__device__ __forceinline__ void peers_arrive(int Z) {
    if (Z > 1) asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
}
__device__ __forceinline__ void peers_wait(int Z) {
    if (Z > 1) asm volatile("barrier.cluster.wait;" ::: "memory");
}

// sum(r, d): this CTA's unnormalised sums of row r, dims d .. d + 3; ml(r): its
// maximum and sum.
template <int HD, int RB, int NTH, typename Sum, typename Ml>
__device__ __forceinline__ void merge_store(ArMerge<HD, RB> &mg, Sum sum, Ml ml, const RowsAttnParams &p, const RowSpan &s,
                                            int head0, int m0, int M, int z, int Z) {
    constexpr int N = ArMerge<HD, RB>::kGroups;
    const int per = (N + Z - 1) / Z;
    peers_wait(Z);
    for (int e = threadIdx.x; e < N; e += NTH) {
        const int owner = e / per, at = z * per + e - owner * per;
        const float4 v = sum(e / (HD / 4), e % (HD / 4) * 4);
        asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(mapa_shared(smem_u32(mg.part + at), owner)),
                     "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w)
                     : "memory");
    }
    for (int e = threadIdx.x; e < RB * Z; e += NTH) {
        const float2 v = ml(e % RB);
        asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(mapa_shared(smem_u32(&mg.ml[z][e % RB]), e / RB)),
                     "f"(v.x), "f"(v.y)
                     : "memory");
    }
    if (Z > 1) cluster_sync_all();
    else __syncthreads();
    for (int e = z * per + threadIdx.x; e < min(N, (z + 1) * per); e += NTH) {
        const int m = e / (HD / 4), d = e % (HD / 4) * 4;
        if (m0 + m >= M) continue;
        float gm = -INFINITY;
#pragma unroll 4
        for (int r = 0; r < Z; r++) gm = fmaxf(gm, mg.ml[r][m].x);
        float gl = 0.f;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int r = 0; r < Z; r++) {
            const float2 w = mg.ml[r][m];
            const float4 v = mg.part[r * per + e - z * per];
            if (w.x == -INFINITY && w.y == 0.f) continue;   // this share saw no key of the row
            const float f = w.x == -INFINITY ? 0.f : exp2_approx(w.x - gm);
            gl = fmaf(f, w.y, gl);
            a = make_float4(fmaf(f, v.x, a.x), fmaf(f, v.y, a.y), fmaf(f, v.z, a.z), fmaf(f, v.w, a.w));
        }
        const float il = gl == 0.f ? 0.f : 1.0f / gl;   // no key at all: zeros
        const long long row = (long long)(s.r0 + (m0 + m) / p.group) * p.n_heads + head0 + (m0 + m) % p.group;
        store4<float>(static_cast<float *>(p.out) + row * HD + d, make_float4(a.x * il, a.y * il, a.z * il, a.w * il));
        if (p.lse && d == 0) p.lse[row] = gl == 0.f ? -INFINITY : (gm + log2f(gl)) * 0.69314718055994531f;
    }
}

// ---------------------------------------------------------------------------
// Few rows: RB (4 or 8) packed rows.
//
// Bound by HBM at long contexts: 2 * RB flops per byte.  A warp works on tiles
// of its own - 8 KB of K and as much of V - so nothing but its own copies holds
// it up (16 bytes per lane: a bulk copy per row costs the warp a turn per
// lane): the next tile's K is on its way from when the scores are done, its V
// from when P.V is, and the other warps work meanwhile.  A K row is 16
// bytes longer than a key, so that lanes read one chunk of different keys
// without conflicts.  One token of 32 / 8 heads over 8196 keys: 22.5 us, 3.0
// TB/s - 8 clusters of 10 CTAs, so 80 SMs, of which each moves 37 GB/s, and
// about 8 us of launch, start and merge; 8 rows over 748 keys: 14.3 us.
// Scores: a lane has 32 dims of two keys against RB
// broadcast rows; the running maximum moves only when a score exceeds it by
// more than 2^8, so most tiles need no shuffles across keys.  P.V: a lane has 4
// dims of every row.
// ---------------------------------------------------------------------------

// Warps of a CTA: one CTA fills an SM's shared memory, or (small) four do, for
// tiles of few keys.
constexpr int af_warps(int hd, int rb, bool small) { return small ? (rb == 8 ? 2 : 3) : hd == 64 && rb == 8 ? 11 : 12; }
constexpr int kAfTile = 8192;              // K bytes of a warp's tile
constexpr float kAfRescale = 8.0f;         // log2 of the largest weight before the maximum moves
constexpr double kArFixed = 4;             // rounds' worth of a CTA's start and merge

template <int HD, int RB, bool SMALL>
struct AfSmem {
    static constexpr int kWarps = af_warps(HD, RB, SMALL), kThreads = kWarps * 32;
    static constexpr int kKeys = kAfTile / (HD * 4);       // keys of a tile: 16 or 32
    static constexpr int kRow = HD * 4 + 16;               // a K row in shared memory
    static constexpr int kParts = HD / 32;                 // lanes that share a key: 4 or 2
    static constexpr int kAtOnce = 32 / kParts;            // keys that the lanes hold at once: half a tile
    static constexpr int kQRow = HD + 4 * (kParts - 1);    // a query row: its parts on different banks
    struct Tile {
        unsigned char k[kKeys * kRow];
        unsigned char v[kAfTile];
    };
    union {
        Tile tile[kWarps];
        float sums[kWarps][RB][HD];       // the warps' at the end
    };
    float q[RB * kQRow];
    float2 p[kWarps][kKeys][RB];          // 2^(s - m) twice
    float wm[kWarps][RB], wl[kWarps][RB], wf[kWarps][RB];
    float mx[RB], sum[RB];
    ArMerge<HD, RB> merge;
    ArRows<RB> rows;
};

template <int HD, int RB, bool SMALL>
__global__ void __launch_bounds__(AfSmem<HD, RB, SMALL>::kThreads) attn_rows_few_kernel(const RowsAttnParams p) {
    using Sm = AfSmem<HD, RB, SMALL>;
    constexpr int kAfWarps = Sm::kWarps, kAfThreads = Sm::kThreads;
    static_assert(sizeof(Sm) <= 227 * 1024, "fits an SM");
    extern __shared__ __align__(128) unsigned char smem_raw[];
    Sm &sh = *reinterpret_cast<Sm *>(smem_raw);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int z = blockIdx.x % p.shares, Z = p.shares;
    const int m0 = blockIdx.x / p.shares * RB, kvh = blockIdx.y, stream = blockIdx.z;
    const RowSpan s = row_span(p.r, stream);
    const int M = s.n * p.group;
    if (m0 >= M) return;   // the whole cluster leaves
    const bool tree = p.r.parent != nullptr;
    const int i0 = m0 / p.group, i1 = (min(m0 + RB, M) - 1) / p.group + 1;
    const KeyRange kr = key_range(p.c, s, i0, i1, p.window, tree);
    const int lo_slot = cache_slot(p.c, kr.lo);
    const int total = kr.total(), tiles = (total + Sm::kKeys - 1) / Sm::kKeys;
    // the warp's tiles: every (Z * kAfWarps)-th
    const int t0 = z + warp * Z, step = Z * kAfWarps;
    const long long base = p.layer_off + (long long)stream * p.c.stream_stride + (long long)kvh * p.c.head_stride;
    const char *kb = p.c.k + base * 4, *vb = p.c.v + base * 4;
    const long long slot_bytes = p.c.slot_stride * 4;
    const int head0 = kvh * p.group;
    // a group of copies even where no tile is left, so that the groups count
    constexpr int kCh = HD / 4, kRowsAtOnce = 32 / kCh;   // 16-byte chunks of a row
    const int ch = lane % kCh, jr = lane / kCh;
    typename Sm::Tile &tl = sh.tile[warp];
    auto fetch = [&](int t, bool is_v) {
        const int idx0 = t * Sm::kKeys;
        if (t < tiles) {
            const char *src = is_v ? vb : kb;
            const int row = is_v ? HD * 4 : Sm::kRow;
            const uint32_t dst = smem_u32(is_v ? tl.v : tl.k) + jr * row + ch * 16;
            int slot0 = lo_slot + (idx0 - kr.ns);   // of index idx0, past the sinks
            if (slot0 >= p.c.cap) slot0 -= p.c.ring;
            const bool run = idx0 >= kr.ns && idx0 + Sm::kKeys <= total && slot0 + Sm::kKeys <= p.c.cap;
            constexpr int kIts = Sm::kKeys / kRowsAtOnce;
            if (run) {
                const char *a = src + (slot0 + jr) * slot_bytes + ch * 16;
                const long long step_bytes = kRowsAtOnce * slot_bytes;
#pragma unroll
                for (int it = 0; it < kIts; it++, a += step_bytes) cp_async16(dst + it * kRowsAtOnce * row, a, true);
            } else {
#pragma unroll 1
                for (int it = 0; it < kIts; it++) {
                    const int idx = idx0 + it * kRowsAtOnce + jr;
                    int slot = idx;
                    if (idx >= kr.ns) {
                        slot = lo_slot + (idx - kr.ns);
                        if (slot >= p.c.cap) slot -= p.c.ring;
                    }
                    const bool ok = idx < total;
                    cp_async16(dst + it * kRowsAtOnce * row, src + (ok ? slot * slot_bytes + ch * 16 : 0), ok);
                }
            }
        }
        cp_async_commit();
    };
    peers_arrive(Z);
    fetch(t0, false);
    fetch(t0, true);

    load_queries<HD, RB>(sh.q, Sm::kQRow, Sm::kParts, p, s, head0, m0, M);
    setup_rows<RB>(sh.rows, p, s, m0, M);
    __syncthreads();

    constexpr int kLanesPerKey = HD / 4, kPvKeys = 32 / kLanesPerKey;   // P.V
    const int j = lane % Sm::kAtOnce, part = lane / Sm::kAtOnce;        // scores: keys j and j + kAtOnce
    const int sub = lane / kLanesPerKey, d4 = lane % kLanesPerKey * 4;
    float mr[RB], l[RB];   // l: this lane's keys only
    uint64_t o[RB][2];     // pairs of dims
#pragma unroll
    for (int r = 0; r < RB; r++) {
        mr[r] = -INFINITY;
        l[r] = 0.f;
        o[r][0] = o[r][1] = 0;
    }
    // keys that every row of the tile sees, in the walk's order
    const int up_min = tree ? s.pos - 1 : s.pos + i0;
    int core_s = kr.ns + (p.window > 0 ? max(0, min(s.pos + i1 - p.window - kr.lo, kr.nm)) : 0);
    int core_e = kr.ns + max(0, min(up_min - kr.lo + 1, kr.nm));
    if (up_min < kr.ns - 1) core_e = 0;
    else if (core_s == kr.ns) core_s = 0;
    for (int t = t0; t < tiles; t += step) {
        cp_async_wait<1>();   // K is in
        __syncwarp();
        uint64_t a2[2][RB];
#pragma unroll
        for (int r = 0; r < RB; r++) a2[0][r] = a2[1][r] = 0;
#pragma unroll
        for (int c = 0; c < 8; c++) {
            const unsigned char *kp = tl.k + j * Sm::kRow + (part * 8 + c) * 16;
            const ulonglong2 k0 = *reinterpret_cast<const ulonglong2 *>(kp);
            const ulonglong2 k1 = *reinterpret_cast<const ulonglong2 *>(kp + Sm::kAtOnce * Sm::kRow);
#pragma unroll
            for (int r = 0; r < RB; r++) {
                const ulonglong2 q = *reinterpret_cast<const ulonglong2 *>(sh.q + r * Sm::kQRow + part * 36 + c * 4);
                a2[0][r] = fma2(q.x, k0.x, a2[0][r]);
                a2[1][r] = fma2(q.x, k1.x, a2[1][r]);
                a2[0][r] = fma2(q.y, k0.y, a2[0][r]);
                a2[1][r] = fma2(q.y, k1.y, a2[1][r]);
            }
        }
        __syncwarp();
        fetch(t + step, false);
        float acc[2][RB];
#pragma unroll
        for (int x = 0; x < 2; x++)
#pragma unroll
            for (int r = 0; r < RB; r++) {
                float a, b;
                unpair(a2[x][r], a, b);
                acc[x][r] = a + b;
#pragma unroll
                for (int d = Sm::kAtOnce; d < 32; d *= 2) acc[x][r] += __shfl_xor_sync(0xffffffffu, acc[x][r], d);
            }
        uint32_t vis[2] = {(1u << RB) - 1u, (1u << RB) - 1u};
        const bool whole = t * Sm::kKeys >= core_s && (t + 1) * Sm::kKeys <= core_e;
        if (!whole) {
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const int idx = t * Sm::kKeys + x * Sm::kAtOnce + j, at = kr.position(idx);
                vis[x] = 0;
                if (idx < total)
#pragma unroll
                    for (int r = 0; r < RB; r++)
                        if (row_sees<RB>(sh.rows, r, at, s.pos, p.c.n_sink, tree)) vis[x] |= 1u << r;
#pragma unroll
                for (int r = 0; r < RB; r++)
                    if (!((vis[x] >> r) & 1u)) acc[x][r] = -INFINITY;
            }
        }
        bool move = false;
#pragma unroll
        for (int r = 0; r < RB; r++) {
            const float a = fmaxf(acc[0][r], acc[1][r]);
            move |= mr[r] == -INFINITY ? a > -INFINITY : a > mr[r] + kAfRescale;
        }
        if (__any_sync(0xffffffffu, move)) {
#pragma unroll
            for (int r = 0; r < RB; r++) {
                float mt = fmaxf(acc[0][r], acc[1][r]);
#pragma unroll
                for (int d = Sm::kAtOnce / 2; d > 0; d >>= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, d));
                if (mt > mr[r]) {
                    const float al = mr[r] == -INFINITY ? 0.f : exp2_approx(mr[r] - mt);
                    mr[r] = mt;
                    l[r] *= al;
                    o[r][0] = mul2(o[r][0], pair(al, al));
                    o[r][1] = mul2(o[r][1], pair(al, al));
                }
            }
        }
#pragma unroll
        for (int r = 0; r < RB; r++) {
            const float base = mr[r] == -INFINITY ? 0.f : mr[r];
            acc[0][r] = exp2_approx(acc[0][r] - base);   // (0 for a masked key)
            acc[1][r] = exp2_approx(acc[1][r] - base);
            if (part == 0) l[r] += acc[0][r] + acc[1][r];
        }
        if (part < 2)   // one of the lanes of a key stores its first, one its second weights
#pragma unroll
            for (int r = 0; r < RB; r += 2) {
                const float a = part ? acc[1][r] : acc[0][r], b = part ? acc[1][r + 1] : acc[0][r + 1];
                *reinterpret_cast<float4 *>(&sh.p[warp][j + part * Sm::kAtOnce][r]) = make_float4(a, a, b, b);
            }
        cp_async_wait<1>();   // V is in
        __syncwarp();
        auto weigh = [&](int jj, const ulonglong2 &v, uint32_t vj) {
#pragma unroll
            for (int r = 0; r < RB; r += 2) {
                const ulonglong2 w = *reinterpret_cast<const ulonglong2 *>(&sh.p[warp][jj][r]);
                if ((vj >> r) & 1u) {
                    o[r][0] = fma2(w.x, v.x, o[r][0]);
                    o[r][1] = fma2(w.x, v.y, o[r][1]);
                }
                if ((vj >> (r + 1)) & 1u) {
                    o[r + 1][0] = fma2(w.y, v.x, o[r + 1][0]);
                    o[r + 1][1] = fma2(w.y, v.y, o[r + 1][1]);
                }
            }
        };
        add_values<HD, Sm::kKeys, RB>(o, tl.v, vis, sub, d4, weigh);
        __syncwarp();
        fetch(t + step, true);
    }
    cp_async_wait<0>();
    __syncthreads();   // every tile is done with: the sums take their memory
#pragma unroll
    for (int r = 0; r < RB; r++) {
        float4 v;
        unpair(o[r][0], v.x, v.y);
        unpair(o[r][1], v.z, v.w);
        if (kPvKeys == 2) {
            v.x += __shfl_xor_sync(0xffffffffu, v.x, 16);
            v.y += __shfl_xor_sync(0xffffffffu, v.y, 16);
            v.z += __shfl_xor_sync(0xffffffffu, v.z, 16);
            v.w += __shfl_xor_sync(0xffffffffu, v.w, 16);
        }
        const float lt = warp_sum(l[r]);
        if (sub == 0) *reinterpret_cast<float4 *>(&sh.sums[warp][r][d4]) = v;
        if (lane == 0) {
            sh.wm[warp][r] = mr[r];
            sh.wl[warp][r] = lt;
        }
    }
    __syncthreads();
    static_assert(kAfWarps * RB <= kAfThreads, "a thread per (warp, row)");
    if (threadIdx.x < kAfWarps * RB) {   // the warps' weights; a warp that saw no key of a row has sums of 0
        const int w = threadIdx.x / RB, r = threadIdx.x % RB;
        float gm = -INFINITY;
#pragma unroll
        for (int x = 0; x < kAfWarps; x++) gm = fmaxf(gm, sh.wm[x][r]);
        sh.wf[w][r] = sh.wm[w][r] == -INFINITY ? 0.f : exp2_approx(sh.wm[w][r] - gm);
        if (w == 0) sh.mx[r] = gm;
    }
    __syncthreads();
    merge_store<HD, RB, kAfThreads>(
        sh.merge,
        [&](int r, int d) {   // in warp order
            float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kAfWarps; w++) {
                const float f = sh.wf[w][r];
                const float4 v = *reinterpret_cast<const float4 *>(&sh.sums[w][r][d]);
                a = make_float4(fmaf(f, v.x, a.x), fmaf(f, v.y, a.y), fmaf(f, v.z, a.z), fmaf(f, v.w, a.w));
            }
            return a;
        },
        [&](int r) {
            float gl = 0.f;
#pragma unroll
            for (int w = 0; w < kAfWarps; w++) gl = fmaf(sh.wf[w][r], sh.wl[w][r], gl);
            return make_float2(sh.mx[r], gl);
        },
        p, s, head0, m0, M, z, Z);
}

// ---------------------------------------------------------------------------
// Many rows: 64 packed rows, 8 per warp.
//
// Bound by the fp32 pipes: 4 * HD flops per (packed row, key).  The 8 warps
// share a tile of 64 keys, the next one under way: a lane has two keys against
// its warp's 8 rows for the scores and 4 dims of the 8 rows for P.V, two
// multiply-adds an instruction, so that shared memory (a K chunk and 8 query
// chunks for 32 pairs of multiply-adds) and the FMA pipes are about equally
// busy; the probabilities stay within the warp.
// ---------------------------------------------------------------------------

constexpr int kArManyRows = 64;
constexpr int kArManyWarps = 8;
constexpr int kArManyThreads = kArManyWarps * 32;
constexpr int kArWarpRows = kArManyRows / kArManyWarps;
constexpr int kArManyKeys = 64;

template <int HD>
struct ArManySmem {
    static constexpr int kRow = HD * 4 + 16;   // a K row: lanes read one chunk of different keys without conflicts
    struct Tile {
        unsigned char k[kArManyKeys * kRow];
        unsigned char v[kArManyKeys * HD * 4];
    };
    union {
        Tile tile[2];
        float sums[kArManyRows][HD];           // at the end
    };
    float q[kArManyRows * HD];
    float p[kArManyWarps][kArManyKeys][kArWarpRows];
    float mx[kArManyRows], sum[kArManyRows];
    ArRows<kArManyRows> rows;
};

constexpr size_t many_smem(int hd, int ctas) {
    return hd == 64 ? sizeof(ArManySmem<64>) + (ctas == 1 ? sizeof(ArMerge<64, kArManyRows>) : 0)
                    : sizeof(ArManySmem<128>) + sizeof(ArMerge<128, kArManyRows>);
}
// A round of two CTAs on an SM, of one alone: the launch takes them where more
// tiles than SMs would run in turn (64-dim heads, trees of 61 rows over short
// contexts, 512 tiles: 94 -> 35 us; 1605 tiles of up to 730 keys 392 -> 360,
// 468 of 70 65 -> 51; near the rule's edge up to a tenth is lost, 210 tiles of
// 800 keys 85 -> 96; what fits one wave is faster alone, 14.5 against 16.5 us).
constexpr double kArTwo = 1.8;

// CTAS: on an SM.  Two fit with heads of 64, in 128 registers each and one
// share: the merge's memory is then q's and p's, which no peer writes early.
template <int HD, int CTAS>
__global__ void __launch_bounds__(kArManyThreads, CTAS) attn_rows_many_kernel(const RowsAttnParams p) {
    using Sm = ArManySmem<HD>;
    constexpr int RB = kArManyRows, WR = kArWarpRows, kKeys = kArManyKeys;
    constexpr bool kOver = CTAS > 1;
    static_assert(many_smem(HD, CTAS) <= (228 / CTAS - 1) * 1024, "they fit an SM");
    extern __shared__ __align__(128) unsigned char smem_raw[];
    Sm &sh = *reinterpret_cast<Sm *>(smem_raw);
    static_assert(!kOver || sizeof(ArMerge<HD, RB>) <= sizeof(sh.q) + sizeof(sh.p), "it fits there");
    ArMerge<HD, RB> &merge = *reinterpret_cast<ArMerge<HD, RB> *>(kOver ? reinterpret_cast<unsigned char *>(sh.q) : smem_raw + sizeof(Sm));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int Z = kOver ? 1 : p.shares, z = blockIdx.x % Z;
    const int m0 = blockIdx.x / Z * RB, kvh = blockIdx.y, stream = blockIdx.z;
    const RowSpan s = row_span(p.r, stream);
    const int M = s.n * p.group;
    if (m0 >= M) return;   // the whole cluster leaves
    const bool tree = p.r.parent != nullptr;
    const int i0 = m0 / p.group, i1 = (min(m0 + RB, M) - 1) / p.group + 1;
    const KeyRange kr = key_range(p.c, s, i0, i1, p.window, tree);
    const int lo_slot = cache_slot(p.c, kr.lo);
    const int total = kr.total(), tiles = (total + kKeys - 1) / kKeys;
    const int t0 = (int)((long long)z * tiles / Z), t1 = (int)((long long)(z + 1) * tiles / Z);
    const long long base = p.layer_off + (long long)stream * p.c.stream_stride + (long long)kvh * p.c.head_stride;
    const char *kb = p.c.k + base * 4, *vb = p.c.v + base * 4;
    const long long slot_bytes = p.c.slot_stride * 4;
    const int head0 = kvh * p.group;

    constexpr int kCh = HD / 4, kRowsAtOnce = kArManyThreads / kCh, kIts = kKeys / kRowsAtOnce;
    const int ch = threadIdx.x % kCh, jr = threadIdx.x / kCh;
    auto fetch = [&](int t, int buf) {
        const int idx0 = t * kKeys;
        const uint32_t kd = smem_u32(sh.tile[buf].k) + jr * Sm::kRow + ch * 16;
        const uint32_t vd = smem_u32(sh.tile[buf].v) + jr * (HD * 4) + ch * 16;
        int slot0 = lo_slot + (idx0 - kr.ns);   // of index idx0, past the sinks
        if (slot0 >= p.c.cap) slot0 -= p.c.ring;
        if (idx0 >= kr.ns && idx0 + kKeys <= total && slot0 + kKeys <= p.c.cap) {
            long long off = (slot0 + jr) * slot_bytes + ch * 16;
#pragma unroll
            for (int it = 0; it < kIts; it++, off += kRowsAtOnce * slot_bytes) {
                cp_async16(kd + it * kRowsAtOnce * Sm::kRow, kb + off, true);
                cp_async16(vd + it * kRowsAtOnce * (HD * 4), vb + off, true);
            }
        } else {
#pragma unroll 1
            for (int it = 0; it < kIts; it++) {
                const int idx = idx0 + it * kRowsAtOnce + jr;
                int slot = idx;
                if (idx >= kr.ns) {
                    slot = lo_slot + (idx - kr.ns);
                    if (slot >= p.c.cap) slot -= p.c.ring;
                }
                const bool ok = idx < total;
                const long long off = ok ? slot * slot_bytes + ch * 16 : 0;
                cp_async16(kd + it * kRowsAtOnce * Sm::kRow, kb + off, ok);
                cp_async16(vd + it * kRowsAtOnce * (HD * 4), vb + off, ok);
            }
        }
    };
    peers_arrive(Z);
    if (t0 < t1) fetch(t0, 0);
    cp_async_commit();
    load_queries<HD, RB>(sh.q, HD, 1, p, s, head0, m0, M);
    setup_rows<RB>(sh.rows, p, s, m0, M);

    const int up_min = tree ? s.pos - 1 : s.pos + i0;
    int core_s = kr.ns + (p.window > 0 ? max(0, min(s.pos + i1 - p.window - kr.lo, kr.nm)) : 0);
    int core_e = kr.ns + max(0, min(up_min - kr.lo + 1, kr.nm));
    if (up_min < kr.ns - 1) core_e = 0;
    else if (core_s == kr.ns) core_s = 0;

    constexpr int kLanesPerKey = HD / 4, kPvKeys = 32 / kLanesPerKey;
    const int sub = lane / kLanesPerKey, d4 = lane % kLanesPerKey * 4;
    float mr[WR], l[WR];   // l: this lane's keys only
    uint64_t o[WR][2];     // pairs of dims
#pragma unroll
    for (int r = 0; r < WR; r++) {
        mr[r] = -INFINITY;
        l[r] = 0.f;
        o[r][0] = o[r][1] = 0;
    }
    const float *qw = sh.q + warp * WR * HD;
    const bool idle = m0 + warp * WR >= M;   // none of the warp's rows exist

    for (int t = t0; t < t1; t++) {
        const int buf = (t - t0) & 1;
        cp_async_wait<0>();
        __syncthreads();   // tile t is in; every warp is done with tile t - 1
        if (t + 1 < t1) fetch(t + 1, buf ^ 1);
        cp_async_commit();
        if (idle) continue;
        const typename Sm::Tile &tl = sh.tile[buf];

        uint64_t a2[2][WR];
#pragma unroll
        for (int r = 0; r < WR; r++) a2[0][r] = a2[1][r] = 0;
#pragma unroll 4
        for (int c = 0; c < HD / 4; c++) {
            const ulonglong2 k0 = *reinterpret_cast<const ulonglong2 *>(tl.k + lane * Sm::kRow + c * 16);
            const ulonglong2 k1 = *reinterpret_cast<const ulonglong2 *>(tl.k + (lane + 32) * Sm::kRow + c * 16);
#pragma unroll
            for (int r = 0; r < WR; r++) {
                const ulonglong2 q = *reinterpret_cast<const ulonglong2 *>(qw + r * HD + c * 4);
                a2[0][r] = fma2(q.x, k0.x, a2[0][r]);
                a2[1][r] = fma2(q.x, k1.x, a2[1][r]);
                a2[0][r] = fma2(q.y, k0.y, a2[0][r]);
                a2[1][r] = fma2(q.y, k1.y, a2[1][r]);
            }
        }
        float acc[2][WR];
#pragma unroll
        for (int x = 0; x < 2; x++)
#pragma unroll
            for (int r = 0; r < WR; r++) {
                float a, b;
                unpair(a2[x][r], a, b);
                acc[x][r] = a + b;
            }
        uint32_t vis[2] = {(1u << WR) - 1u, (1u << WR) - 1u};
        if (!(t * kKeys >= core_s && (t + 1) * kKeys <= core_e)) {
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const int idx = t * kKeys + lane + 32 * x, at = kr.position(idx);
                vis[x] = 0;
                if (idx < total)
#pragma unroll
                    for (int r = 0; r < WR; r++)
                        if (row_sees<RB>(sh.rows, warp * WR + r, at, s.pos, p.c.n_sink, tree)) vis[x] |= 1u << r;
#pragma unroll
                for (int r = 0; r < WR; r++)
                    if (!((vis[x] >> r) & 1u)) acc[x][r] = -INFINITY;
            }
        }
        bool move = false;
#pragma unroll
        for (int r = 0; r < WR; r++) {
            const float a = fmaxf(acc[0][r], acc[1][r]);
            move |= mr[r] == -INFINITY ? a > -INFINITY : a > mr[r] + kAfRescale;
        }
        if (__any_sync(0xffffffffu, move)) {
#pragma unroll
            for (int r = 0; r < WR; r++) {
                float mt = fmaxf(acc[0][r], acc[1][r]);
#pragma unroll
                for (int d = 16; d > 0; d >>= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, d));
                if (mt > mr[r]) {
                    const float al = mr[r] == -INFINITY ? 0.f : exp2_approx(mr[r] - mt);
                    mr[r] = mt;
                    l[r] *= al;
                    o[r][0] = mul2(o[r][0], pair(al, al));
                    o[r][1] = mul2(o[r][1], pair(al, al));
                }
            }
        }
#pragma unroll
        for (int r = 0; r < WR; r++) {
            const float b = mr[r] == -INFINITY ? 0.f : mr[r];
            acc[0][r] = exp2_approx(acc[0][r] - b);   // (0 for a masked key)
            acc[1][r] = exp2_approx(acc[1][r] - b);
            l[r] += acc[0][r] + acc[1][r];
        }
#pragma unroll
        for (int x = 0; x < 2; x++)
#pragma unroll
            for (int r = 0; r < WR; r += 4)
                *reinterpret_cast<float4 *>(&sh.p[warp][lane + 32 * x][r]) =
                    make_float4(acc[x][r], acc[x][r + 1], acc[x][r + 2], acc[x][r + 3]);
        __syncwarp();
        auto weigh = [&](int jj, const ulonglong2 &v, uint32_t vj) {
            float w[WR];
#pragma unroll
            for (int r = 0; r < WR; r += 4)
                *reinterpret_cast<float4 *>(w + r) = *reinterpret_cast<const float4 *>(&sh.p[warp][jj][r]);
#pragma unroll
            for (int r = 0; r < WR; r++)
                if ((vj >> r) & 1u) {
                    o[r][0] = fma2(pair(w[r], w[r]), v.x, o[r][0]);
                    o[r][1] = fma2(pair(w[r], w[r]), v.y, o[r][1]);
                }
        };
        add_values<HD, kKeys, WR>(o, tl.v, vis, sub, d4, weigh);
        __syncwarp();
    }
    cp_async_wait<0>();
    __syncthreads();   // the tiles are done with: their memory takes the sums
#pragma unroll
    for (int r = 0; r < WR; r++) {
        float4 v;
        unpair(o[r][0], v.x, v.y);
        unpair(o[r][1], v.z, v.w);
        if (kPvKeys == 2) {
            v.x += __shfl_xor_sync(0xffffffffu, v.x, 16);
            v.y += __shfl_xor_sync(0xffffffffu, v.y, 16);
            v.z += __shfl_xor_sync(0xffffffffu, v.z, 16);
            v.w += __shfl_xor_sync(0xffffffffu, v.w, 16);
        }
        const float lt = warp_sum(l[r]);
        if (sub == 0) *reinterpret_cast<float4 *>(&sh.sums[warp * WR + r][d4]) = v;
        if (lane == 0) {
            sh.mx[warp * WR + r] = mr[r];
            sh.sum[warp * WR + r] = lt;
        }
    }
    __syncthreads();
    merge_store<HD, RB, kArManyThreads>(
        merge, [&](int r, int d) { return *reinterpret_cast<const float4 *>(&sh.sums[r][d]); },
        [&](int r) { return make_float2(sh.mx[r], sh.sum[r]); }, p, s, head0, m0, M, z, Z);
}

// How one kernel would run a call: its cluster size and what that costs.
struct Plan {
    double cost = 1e30;
    int shares = 0;
};

// rb: packed rows of a tile, round: keys that a CTA takes at once.  Key shares
// of a tile, each a CTA of its cluster: the fewest rounds until the last wave of
// clusters is done, with kArFixed for a CTA's start and merge.  each: a round's
// time, of that of a CTA alone on its SM.
template <typename K>
cudaError_t plan(ClusterKernel &ck, K kernel, size_t smem, int threads, int rb, int round, double each, int most_shares,
                 const RowsAttnParams &p, Plan *out) {
    int dev = 0;
    cudaError_t e = cluster_prepare(ck, kernel, smem, &dev);
    if (e != cudaSuccess) return e;
    const long long M = (long long)p.r.max_rows * p.group, tiles = (M + rb - 1) / rb;
    const long long clusters = tiles * p.c.n_kv_heads * p.c.n_streams;
    const double rounds = (double)most_keys(p, rb) / round;
    for (int Z = 1; Z <= most_shares && (Z == 1 || Z < rounds + 1); Z++) {
        int at_once = 0;
        if ((e = cluster_active(ck, kernel, dev, threads, smem, Z, &at_once)) != cudaSuccess) return e;
        if (at_once < 1) continue;
        const double t = (double)((clusters + at_once - 1) / at_once) * (std::max(1.0, rounds / Z) * each + kArFixed);
        if (t < out->cost) {
            out->cost = t;
            out->shares = Z;
        }
    }
    return out->shares ? cudaSuccess : cudaErrorInvalidConfiguration;
}

template <typename K>
cudaError_t launch(K kernel, size_t smem, int threads, int rb, int ctas, int shares, RowsAttnParams p, cudaStream_t st,
                   RowsPlan *only) {
    if (only) {
        *only = {rb, ctas, shares};
        return cudaSuccess;
    }
    const long long M = (long long)p.r.max_rows * p.group, tiles = (M + rb - 1) / rb;
    p.shares = shares;
    cudaLaunchAttribute a;
    const cudaLaunchConfig_t cfg = cluster_config(dim3((unsigned)(shares * tiles), p.c.n_kv_heads, p.c.n_streams), threads, smem,
                                                  shares, &a, st);
    return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <int HD, int RB>
cudaError_t plan_few(const RowsAttnParams &p, Plan *large, Plan *small) {
    using Large = AfSmem<HD, RB, false>;
    using Small = AfSmem<HD, RB, true>;
    static ClusterKernel cl, cs;
    const cudaError_t e = plan(cl, attn_rows_few_kernel<HD, RB, false>, sizeof(Large), Large::kThreads, RB,
                               Large::kKeys * Large::kWarps, 1.0, kMaxCluster, p, large);
    if (e != cudaSuccess) return e;
    return plan(cs, attn_rows_few_kernel<HD, RB, true>, sizeof(Small), Small::kThreads, RB, Small::kKeys * Small::kWarps, 1.0,
                kMaxCluster, p, small);
}
template <int HD, int RB>
cudaError_t launch_few(const Plan &large, const Plan &small, const RowsAttnParams &p, cudaStream_t st, RowsPlan *only) {
    using Large = AfSmem<HD, RB, false>;
    using Small = AfSmem<HD, RB, true>;
    return small.cost < large.cost
               ? launch(attn_rows_few_kernel<HD, RB, true>, sizeof(Small), Small::kThreads, RB, 4, small.shares, p, st, only)
               : launch(attn_rows_few_kernel<HD, RB, false>, sizeof(Large), Large::kThreads, RB, 1, large.shares, p, st, only);
}

// Microseconds of a round, heads of 128: of the few-row kernels (HBM and the
// loads' latency), and of the many-row one with up to 4 of its warps at work -
// one to a scheduler - and with all 8.  Tiles of 8 rows each take their own pass
// over the keys but spread over more SMs; measured, few against many (32 / 8
// heads): one stream, 4096 keys, 40 packed rows 42 / 62 us, 64 rows 54 / 64;
// 8 streams, 512 keys, 24 rows 37 / 33, 40 rows 55 / 47; 4096 keys, 64 rows
// 361 / 266.
constexpr double kArFewRound = 4.2, kArManyRound4 = 4.9, kArManyRound8 = 7.8;

template <int HD>
cudaError_t launch_dim(const RowsAttnParams &p, cudaStream_t st, RowsPlan *only) {
    const long long M = (long long)p.r.max_rows * p.group;
    Plan large, small, many, two;
    cudaError_t e = M <= 4 ? plan_few<HD, 4>(p, &large, &small) : plan_few<HD, 8>(p, &large, &small);
    if (e != cudaSuccess) return e;
    if (M <= 4) return launch_few<HD, 4>(large, small, p, st, only);
    constexpr size_t kSmem = many_smem(HD, 1);
    static ClusterKernel ck;
    e = plan(ck, attn_rows_many_kernel<HD, 1>, kSmem, kArManyThreads, kArManyRows, kArManyKeys, 1.0, kMaxCluster, p, &many);
    if (e != cudaSuccess) return e;
    if constexpr (HD == 64) {
        static ClusterKernel ck2;
        e = plan(ck2, attn_rows_many_kernel<HD, 2>, many_smem(HD, 2), kArManyThreads, kArManyRows, kArManyKeys, kArTwo, 1, p, &two);
        if (e != cudaSuccess) return e;
    }
    const double round = (M <= 4 * kArWarpRows ? kArManyRound4 : kArManyRound8) * HD / 128;
    if (std::min(large.cost, small.cost) * kArFewRound < std::min(many.cost, two.cost) * round)
        return launch_few<HD, 8>(large, small, p, st, only);
    if constexpr (HD == 64)
        if (two.cost < many.cost)
            return launch(attn_rows_many_kernel<HD, 2>, many_smem(HD, 2), kArManyThreads, kArManyRows, 2, 1, p, st, only);
    return launch(attn_rows_many_kernel<HD, 1>, kSmem, kArManyThreads, kArManyRows, 1, many.shares, p, st, only);
}

}  // namespace

cudaError_t launch_attn_rows(const RowsAttnParams &p, cudaStream_t st, RowsPlan *only) {
    if (p.c.dtype != ELEM_F32) return launch_attn_rows_tc(p, st, only);
    return p.c.head_dim == 64 ? launch_dim<64>(p, st, only) : launch_dim<128>(p, st, only);
}

}  // namespace vc
