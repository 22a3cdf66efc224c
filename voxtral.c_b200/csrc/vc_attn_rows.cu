// vc_attn_rows.cu - attention of a call's rows over a cache slab, with a
// sliding window, sinks that stay visible, and trees of drafted rows: the
// CUDA-core kernels.
//
// o = sum_j 2^(s_j - m) v_j / l, s = scale * log2(e) * q.k, over the keys that
// the row sees (vc_rows.cuh), in one pass with a running maximum m and sum l
// in fp32.  A masked key adds nothing, whatever its K and V hold.
//
// A CTA takes a tile of RB query rows of one (stream, KV head) - row i and
// query head g of the group are packed as m = i * group + g, so a KV head's
// keys are read once for its whole group - and a share of the keys that the
// tile sees.  The shares of a tile are the CTAs of one cluster; they merge
// through distributed shared memory, in rank order, so there is no workspace,
// no ticket and no second launch, and a result does not depend on timing.
#include "vc_rows.cuh"
#include "vc_tc.cuh"

#include <algorithm>
#include <atomic>

namespace vc {

using namespace tc;

namespace {

constexpr int kArThreads = 128;       // 4 warps
constexpr int kArTileBytes = 16384;   // K (and V) bytes of a key tile

template <typename T, int HD>
struct ArShape {
    static constexpr int kChunk = 16 / (int)sizeof(T);                   // elements per 16 bytes
    static constexpr int kChunks = HD / kChunk;                          // 16-byte chunks per key
    static constexpr int kKeys = kArTileBytes / (HD * (int)sizeof(T));   // keys per tile
    static constexpr int kPerLane = kKeys / 32;                          // keys per lane
    static constexpr int kLanesPerKey = HD / 4;                          // P.V: 4 dims per lane
    static constexpr int kKeysAtOnce = 32 / kLanesPerKey;                // P.V: keys per warp step
};

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

// The tile's query rows, scaled, into shared memory as fp32 (zeros past M).
template <typename T, int HD, int RB>
__device__ __forceinline__ void load_queries(float *q, const RowsAttnParams &p, const RowSpan &s, int head0, int m0, int M) {
    for (int e = threadIdx.x; e < RB * HD / 4; e += blockDim.x) {
        const int m = e / (HD / 4), d = e % (HD / 4) * 4;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (m0 + m < M) {
            const int i = (m0 + m) / p.group, g = (m0 + m) % p.group;
            v = load4<T>(static_cast<const T *>(p.q) + ((long long)(s.r0 + i) * p.n_heads + head0 + g) * HD + d);
            v.x *= p.scale_log2;
            v.y *= p.scale_log2;
            v.z *= p.scale_log2;
            v.w *= p.scale_log2;
        }
        *reinterpret_cast<float4 *>(q + m * HD + d) = v;
    }
}

// Asynchronous copy of key tile t's K and V rows; rows past `end` become
// zeros.  K rows are chunk-swizzled (chunk c of key j at c ^ (j & 7)), so that
// 32 lanes reading chunk c of 32 keys do not conflict.
template <typename T, int HD>
__device__ __forceinline__ void load_tile(unsigned char *dst, const char *kb, const char *vb, long long slot_bytes,
                                          const KeyRange &kr, int lo_slot, const CacheView &c, int idx0, int end) {
    using S = ArShape<T, HD>;
    const uint32_t k_s = smem_u32(dst), v_s = k_s + kArTileBytes;
#pragma unroll
    for (int it = 0; it < kArTileBytes / 16 / kArThreads; it++) {
        const int e = threadIdx.x + it * kArThreads;
        const int j = e / S::kChunks, ch = e % S::kChunks;
        const int idx = idx0 + j;
        int slot = idx;
        if (idx >= kr.ns) {
            slot = lo_slot + (idx - kr.ns);
            if (slot >= c.cap) slot -= c.ring;
        }
        const bool ok = idx < end;
        const long long off = ok ? slot * slot_bytes + ch * 16 : 0;
        cp_async16(k_s + j * (HD * (int)sizeof(T)) + ((ch ^ (j & 7)) << 4), kb + off, ok);
        cp_async16(v_s + j * (HD * (int)sizeof(T)) + (ch << 4), vb + off, ok);
    }
}

// One 16-byte chunk of a key row in shared memory as fp32.
template <typename T>
struct Chunk {
    float f[8];
    __device__ __forceinline__ explicit Chunk(const unsigned char *p) {
        const uint4 u = *reinterpret_cast<const uint4 *>(p);
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
struct Chunk<float> {
    float f[4];
    __device__ __forceinline__ explicit Chunk(const unsigned char *p) {
        const float4 a = *reinterpret_cast<const float4 *>(p);
        f[0] = a.x;
        f[1] = a.y;
        f[2] = a.z;
        f[3] = a.w;
    }
};

// Merges the cluster's shares of a tile and writes the rows.  Every CTA has
// put its rows' unnormalised sums o [RB][HD], maxima and sums into its own
// shared memory; rank z takes every Z-th group of 4 dims.
template <typename T, int HD, int RB>
__device__ __forceinline__ void merge_store(const float *o, const float *mx, const float *sum, const RowsAttnParams &p,
                                            const RowSpan &s, int head0, int m0, int M, int z, int Z) {
    if (Z > 1) cluster_sync_all();
    else __syncthreads();
    const uint32_t o_s = smem_u32(o), m_s = smem_u32(mx), l_s = smem_u32(sum);
    for (int e = threadIdx.x + z * kArThreads; e < RB * HD / 4; e += Z * kArThreads) {
        const int m = e / (HD / 4), d = e % (HD / 4) * 4;
        if (m0 + m >= M) continue;
        float gm = -INFINITY;
        for (int r = 0; r < Z; r++) gm = fmaxf(gm, ld_dsmem_f1(mapa_shared(m_s + 4 * m, r)));
        float gl = 0.f;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int r = 0; r < Z; r++) {
            const float mr = ld_dsmem_f1(mapa_shared(m_s + 4 * m, r));
            const float w = mr == -INFINITY ? 0.f : exp2_approx(mr - gm);
            const float l = ld_dsmem_f1(mapa_shared(l_s + 4 * m, r));
            const float4 v = ld_dsmem_f4(mapa_shared(o_s + 4 * (m * HD + d), r));
            if (mr == -INFINITY && l == 0.f) continue;   // this share saw no key of the row
            gl = fmaf(w, l, gl);
            a.x = fmaf(w, v.x, a.x);
            a.y = fmaf(w, v.y, a.y);
            a.z = fmaf(w, v.z, a.z);
            a.w = fmaf(w, v.w, a.w);
        }
        const float il = gl == 0.f ? 0.f : 1.0f / gl;   // no key at all: zeros
        const long long row = (long long)(s.r0 + (m0 + m) / p.group) * p.n_heads + head0 + (m0 + m) % p.group;
        store4<T>(static_cast<T *>(p.out) + row * HD + d, make_float4(a.x * il, a.y * il, a.z * il, a.w * il));
        if (p.lse && d == 0) p.lse[row] = gl == 0.f ? -INFINITY : (gm + log2f(gl)) * 0.69314718055994531f;
    }
    if (Z > 1) cluster_sync_all();   // no CTA leaves while a peer still reads its share
}

// ---------------------------------------------------------------------------
// Few rows: RB (4 or 8) packed rows, one token of one KV head's group.
//
// Bound by HBM: a tile is 32 KB of keys and 2 * RB flops per byte.  The four
// warps split a key's dims for the scores (each lane one key or more, so that
// a K chunk is read from shared memory once for all RB rows) and the tile's
// keys for P.V (each lane 4 dims); three tiles are in flight per CTA.
// ---------------------------------------------------------------------------

template <typename T, int HD, int RB>
struct ArFewSmem {
    static constexpr int kKeys = ArShape<T, HD>::kKeys;
    static constexpr int kStages = 3;
    unsigned char kv[kStages][2 * kArTileBytes];
    float q[RB * HD];
    float part[4][RB][kKeys];     // the warps' partial scores
    float p[kKeys][RB];           // 2^(s - m), or -1 for a masked key
    float alpha[RB];              // the rows' rescale factors of this tile
    float mx[RB], sum[RB];
    int masked[4];                // a warp's rows have a masked key in this tile
    ArRows<RB> rows;
};

template <typename T, int HD, int RB>
__global__ void __launch_bounds__(kArThreads) attn_rows_few_kernel(const RowsAttnParams p) {
    using S = ArShape<T, HD>;
    using Sm = ArFewSmem<T, HD, RB>;
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
    const int total = kr.total(), tiles = (total + S::kKeys - 1) / S::kKeys;
    const int t0 = (int)((long long)z * tiles / Z), t1 = (int)((long long)(z + 1) * tiles / Z);
    const long long base = p.layer_off + (long long)stream * p.c.stream_stride + (long long)kvh * p.c.head_stride;
    const char *kb = p.c.k + base * (long long)sizeof(T), *vb = p.c.v + base * (long long)sizeof(T);
    const long long slot_bytes = p.c.slot_stride * (long long)sizeof(T);
    const int head0 = kvh * p.group;

#pragma unroll
    for (int i = 0; i < Sm::kStages - 1; i++) {
        if (t0 + i < t1)
            load_tile<T, HD>(sh.kv[i], kb, vb, slot_bytes, kr, lo_slot, p.c, (t0 + i) * S::kKeys, total);
        cp_async_commit();
    }
    load_queries<T, HD, RB>(sh.q, p, s, head0, m0, M);
    setup_rows<RB>(sh.rows, p, s, m0, M);

    constexpr int kRowsPerWarp = RB / 4;
    float m_run[kRowsPerWarp], l_run[kRowsPerWarp];
#pragma unroll
    for (int r = 0; r < kRowsPerWarp; r++) {
        m_run[r] = -INFINITY;
        l_run[r] = 0.f;
    }
    float4 o[RB];
#pragma unroll
    for (int r = 0; r < RB; r++) o[r] = make_float4(0.f, 0.f, 0.f, 0.f);

    for (int t = t0; t < t1; t++) {
        const int st = (t - t0) % Sm::kStages;
        cp_async_wait<Sm::kStages - 2>();
        __syncthreads();   // tile t is in; every warp is done with tile t - 1
        if (t + Sm::kStages - 1 < t1)
            load_tile<T, HD>(sh.kv[(t - t0 + Sm::kStages - 1) % Sm::kStages], kb, vb, slot_bytes, kr, lo_slot, p.c,
                             (t + Sm::kStages - 1) * S::kKeys, total);
        cp_async_commit();

        // scores of this warp's quarter of the dims
        float acc[RB][S::kPerLane];
#pragma unroll
        for (int r = 0; r < RB; r++)
#pragma unroll
            for (int x = 0; x < S::kPerLane; x++) acc[r][x] = 0.f;
#pragma unroll
        for (int c = 0; c < S::kChunks / 4; c++) {
            const int ch = warp * (S::kChunks / 4) + c;
#pragma unroll
            for (int x = 0; x < S::kPerLane; x++) {
                const int j = lane + 32 * x;
                const Chunk<T> k(sh.kv[st] + j * (HD * (int)sizeof(T)) + ((ch ^ (j & 7)) << 4));
#pragma unroll
                for (int r = 0; r < RB; r++)
#pragma unroll
                    for (int y = 0; y < S::kChunk; y += 4) {
                        const float4 qv = *reinterpret_cast<const float4 *>(sh.q + r * HD + ch * S::kChunk + y);
                        acc[r][x] = fmaf(qv.x, k.f[y], acc[r][x]);
                        acc[r][x] = fmaf(qv.y, k.f[y + 1], acc[r][x]);
                        acc[r][x] = fmaf(qv.z, k.f[y + 2], acc[r][x]);
                        acc[r][x] = fmaf(qv.w, k.f[y + 3], acc[r][x]);
                    }
            }
        }
#pragma unroll
        for (int r = 0; r < RB; r++)
#pragma unroll
            for (int x = 0; x < S::kPerLane; x++) sh.part[warp][r][lane + 32 * x] = acc[r][x];
        __syncthreads();

        // softmax: warp w takes rows w, w + 4
        bool any_masked = false;
#pragma unroll
        for (int rr = 0; rr < kRowsPerWarp; rr++) {
            const int r = warp + 4 * rr;
            float sc[S::kPerLane];
            bool vis[S::kPerLane];
            float mt = -INFINITY;
#pragma unroll
            for (int x = 0; x < S::kPerLane; x++) {
                const int j = lane + 32 * x, idx = t * S::kKeys + j;
                sc[x] = (sh.part[0][r][j] + sh.part[1][r][j]) + (sh.part[2][r][j] + sh.part[3][r][j]);
                vis[x] = idx < total && row_sees<RB>(sh.rows, r, kr.position(idx), s.pos, p.c.n_sink, tree);
                any_masked |= !vis[x];
                if (vis[x]) mt = fmaxf(mt, sc[x]);
            }
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, d));
            const float mn = fmaxf(m_run[rr], mt);
            const float b = mn == -INFINITY ? 0.f : mn;
            const float al = m_run[rr] == -INFINITY ? 0.f : exp2_approx(m_run[rr] - b);
            float ls = 0.f;
#pragma unroll
            for (int x = 0; x < S::kPerLane; x++) {
                const float pv = exp2_approx(sc[x] - b);
                if (vis[x]) ls += pv;
                sh.p[lane + 32 * x][r] = vis[x] ? pv : -1.f;
            }
            l_run[rr] = l_run[rr] * al + warp_sum(ls);
            m_run[rr] = mn;
            if (lane == 0) sh.alpha[r] = al;
        }
        any_masked = __any_sync(0xffffffffu, any_masked);
        if (lane == 0) sh.masked[warp] = any_masked;
        __syncthreads();

        // o = o * alpha + P V over this warp's quarter of the keys
        const unsigned char *vt = sh.kv[st] + kArTileBytes;
        const int sub = lane / S::kLanesPerKey, d4 = lane % S::kLanesPerKey * 4;
#pragma unroll
        for (int r = 0; r < RB; r++) {
            const float al = sh.alpha[r];
            o[r].x *= al;
            o[r].y *= al;
            o[r].z *= al;
            o[r].w *= al;
        }
        const bool masked = (sh.masked[0] | sh.masked[1] | sh.masked[2] | sh.masked[3]) != 0;
#pragma unroll 4
        for (int x = 0; x < S::kKeys / 4 / S::kKeysAtOnce; x++) {
            const int j = warp * (S::kKeys / 4) + x * S::kKeysAtOnce + sub;
            const float4 v = load4<T>(reinterpret_cast<const T *>(vt) + j * HD + d4);
            float pr[RB];
#pragma unroll
            for (int r = 0; r < RB; r += 4)
                *reinterpret_cast<float4 *>(pr + r) = *reinterpret_cast<const float4 *>(&sh.p[j][r]);
#pragma unroll
            for (int r = 0; r < RB; r++) {
                if (masked && pr[r] < 0.f) continue;
                o[r].x = fmaf(pr[r], v.x, o[r].x);
                o[r].y = fmaf(pr[r], v.y, o[r].y);
                o[r].z = fmaf(pr[r], v.z, o[r].z);
                o[r].w = fmaf(pr[r], v.w, o[r].w);
            }
        }
    }
    cp_async_wait<0>();
    __syncthreads();   // the tiles are done with: their memory takes the partial sums

    float *red = reinterpret_cast<float *>(sh.kv[0]);            // [4 warps][RB][HD]
    float *of = reinterpret_cast<float *>(sh.kv[1]);             // [RB][HD]
    static_assert(4 * RB * HD * 4 <= 2 * kArTileBytes, "the warps' partial sums fit a stage");
    {
        const int sub = lane / S::kLanesPerKey, d4 = lane % S::kLanesPerKey * 4;
#pragma unroll
        for (int r = 0; r < RB; r++) {
            float4 v = o[r];
            if (S::kKeysAtOnce == 2) {
                v.x += __shfl_xor_sync(0xffffffffu, v.x, 16);
                v.y += __shfl_xor_sync(0xffffffffu, v.y, 16);
                v.z += __shfl_xor_sync(0xffffffffu, v.z, 16);
                v.w += __shfl_xor_sync(0xffffffffu, v.w, 16);
            }
            if (sub == 0) *reinterpret_cast<float4 *>(red + (warp * RB + r) * HD + d4) = v;
        }
#pragma unroll
        for (int rr = 0; rr < kRowsPerWarp; rr++)
            if (lane == 0) {
                sh.mx[warp + 4 * rr] = m_run[rr];
                sh.sum[warp + 4 * rr] = l_run[rr];
            }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < RB * HD; e += kArThreads)
        of[e] = (red[e] + red[RB * HD + e]) + (red[2 * RB * HD + e] + red[3 * RB * HD + e]);
    merge_store<T, HD, RB>(of, sh.mx, sh.sum, p, s, head0, m0, M, z, Z);
}

// ---------------------------------------------------------------------------
// Many rows: 32 packed rows, 8 per warp.
//
// Bound by the fp32 pipes: 4 * HD flops per (packed row, key).  Every warp
// reads all of a tile's keys for its 8 rows: a lane holds one key or more
// against 8 rows for the scores and 4 dims of 8 rows for P.V, so that a value
// read from shared memory meets 8 multiply-adds; the probabilities stay
// within the warp.
// ---------------------------------------------------------------------------

constexpr int kArManyRows = 32;
constexpr int kArWarpRows = kArManyRows / 4;

template <typename T, int HD>
struct ArManySmem {
    static constexpr int kKeys = ArShape<T, HD>::kKeys;
    static constexpr int kStages = 2;
    unsigned char kv[kStages][2 * kArTileBytes];
    float q[kArManyRows * HD];
    float p[4][kKeys][kArWarpRows];
    float mx[kArManyRows], sum[kArManyRows];
    ArRows<kArManyRows> rows;
};

template <typename T, int HD>
__global__ void __launch_bounds__(kArThreads) attn_rows_many_kernel(const RowsAttnParams p) {
    using S = ArShape<T, HD>;
    using Sm = ArManySmem<T, HD>;
    constexpr int RB = kArManyRows, WR = kArWarpRows;
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
    const int total = kr.total(), tiles = (total + S::kKeys - 1) / S::kKeys;
    const int t0 = (int)((long long)z * tiles / Z), t1 = (int)((long long)(z + 1) * tiles / Z);
    const long long base = p.layer_off + (long long)stream * p.c.stream_stride + (long long)kvh * p.c.head_stride;
    const char *kb = p.c.k + base * (long long)sizeof(T), *vb = p.c.v + base * (long long)sizeof(T);
    const long long slot_bytes = p.c.slot_stride * (long long)sizeof(T);
    const int head0 = kvh * p.group;

    if (t0 < t1) load_tile<T, HD>(sh.kv[0], kb, vb, slot_bytes, kr, lo_slot, p.c, t0 * S::kKeys, total);
    cp_async_commit();
    load_queries<T, HD, RB>(sh.q, p, s, head0, m0, M);
    setup_rows<RB>(sh.rows, p, s, m0, M);

    float m_run[WR], l_run[WR];   // l: this lane's keys only
    float4 o[WR];
#pragma unroll
    for (int r = 0; r < WR; r++) {
        m_run[r] = -INFINITY;
        l_run[r] = 0.f;
        o[r] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    const float *qw = sh.q + warp * WR * HD;
    const bool idle = m0 + warp * WR >= M;   // none of the warp's rows exist

    for (int t = t0; t < t1; t++) {
        const int st = (t - t0) % Sm::kStages;
        cp_async_wait<0>();
        __syncthreads();   // tile t is in; every warp is done with tile t - 1
        if (t + 1 < t1)
            load_tile<T, HD>(sh.kv[st ^ 1], kb, vb, slot_bytes, kr, lo_slot, p.c, (t + 1) * S::kKeys, total);
        cp_async_commit();
        if (idle) continue;

        float acc[WR][S::kPerLane];
#pragma unroll
        for (int r = 0; r < WR; r++)
#pragma unroll
            for (int x = 0; x < S::kPerLane; x++) acc[r][x] = 0.f;
#pragma unroll 2
        for (int ch = 0; ch < S::kChunks; ch++) {
            float k[S::kPerLane][S::kChunk];
#pragma unroll
            for (int x = 0; x < S::kPerLane; x++) {
                const int j = lane + 32 * x;
                const Chunk<T> c(sh.kv[st] + j * (HD * (int)sizeof(T)) + ((ch ^ (j & 7)) << 4));
#pragma unroll
                for (int y = 0; y < S::kChunk; y++) k[x][y] = c.f[y];
            }
#pragma unroll
            for (int r = 0; r < WR; r++)
#pragma unroll
                for (int y = 0; y < S::kChunk; y += 4) {
                    const float4 qv = *reinterpret_cast<const float4 *>(qw + r * HD + ch * S::kChunk + y);
#pragma unroll
                    for (int x = 0; x < S::kPerLane; x++) {
                        acc[r][x] = fmaf(qv.x, k[x][y], acc[r][x]);
                        acc[r][x] = fmaf(qv.y, k[x][y + 1], acc[r][x]);
                        acc[r][x] = fmaf(qv.z, k[x][y + 2], acc[r][x]);
                        acc[r][x] = fmaf(qv.w, k[x][y + 3], acc[r][x]);
                    }
                }
        }

        bool any_masked = false;
#pragma unroll
        for (int r = 0; r < WR; r++) {
            bool vis[S::kPerLane];
            float mt = -INFINITY;
#pragma unroll
            for (int x = 0; x < S::kPerLane; x++) {
                const int idx = t * S::kKeys + lane + 32 * x;
                vis[x] = idx < total &&
                         row_sees<RB>(sh.rows, warp * WR + r, kr.position(idx), s.pos, p.c.n_sink, tree);
                any_masked |= !vis[x];
                if (vis[x]) mt = fmaxf(mt, acc[r][x]);
            }
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, d));
            const float mn = fmaxf(m_run[r], mt);
            const float b = mn == -INFINITY ? 0.f : mn;
            const float al = m_run[r] == -INFINITY ? 0.f : exp2_approx(m_run[r] - b);
            m_run[r] = mn;
            float ls = 0.f;
#pragma unroll
            for (int x = 0; x < S::kPerLane; x++) {
                const float pv = exp2_approx(acc[r][x] - b);
                if (vis[x]) ls += pv;
                acc[r][x] = vis[x] ? pv : -1.f;
            }
            l_run[r] = l_run[r] * al + ls;
            o[r].x *= al;
            o[r].y *= al;
            o[r].z *= al;
            o[r].w *= al;
        }
        any_masked = __any_sync(0xffffffffu, any_masked);
#pragma unroll
        for (int x = 0; x < S::kPerLane; x++)
#pragma unroll
            for (int r = 0; r < WR; r += 4)
                *reinterpret_cast<float4 *>(&sh.p[warp][lane + 32 * x][r]) =
                    make_float4(acc[r][x], acc[r + 1][x], acc[r + 2][x], acc[r + 3][x]);
        __syncwarp();

        const unsigned char *vt = sh.kv[st] + kArTileBytes;
        const int sub = lane / S::kLanesPerKey, d4 = lane % S::kLanesPerKey * 4;
#pragma unroll 4
        for (int x = 0; x < S::kKeys / S::kKeysAtOnce; x++) {
            const int j = x * S::kKeysAtOnce + sub;
            const float4 v = load4<T>(reinterpret_cast<const T *>(vt) + j * HD + d4);
            float pr[WR];
#pragma unroll
            for (int r = 0; r < WR; r += 4)
                *reinterpret_cast<float4 *>(pr + r) = *reinterpret_cast<const float4 *>(&sh.p[warp][j][r]);
#pragma unroll
            for (int r = 0; r < WR; r++) {
                if (any_masked && pr[r] < 0.f) continue;
                o[r].x = fmaf(pr[r], v.x, o[r].x);
                o[r].y = fmaf(pr[r], v.y, o[r].y);
                o[r].z = fmaf(pr[r], v.z, o[r].z);
                o[r].w = fmaf(pr[r], v.w, o[r].w);
            }
        }
        __syncwarp();
    }
    cp_async_wait<0>();
    __syncthreads();   // the tiles are done with: their memory takes the sums

    float *of = reinterpret_cast<float *>(sh.kv[0]);   // [RB][HD]
    static_assert(RB * HD * 4 <= 2 * kArTileBytes, "the sums fit a stage");
    const int sub = lane / S::kLanesPerKey, d4 = lane % S::kLanesPerKey * 4;
#pragma unroll
    for (int r = 0; r < WR; r++) {
        float4 v = o[r];
        if (S::kKeysAtOnce == 2) {
            v.x += __shfl_xor_sync(0xffffffffu, v.x, 16);
            v.y += __shfl_xor_sync(0xffffffffu, v.y, 16);
            v.z += __shfl_xor_sync(0xffffffffu, v.z, 16);
            v.w += __shfl_xor_sync(0xffffffffu, v.w, 16);
        }
        const float l = warp_sum(l_run[r]);
        if (sub == 0) *reinterpret_cast<float4 *>(of + (warp * WR + r) * HD + d4) = v;
        if (lane == 0) {
            sh.mx[warp * WR + r] = m_run[r];
            sh.sum[warp * WR + r] = l;
        }
    }
    merge_store<T, HD, RB>(of, sh.mx, sh.sum, p, s, head0, m0, M, z, Z);
}

// The shared-memory and cluster-size opt-ins of one kernel, once per device.
template <typename K>
cudaError_t prepare_kernel(K kernel, size_t smem, std::atomic<uint64_t> &done) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (done.load() & bit) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess) done.fetch_or(bit);
    return e;
}

template <typename K>
cudaError_t launch_cluster(K kernel, dim3 grid, int Z, size_t smem, const RowsAttnParams &p, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kArThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute a[1];
    a[0].id = cudaLaunchAttributeClusterDimension;
    a[0].val.clusterDim.x = Z;
    a[0].val.clusterDim.y = 1;
    a[0].val.clusterDim.z = 1;
    cfg.attrs = a;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, p);
}

// Key shares of a tile: as many as two CTAs per SM hold, at most one per key
// tile and 16, a cluster's limit.
int shares(long long ctas, long long keys, int tile, int sms) {
    const long long by_sms = std::max<long long>(1, 2ll * sms / ctas), by_keys = (keys + tile - 1) / tile;
    return (int)std::max<long long>(1, std::min<long long>(16, std::min(by_sms, by_keys)));
}

template <typename T, int HD>
cudaError_t launch_typed(const RowsAttnParams &p, int sms, cudaStream_t st) {
    constexpr int kKeys = ArShape<T, HD>::kKeys;
    const long long M = (long long)p.r.max_rows * p.group;
    // most keys that one tile can see
    const long long keys =
        p.window > 0 ? std::min<long long>(p.c.cap, (long long)p.window + p.r.max_rows + p.c.n_sink) : p.c.cap;
    auto go = [&](auto kernel, size_t smem, int rb, std::atomic<uint64_t> &done) {
        cudaError_t e = prepare_kernel(kernel, smem, done);
        if (e != cudaSuccess) return e;
        const long long tiles = (M + rb - 1) / rb;
        RowsAttnParams pp = p;
        pp.shares = shares(tiles * p.c.n_kv_heads * p.c.n_streams, keys, kKeys, sms);
        return launch_cluster(kernel, dim3((unsigned)(pp.shares * tiles), p.c.n_kv_heads, p.c.n_streams), pp.shares, smem,
                              pp, st);
    };
    static std::atomic<uint64_t> d4{0}, d8{0}, d32{0};
    if constexpr (sizeof(T) == 2) return launch_attn_rows_tc(p, sms, st);
    if (M <= 4) return go(attn_rows_few_kernel<T, HD, 4>, sizeof(ArFewSmem<T, HD, 4>), 4, d4);
    if (M <= 8) return go(attn_rows_few_kernel<T, HD, 8>, sizeof(ArFewSmem<T, HD, 8>), 8, d8);
    if constexpr (sizeof(T) == 2) return launch_attn_rows_tc(p, sms, st);
    else return go(attn_rows_many_kernel<T, HD>, sizeof(ArManySmem<T, HD>), kArManyRows, d32);
}

template <typename T>
cudaError_t launch_dim(const RowsAttnParams &p, int sms, cudaStream_t st) {
    return p.c.head_dim == 64 ? launch_typed<T, 64>(p, sms, st) : launch_typed<T, 128>(p, sms, st);
}

}  // namespace

cudaError_t launch_attn_rows(const RowsAttnParams &p, int sms, cudaStream_t st) {
    switch (p.c.dtype) {
        case ELEM_F32: return launch_dim<float>(p, sms, st);
        case ELEM_BF16: return launch_dim<__nv_bfloat16>(p, sms, st);
        default: return launch_dim<__half>(p, sms, st);
    }
}

}  // namespace vc
