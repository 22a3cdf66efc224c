// vc_rows.cuh - what the row operators share (rotary append, window and tree
// attention, cache commit and fork): the cache slab, the rows of a call, and
// which keys a row sees.
//
// Position j of a stream lives in slot j while j < n_sink (kept for good) and
// in slot n_sink + (j - n_sink) mod ring beyond, ring = cap - n_sink; with
// n_sink = 0 this is the decoder's ring.
//
// A stream's rows i = 0 .. n-1 are stored at positions pos + i.  Row i stands
// at the logical position p = pos + i, or pos + depth(i) in a tree.  It sees
// the stored keys j with
//   j <= up:  j < n_sink or j >= low             (low = p - window + 1)
//   j >  up:  bit (j - pos) of the row's ancestor mask (trees only)
// where up = p, or pos - 1 in a tree, among those that the ring still holds.
#pragma once

#include "vc_common.cuh"
#include "vc_internal.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <limits.h>

namespace vc {

__device__ __forceinline__ int cache_slot(const CacheView &c, int j) {
    return j < c.n_sink ? j : c.n_sink + (j - c.n_sink) % c.ring;
}

// element offset of (stream, slot 0, head 0) in one layer
__device__ __forceinline__ long long cache_base(const CacheView &c, int layer, int stream) {
    return (long long)layer * c.layer_stride + (long long)stream * c.stream_stride;
}

struct RowSpan {
    int r0;     // the stream's first row
    int n;      // its rows; 0: none, or the stream sits out
    int pos;    // storage and logical position of row 0
};

// The stream's rows, clamped to what the caller declared: whatever the device
// arrays hold, no row outside [0, n_rows) and no more than max_rows of them.
__device__ __forceinline__ RowSpan row_span(const RowsView &r, int stream) {
    RowSpan s;
    s.pos = __ldg(r.pos + stream);
    int a = stream, b = stream + 1;
    if (r.start) {
        a = __ldg(r.start + stream);
        b = __ldg(r.start + stream + 1);
    }
    s.r0 = min(max(a, 0), r.n_rows);
    s.n = min(min(b, r.n_rows) - s.r0, r.max_rows);
    if (s.n < 0 || s.pos < 0 || s.pos > kMaxPosition) s.n = 0;
    return s;
}

// The keys of rows [i0, i1) of a stream, in the order the kernels walk them:
// positions [0, ns), then [lo, lo + nm).
struct KeyRange {
    int ns, lo, nm;
    __device__ int total() const { return ns + nm; }
    __device__ int position(int idx) const { return idx < ns ? idx : lo + (idx - ns); }
};

__device__ __forceinline__ KeyRange key_range(const CacheView &c, const RowSpan &s, int i0, int i1, int window,
                                              bool tree) {
    KeyRange k;
    const int hi = s.pos + i1;
    const int held = max(c.n_sink, s.pos + s.n - c.ring);
    const int first = s.pos + (tree ? 0 : i0);   // a tree's depths start at 0
    k.lo = window > 0 ? max(held, first - window + 1) : held;
    k.ns = min(c.n_sink, hi);
    k.nm = max(0, hi - k.lo);
    return k;
}

// A stream's parents in shared memory: a parent that is not an earlier row of
// the stream counts as none, so every walk ends.
__device__ __forceinline__ void load_parents(short *dst, const RowsView &r, const RowSpan &s, int tid, int nt) {
    for (int i = tid; i < s.n; i += nt) {
        const int p = __ldg(r.parent + s.r0 + i);
        dst[i] = (short)(p >= 0 && p < i ? p : -1);
    }
}

// Row i's ancestors and itself as bits, its depth as the result.
__device__ __forceinline__ int ancestor_bits(uint32_t *bits, const short *parent, int i) {
    int depth = -1;
    for (int a = i; a >= 0; a = parent[a]) {
        bits[a >> 5] |= 1u << (a & 31);
        depth++;
    }
    return depth;
}

// Drops the ancestors that the window leaves out: those more than window - 1
// levels above row i, unless they stand among the first n_sink positions.
__device__ __forceinline__ void window_bits(uint32_t *bits, const short *parent, int i, int depth, int pos, int n_sink,
                                            int window) {
    if (window <= 0) return;
    int d = depth;
    for (int a = i; a >= 0; a = parent[a], d--)
        if (d <= depth - window && pos + d >= n_sink) bits[a >> 5] &= ~(1u << (a & 31));
}

// Two fp32 values as a pair of T, each rounded to nearest even.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t u);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t u) {
    return make_float2(bf16lo(u), bf16hi(u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t u) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&u));
}

// 4 consecutive elements of T, at a multiple of 4 elements, as fp32.
template <typename T>
__device__ __forceinline__ float4 load4(const T *p) {
    const uint2 u = *reinterpret_cast<const uint2 *>(p);
    const float2 a = unpack2<T>(u.x), b = unpack2<T>(u.y);
    return make_float4(a.x, a.y, b.x, b.y);
}
template <>
__device__ __forceinline__ float4 load4<float>(const float *p) {
    return *reinterpret_cast<const float4 *>(p);
}
template <typename T>
__device__ __forceinline__ void store4(T *p, float4 v) {
    *reinterpret_cast<uint2 *>(p) = make_uint2(pack2<T>(v.x, v.y), pack2<T>(v.z, v.w));
}
template <>
__device__ __forceinline__ void store4<float>(float *p, float4 v) {
    *reinterpret_cast<float4 *>(p) = v;
}

// 16 bytes from global to shared memory, or zeros (ok = false: nothing is read)
__device__ __forceinline__ void cp_async16(uint32_t dst_smem, const void *src, bool ok) {
    const int n = ok ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst_smem), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two fp32 values per register pair: one issue slot for two results.
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t p, float &a, float &b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float fmax_nan(float a, float b) {   // NaN if either is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

}  // namespace vc
