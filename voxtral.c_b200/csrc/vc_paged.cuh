// vc_paged.cuh - what the operators over a paged cache in 8 bits share: pages,
// rows, conversions to and from e4m3.
//
// Position j of a stream lives in slot j mod P of page table[stream][j / P], P a
// power of two; a number is its e4m3 value times the scale of its page and head.
#pragma once

#include "vc_rows.cuh"

#include <cuda_fp8.h>

namespace vc {

// The stream's page at index i, or -1: none, or a number that is no page.
__device__ __forceinline__ int page_at(const PagedView &c, int stream, int i) {
    const int g = __ldg(c.table + (long long)stream * c.table_stride + i);
    return g >= 0 && g < c.n_pages ? g : -1;
}
// Byte offset of (layer, page, head), slot 0, and the index of its scale.
__device__ __forceinline__ long long page_base(const PagedView &c, int layer, int page, int head) {
    return (long long)layer * c.layer_stride + (long long)page * c.page_stride + (long long)head * c.head_stride;
}
__device__ __forceinline__ long long scale_at(const PagedView &c, int layer, int page, int head) {
    return ((long long)layer * c.n_pages + page) * c.n_kv_heads + head;
}

// The stream's rows as row_span tells them, those past the table left out.
__device__ __forceinline__ RowSpan paged_span(const RowsView &r, const PagedView &c, int stream) {
    RowSpan s = row_span(r, stream);
    s.n = max(0, min(s.n, c.table_stride * c.page - s.pos));
    return s;
}

// Four fp32 values as e4m3, rounded to nearest even; NaN stays NaN, larger ones
// than 448 become 448.
__device__ __forceinline__ uint32_t to_e4m3x4(float4 v) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v.x, v.y), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v.z, v.w), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
}
// Two e4m3 values as fp16 (exact).
__device__ __forceinline__ __half2 from_e4m3x2(uint32_t two) {
    return __half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3));
}
__device__ __forceinline__ float4 from_e4m3x4(uint32_t four) {
    const float2 a = __half22float2(from_e4m3x2(four & 0xffffu)), b = __half22float2(from_e4m3x2(four >> 16));
    return make_float4(a.x, a.y, b.x, b.y);
}

}  // namespace vc
