// vc_attn_tc.cuh - what the tensor-core attention kernels share: operand
// descriptors, a warp's MMA instructions, TMEM loads and stores, 2^x on the FMA
// pipe.
#pragma once

#include "vc_rows.cuh"
#include "vc_tc.cuh"

#include <math.h>
#include <type_traits>

namespace vc {
namespace tc {

constexpr int kAtRows = 128;            // packed rows per MMA tile = TMEM lanes

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

}  // namespace tc
}  // namespace vc
