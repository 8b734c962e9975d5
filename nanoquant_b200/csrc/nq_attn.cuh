// What the kernels between the projections share: 16-bit elements, places in a paged cache, softmax in powers of two.
#pragma once

#include <initializer_list>

#include "nq_common.cuh"

namespace nq {

constexpr int kHeadMaxCols = 256;       // elements of a head

template <bool BF16>
__device__ __forceinline__ float head_float(uint32_t w, int half) {
    if constexpr (BF16) return __uint_as_float(half ? w & 0xffff0000u : w << 16);
    else return __half2float(__ushort_as_half((unsigned short)(half ? w >> 16 : w & 0xffffu)));
}
template <bool BF16>
__device__ __forceinline__ uint32_t head_pack(float lo, float hi) {
    uint32_t r;
    if constexpr (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// 2^x, 2 ulp; 0 for -infinity.
__device__ __forceinline__ float exp2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ uint64_t pair_of(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void pair_split(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t pair_fma(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t pair_add(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t pair_mul(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

inline bool multiple_of_8(std::initializer_list<int64_t> v) {
    for (int64_t x : v)
        if (x & 7) return false;
    return true;
}
inline bool page_size_ok(int n) { return n >= 8 && (n & (n - 1)) == 0; }
inline int log2_of(int n) {
    int r = 0;
    while ((1 << r) < n) ++r;
    return r;
}

}  // namespace nq
