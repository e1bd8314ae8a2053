// mf_attn.cuh -- pieces that the attention kernels over a paged cache share.
#pragma once

#include "mf_vec.cuh"

namespace mf {

constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLn2 = 0.693147180559945309f;

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    if constexpr (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <bool BF16>
__device__ __forceinline__ void unpack2(uint32_t v, float& lo, float& hi) {
    if constexpr (BF16) {
        lo = __uint_as_float(v << 16);
        hi = __uint_as_float(v & 0xffff0000u);
    } else {
        f16x2_to_f32x2(v, lo, hi);
    }
}
__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// Four FP8 codes -> two f16x2, exact: codes 0, 1 and codes 2, 3.
template <int DT>
__device__ __forceinline__ void fp8x4_to_f16(uint32_t four, uint32_t& low, uint32_t& high) {
    if constexpr (DT == MF_DT_F8E4M3) {
        asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
            : "=r"(low), "=r"(high)
            : "r"(four));
    } else {
        low = __byte_perm(four, 0u, 0x1404u);
        high = __byte_perm(four, 0u, 0x3424u);
    }
}
// exp2(m_old - m_new) for m_old <= m_new, 1 where both are the same infinity.
__device__ __forceinline__ float rescale(float m_old, float m_new) {
    return m_old == m_new ? 1.0f : exp2_fast(m_old - m_new);
}

__device__ __forceinline__ float rcp_fast(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// A capped score times log2(e), softcap log2(e) tanh(y), of p = 2 log2(e) y.  With e = exp2(p), tanh(y) = 1 - 2 / (1 + e)
// takes one exponential and one reciprocal and has its limits at both ends, but is only good to 2^-22 of 1: a score far
// below the cap would lose bits.  Below y = 0.4 a polynomial in p^2 stands in (tanh(y) / y by minimax of the relative
// error, 1e-7), above, 2^-22 is 5e-7 of tanh(y).  A warp whose scores are all below takes the polynomial alone: 256
// requests ragged to 8192 tokens, E4M3, take 399 us with a cap of 30 and without one (401 with the exponential form
// up to a cap of 64 and tanhf above).
constexpr float kSmallCapped = 1.15415603f;  // 0.4 * 2 log2(e)
__device__ __forceinline__ float cap_small(float p, float softcap) {
    const float v = p * p;
    return p * softcap * __fmaf_rn(__fmaf_rn(__fmaf_rn(v, -4.1202753e-5f, 9.5731476e-4f), v, -0.020017692f), v, 0.49999995f);
}
__device__ __forceinline__ float2 cap_small2(float2 p, float softcap) {
    const float2 v = __fmul2_rn(p, p);
    auto both = [](float x) { return make_float2(x, x); };
    return __fmul2_rn(__fmul2_rn(p, both(softcap)),
                      __ffma2_rn(__ffma2_rn(__ffma2_rn(v, both(-4.1202753e-5f), both(9.5731476e-4f)), v, both(-0.020017692f)), v, both(0.49999995f)));
}
__device__ __forceinline__ float cap_large(float p, float cap) {
    return __fmaf_rn(-2.0f * cap, rcp_fast(1.0f + exp2_fast(p)), cap);
}

// An even cut of `total` into `parts`: part i starts at total * i / parts, in 32 bits (parts are below 2^15).
struct Cut {
    int32_t total, parts, q, rem;
    __device__ __forceinline__ Cut(int32_t total_, int32_t parts_)
        : total(total_), parts(parts_), q(total_ / parts_), rem(total_ % parts_) {}
    __device__ __forceinline__ int32_t start(int32_t i) const { return q * i + rem * i / parts; }
    // the part that x is in, of a cut without empty parts
    __device__ __forceinline__ int32_t part_of(int32_t x) const {
        int32_t i = min(parts - 1, static_cast<int32_t>((static_cast<float>(x) + 0.5f) * static_cast<float>(parts) / static_cast<float>(total)));
        while (start(i) > x) --i;
        while (i + 1 < parts && start(i + 1) <= x) ++i;
        return i;
    }
};

}  // namespace mf
