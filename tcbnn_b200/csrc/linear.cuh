// Products of real-valued rows: y[m][n] = act(s[n] * sum_k x[m][k] * w[n][k] + b[n]) + r[m][n], x in bf16 or fp16,
// w of the same type (s = 1) or packed signs of +-1 with a scale per output.  Sums, scale, bias, activation and
// residual are fp32; the result is rounded once, to x's type or not at all.  Types, arguments and what happens to a sum.
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace tcbnn {
namespace linear {

enum Type { FP32 = 0, FP16 = 1, BF16 = 2 };
enum Activation { NONE = 0, RELU = 1, GELU = 2, GELU_TANH = 3, SILU = 4 };

struct Args {
    const void* x; const void* W; const float* scale; const void* bias; const void* residual; void* out;
    int M, N, K;
    long long ldx, ldw, ldr, ldo;                      // elements; words for packed weights
    int type, out_type, bias_type, activation;
};

__device__ __forceinline__ float load(const void* p, long long i, int type) {
    if (type == FP32) return reinterpret_cast<const float*>(p)[i];
    if (type == FP16) return __half2float(reinterpret_cast<const __half*>(p)[i]);
    return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void store(void* p, long long i, int type, float v) {
    if (type == FP32) reinterpret_cast<float*>(p)[i] = v;
    else if (type == FP16) reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
    else reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}
// Activations.  The accurate forms are off by a few units in the last place of the result, far out in the negative tail as well (there the
// roundings of an exponent v weigh |v|).  The short forms are for 16-bit results of whole tiles, where their instructions show (fp32 results of
// 1024 x 512 -> 1024 with gelu: 8.1 us, by the short form 7.4): off by about a hundredth of a rounding to 16 bits.
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// z / (1 + e^{-v}) by the exponential of -|v|, which neither overflows nor cancels; a product z e^{-|v|} below the normal numbers is 0
template <bool SHORT>
__device__ __forceinline__ float over_one_plus_exp(float z, float v) {
    const float w = SHORT ? __expf(-fabsf(v)) : expf(-fabsf(v));
    float y;
    asm("div.approx.ftz.f32 %0, %1, %2;" : "=f"(y) : "f"(v < 0.f ? z * w : z), "f"(1.f + w));
    return y;
}
// z Phi(z), where Phi(-|z|) = e^{-z^2 / 2} Q: Q by a polynomial in t = 1 / (1 + k |z|) without constant term, the shape of 7.1.26 of Abramowitz
// and Stegun.  Coefficients and k: least largest relative error of Q over |z| <= 13.6, behind which the product is below the normal
// numbers; 5 units of 2^-24 as fp32 evaluates it, the short one 68.
template <bool SHORT>
__device__ __forceinline__ float gelu(float z) {
    float q;
    if (SHORT) {
        const float t = __fdividef(1.f, fmaf(0.307591438f, fabsf(z), 1.f));
        q = fmaf(fmaf(-0.0757672802f, t, 0.191610958f), t, 0.00538595912f);
        q = t * fmaf(fmaf(fmaf(q, t, 0.13725508f), t, 0.118539558f), t, 0.122974204f) * ex2(-0.721347520f * z * z);
    } else {
        const float t = __fdividef(1.f, fmaf(0.342946798f, fabsf(z), 1.f));
        q = fmaf(fmaf(-0.0270156274f, t, 0.140884452f), t, -0.267972608f);
        q = fmaf(fmaf(fmaf(q, t, 0.188897667f), t, -0.0375840724f), t, 0.112119676f);
        q = t * fmaf(fmaf(fmaf(q, t, 0.116665187f), t, 0.137205251f), t, 0.13680008f) * expf(-0.5f * (z * z));
    }
    return z * (z < 0.f ? q : 1.f - q);
}
template <bool SHORT = false>
__device__ __forceinline__ float activate(float z, int a) {
    if (a == RELU) return z < 0.f ? 0.f : z;           // (NaN stays)
    if (a == GELU) return gelu<SHORT>(z);
    // (the tanh form: 1 + tanh u = 2 / (1 + e^{-2u}))
    if (a == GELU_TANH) return over_one_plus_exp<SHORT>(z, 1.59576912160573071f * (z + 0.044715f * z * z * z));
    if (a == SILU) return over_one_plus_exp<SHORT>(z, z);
    return z;
}

}  // namespace linear
}  // namespace tcbnn
