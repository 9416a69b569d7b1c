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
// z / (1 + e^{-z}); the exponential and the division are off by a few 2^-22 of the result, and e^{-z} by |z| 2^-23 more, which counts
// where it is not small against 1: 2^-21 |z| in all.
__device__ __forceinline__ float over_one_plus_exp(float z, float minus_u) { return __fdividef(z, 1.f + __expf(minus_u)); }
// z Phi(z) by the polynomial 7.1.26 of Abramowitz and Stegun for erfc on x = |z| / sqrt 2, off by at most 1.5e-7: no cancellation for
// negative z, and a third of the instructions of 0.5 z (1 + erff(x)).
__device__ __forceinline__ float gelu(float z) {
    const float x = fabsf(z) * 0.70710678118654752f, t = __fdividef(1.f, fmaf(0.3275911f, x, 1.f));
    const float poly = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f), 0.254829592f);
    const float half = 0.5f * poly * __expf(-x * x);                     // half of erfc(x): Phi(-|z|)
    return z * (z < 0.f ? half : 1.f - half);
}
__device__ __forceinline__ float activate(float z, int a) {
    if (a == RELU) return z < 0.f ? 0.f : z;           // (NaN stays)
    if (a == GELU) return gelu(z);
    // (the tanh form: 1 + tanh u = 2 / (1 + e^{-2u}))
    if (a == GELU_TANH) return over_one_plus_exp(z, -1.59576912160573071f * (z + 0.044715f * z * z * z));
    if (a == SILU) return over_one_plus_exp(z, -z);
    return z;
}

}  // namespace linear
}  // namespace tcbnn
