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
__device__ __forceinline__ float activate(float z, int a) {
    if (a == RELU) return z < 0.f ? 0.f : z;           // (NaN stays)
    if (a == GELU) return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
    if (a == GELU_TANH) return 0.5f * z * (1.f + tanhf(0.79788456080286536f * (z + 0.044715f * z * z * z)));
    if (a == SILU) return z / (1.f + expf(-z));
    return z;
}

}  // namespace linear
}  // namespace tcbnn
