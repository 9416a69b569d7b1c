// Products of real-valued rows: y[m][n] = act(s[n] * sum_k x[m][k] * w[n][k] + b[n]) + r[m][n], x in bf16 or fp16,
// w of the same type (s = 1) or packed signs of +-1 with a scale per output.  Sums, scale, bias, activation and
// residual are fp32; the result is rounded once, to x's type or not at all.
//
// This form computes 64 x 64 outputs per block from shared memory with fp32 multiply-adds, any strides.
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

template <bool BITS>
__device__ __forceinline__ void tile_64(const Args& a) {
    __shared__ float sx[16][65], sw[16][65];
    const int n0 = blockIdx.x * 64, m0 = blockIdx.y * 64, t = threadIdx.x, tn = t & 15, tm = t >> 4;
    float acc[4][4] = {};
    for (int k0 = 0; k0 < a.K; k0 += 16) {
        for (int i = t; i < 1024; i += 256) {
            const int r = i >> 4, k = i & 15;
            float x = 0.f, w = 0.f;
            if (k0 + k < a.K) {
                if (m0 + r < a.M) x = load(a.x, (m0 + r) * a.ldx + k0 + k, a.type);
                if (n0 + r < a.N) {
                    if (BITS) w = reinterpret_cast<const uint32_t*>(a.W)[(n0 + r) * a.ldw + ((k0 + k) >> 5)] >> (31 - ((k0 + k) & 31)) & 1u ? 1.f : -1.f;
                    else w = load(a.W, (n0 + r) * a.ldw + k0 + k, a.type);
                }
            }
            sx[k][r] = x;
            sw[k][r] = w;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 16; k++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] = fmaf(sx[k][tm + 16 * i], sw[k][tn + 16 * j], acc[i][j]);
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int m = m0 + tm + 16 * i, n = n0 + tn + 16 * j;
            if (m >= a.M || n >= a.N) continue;
            float z = acc[i][j];
            if (BITS && a.scale) z *= a.scale[n];
            if (a.bias) z += load(a.bias, n, a.bias_type);
            z = activate(z, a.activation);
            if (a.residual) z += load(a.residual, m * a.ldr + n, a.out_type);
            store(a.out, m * a.ldo + n, a.out_type, z);
        }
}

}  // namespace linear
}  // namespace tcbnn
