// Products of few real-valued rows with packed binary weights (linear.cuh) on warp-level MMAs (mma.sync m16n8k16, fp32 sums).
//
// Expanded, a weight is a sixteenth of what it weighs dense, so that with few rows neither memory nor the tensor cores bound the
// product but the expansion, two logic operations per pair of weights, and everything that waits.  Here nothing does: a warp expands the
// bits straight into an MMA's fragments, and no barrier lies in its loop.  K is cut into slices over a block's warps, which meet in
// shared memory, in order, and finish the outputs together.
//
// The MMA's rows are outputs (RT times 16 per block), its columns rows of x, eight per block.  Which elements of K meet in which MMA is free
// as long as both operands agree: of 256 elements lane t of the four that share a row takes words 2t and 2t + 1 -- eight bytes of W, a
// whole sector with its neighbours -- and of x the 64 elements that belong to them, 128 consecutive bytes.
#pragma once
#include "linear_umma.cuh"

namespace tcbnn {
namespace linear {

constexpr int kSmallWarps = 16;
__host__ __device__ constexpr size_t small_bytes(int rt, int warps) { return (size_t)warps * 8 * (rt * 16 + 4) * 4; }

__device__ __forceinline__ void mma_16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, bool bf16) {
    if (bf16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// eight elements of a row of x from element k on, zeros behind the last
__device__ __forceinline__ uint4 eight(const uint16_t* row, int k, int K, bool wide) {
    if (wide && k + 8 <= K) return ld_dep(reinterpret_cast<const uint4*>(row + k));
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++)
        w[i] = (k + 2 * i < K ? (uint32_t)row[k + 2 * i] : 0u) | (k + 2 * i + 1 < K ? (uint32_t)row[k + 2 * i + 1] << 16 : 0u);
    return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int RT, bool BF>
__device__ __forceinline__ void bit_linear_small(const Args& a, float* sums) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, warps = blockDim.x >> 5;
    const int n0 = blockIdx.x * RT * 16, m0 = blockIdx.y * 8, pieces = (a.K + 255) >> 8;
    const bool wide = ((reinterpret_cast<uintptr_t>(a.x) | (uintptr_t)(a.ldx * 2)) & 15) == 0;
    constexpr uint32_t minus = BF ? 0xBF80BF80u : 0xBC00BC00u;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    float acc[RT][4] = {};
    const uint32_t* w_row[RT][2];
#pragma unroll
    for (int i = 0; i < RT; i++)
#pragma unroll
        for (int h = 0; h < 2; h++) w_row[i][h] = reinterpret_cast<const uint32_t*>(a.W) + (long long)min(n0 + i * 16 + h * 8 + g, a.N - 1) * a.ldw + 2 * t;
    const bool row = m0 + g < a.M;
    const uint16_t* x_row = reinterpret_cast<const uint16_t*>(a.x) + (long long)(row ? m0 + g : 0) * a.ldx;
    // (Behind the last word of a row there is none to load: its elements of x are zeros.)
    auto words = [&](uint2 (&w)[RT][2], int p) {
#pragma unroll
        for (int i = 0; i < RT; i++)
#pragma unroll
            for (int h = 0; h < 2; h++) w[i][h] = p * 8 + 2 * t < a.ldw ? ld_dep(reinterpret_cast<const uint2*>(w_row[i][h] + p * 8)) : make_uint2(0, 0);
    };
    auto elements = [&](uint4 (&x)[4], int p, int u) {   // 32 of a lane's row, those of word u
#pragma unroll
        for (int q = 0; q < 4; q++) x[q] = row ? eight(x_row, p * 256 + 64 * t + 32 * u + 8 * q, a.K, wide) : make_uint4(0, 0, 0, 0);
    };
    uint2 w[RT][2], next[RT][2];
    uint4 x[2][4];
    if (warp < pieces) words(w, warp);
    for (int p = warp; p < pieces; p += warps) {
        elements(x[0], p, 0);
        elements(x[1], p, 1);
        if (p + warps < pieces) words(next, p + warps);
#pragma unroll
        for (int u = 0; u < 2; u++) {                    // 128 elements of K, eight MMAs
#pragma unroll
            for (int i = 0; i < RT; i++) {
                // as in expand_signs, eight elements of a word at a time
                uint32_t z[2][2];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const uint32_t v = u ? w[i][h].y : w[i][h].x;
                    z[h][0] = __byte_perm(v, v << 1, 0x7632);
                    z[h][1] = __byte_perm(v, v << 1, 0x5410);
                }
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    uint32_t f[2][4];
#pragma unroll
                    for (int c = 0; c < 4; c++)
#pragma unroll
                        for (int h = 0; h < 2; h++) f[c >> 1][2 * (c & 1) + h] = ((z[h][q >> 1] << (2 * (4 * (q & 1) + c))) & 0x80008000u) ^ minus;
                    mma_16(acc[i], f[0], x[u][q].x, x[u][q].y, BF);
                    mma_16(acc[i], f[1], x[u][q].z, x[u][q].w, BF);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < RT; i++)
#pragma unroll
            for (int h = 0; h < 2; h++) w[i][h] = next[i][h];
    }
    // [warp][token][output], rows 4 apart from a multiple of 16 so that a warp's stores meet different banks
    constexpr int PITCH = RT * 16 + 4;
#pragma unroll
    for (int i = 0; i < RT; i++)
#pragma unroll
        for (int c = 0; c < 4; c++) sums[(warp * 8 + 2 * t + (c & 1)) * PITCH + i * 16 + g + 8 * (c >> 1)] = acc[i][c];
    __syncthreads();
    for (int i = threadIdx.x; i < RT * 16 * 8; i += blockDim.x) {
        const int token = i / (RT * 16), o = i - token * (RT * 16), n = n0 + o, m = m0 + token;
        if (m >= a.M || n >= a.N) continue;
        float z = 0.f;
        for (int v = 0; v < warps; v++) z += sums[(v * 8 + token) * PITCH + o];
        z = fmaf(z, a.scale ? ld_dep(a.scale + n) : 1.f, a.bias ? load(a.bias, n, a.bias_type) : 0.f);
        z = activate(z, a.activation);
        if (a.residual) z += load(a.residual, m * a.ldr + n, a.out_type);
        store(a.out, m * a.ldo + n, a.out_type, z);
    }
}

}  // namespace linear
}  // namespace tcbnn
