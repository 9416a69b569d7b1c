// Products of few real-valued rows (linear.cuh) on warp-level MMAs (mma.sync m16n8k16, fp32 sums): no barrier lies in a warp's loop.  K is
// cut into slices over a block's warps, which meet in shared memory, in order, and finish the outputs together.  The MMA's rows are
// outputs, its columns rows of x, eight or sixteen per block; which elements of K meet in which MMA is free as long as both operands
// agree, so every lane loads what lies together in memory.
//
// Packed weights: expanded, a weight is a sixteenth of what it weighs dense, so that with few rows neither memory nor the tensor cores
// bound the product but the expansion, two logic operations per pair of weights, and everything that waits.  Of 256 elements lane t of the
// four that share a row takes words 2t and 2t + 1 -- eight bytes of W, a whole sector with its neighbours -- and of x the 64 elements
// that belong to them, 128 consecutive bytes.
//
// 1 x 4096 -> 4096 in 4.1 us, 16 x 512 -> 512 in 3.1: launch, one way from memory, expansions (1.3 us), the exchange.
//
// Dense weights: memory bounds it.  A warp has 16 rows x 128 elements (4 KB) on their way while it works on the 4 KB before, 16 warps an
// SM; lane t takes 16 bytes of every 64 of a row.  1 x 4096 -> 4096 in 8.2 us (4.1 TB/s), 1 x 4096 -> 16384 in 24.3 (5.5 TB/s, 0.85 of the
// copy rate); x asked for when it is needed instead of a piece ahead, 11.5 and 40.
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

// Sums of a block's warps, [warp][token][output] with rows of ROWS + 4, so that a warp's stores meet different banks
template <int ROWS, int TOKENS>
__device__ __forceinline__ void finish_small(const Args& a, const float* sums, int n0, int m0, int warps) {
    for (int i = threadIdx.x; i < ROWS * TOKENS; i += blockDim.x) {
        const int token = i / ROWS, o = i - token * ROWS, n = n0 + o, m = m0 + token;
        if (m >= a.M || n >= a.N) continue;
        float z = 0.f;
        for (int v = 0; v < warps; v++) z += sums[(v * TOKENS + token) * (ROWS + 4) + o];
        z = fmaf(z, a.scale ? ld_dep(a.scale + n) : 1.f, a.bias ? load(a.bias, n, a.bias_type) : 0.f);
        z = activate(z, a.activation);
        if (a.residual) z += load(a.residual, m * a.ldr + n, a.out_type);
        store(a.out, m * a.ldo + n, a.out_type, z);
    }
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
    constexpr int PITCH = RT * 16 + 4;
#pragma unroll
    for (int i = 0; i < RT; i++)
#pragma unroll
        for (int c = 0; c < 4; c++) sums[(warp * 8 + 2 * t + (c & 1)) * PITCH + i * 16 + g + 8 * (c >> 1)] = acc[i][c];
    __syncthreads();
    finish_small<RT * 16, 8>(a, sums, n0, m0, warps);
}

// ---- dense weights ----------------------------------------------------------------------------------
constexpr int kDenseWarps = 8, kDensePiece = 128;
// Eight elements from any element on: words from the one that holds the first, turned by half a word where that is its upper half.  Words
// behind the last element of the row are not read (`left` elements exist), elements behind it are zeros.
__device__ __forceinline__ uint4 eight_anywhere(const uint16_t* p, int left) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    const uint32_t* words = reinterpret_cast<const uint32_t*>(at & ~(uintptr_t)3);
    const int odd = (int)(at >> 1) & 1, last = (left - 1 + odd) >> 1;
    uint32_t w[5];
#pragma unroll
    for (int i = 0; i < 5; i++) w[i] = left > 0 ? ld_dep(words + min(i, last)) : 0u;
    uint32_t v[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        v[i] = __funnelshift_r(w[i], w[i + 1], 16 * odd);
        v[i] &= left >= 2 * i + 2 ? 0xFFFFFFFFu : left == 2 * i + 1 ? 0xFFFFu : 0u;
    }
    return make_uint4(v[0], v[1], v[2], v[3]);
}
// WIDE: the rows of both operands start on 16 bytes
template <bool BF, bool WIDE>
__device__ __forceinline__ void linear_small(const Args& a, float* sums) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 8, pieces = (a.K + kDensePiece - 1) / kDensePiece;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    // (rows behind the last: the last again, whose sums nobody stores)
    const uint16_t* row[3];
#pragma unroll
    for (int h = 0; h < 2; h++) row[h] = reinterpret_cast<const uint16_t*>(a.W) + (long long)min(n0 + h * 8 + g, a.N - 1) * a.ldw;
    row[2] = reinterpret_cast<const uint16_t*>(a.x) + (long long)min(m0 + g, a.M - 1) * a.ldx;
    auto ask = [&](uint4 (&v)[4][3], int p) {
#pragma unroll
        for (int q = 0; q < 4; q++)
#pragma unroll
            for (int h = 0; h < 3; h++) {
                const int k = p * kDensePiece + 32 * q + 8 * t;
                v[q][h] = WIDE && k + 8 <= a.K ? ld_dep(reinterpret_cast<const uint4*>(row[h] + k)) : eight_anywhere(row[h] + k, a.K - k);
            }
    };
    float acc[4] = {};
    auto work = [&](const uint4 (&v)[4][3]) {
#pragma unroll
        for (int q = 0; q < 4; q++) {                    // 32 elements of K, two MMAs
            const uint32_t f0[4] = {v[q][0].x, v[q][1].x, v[q][0].y, v[q][1].y}, f1[4] = {v[q][0].z, v[q][1].z, v[q][0].w, v[q][1].w};
            mma_16(acc, f0, v[q][2].x, v[q][2].y, BF);
            mma_16(acc, f1, v[q][2].z, v[q][2].w, BF);
        }
    };
    uint4 v[2][4][3];
    if (warp < pieces) ask(v[0], warp);
    for (int p = warp; p < pieces; p += 2 * kDenseWarps) {
        if (p + kDenseWarps < pieces) ask(v[1], p + kDenseWarps);
        work(v[0]);
        if (p + kDenseWarps >= pieces) break;
        if (p + 2 * kDenseWarps < pieces) ask(v[0], p + 2 * kDenseWarps);
        work(v[1]);
    }
#pragma unroll
    for (int c = 0; c < 4; c++) sums[(warp * 8 + 2 * t + (c & 1)) * 20 + g + 8 * (c >> 1)] = acc[c];
    __syncthreads();
    finish_small<16, 8>(a, sums, n0, m0, kDenseWarps);
}

}  // namespace linear
}  // namespace tcbnn
