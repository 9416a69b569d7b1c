// Products of few real-valued rows (linear.cuh) on warp-level MMAs (mma.sync m16n8k16, fp32 sums): no barrier lies in a warp's loop.  K is
// cut into slices over a block's warps, which meet in shared memory, in order, and finish the outputs together.  The MMA's rows are
// outputs, its columns rows of x, eight to a tile; which elements of K meet in which MMA is free as long as both operands
// agree, so every lane loads what lies together in memory.
//
// Packed weights: expanded, a weight is a sixteenth of what it weighs dense, so that with few rows neither memory nor the tensor cores
// bound the product but the expansion (a shift and a logic operation per pair of weights; three shifts of four are multiplications, on
// the pipe that has nothing else to do), the way of x to every SM, and what waits.  One expansion serves up to 32 rows.  Lane t of the four that
// share a row takes eight elements of every 32: 16 of 64 consecutive bytes of x, and a byte of each of the four words that all four load.  (128
// consecutive bytes of x per lane, for whole words of W, touch four times the lines: 32 x 1000 -> 1000 5.2 us, so 2.6.)
//
// 1 x 4096 -> 4096 in 4.0 us, 16 x 512 -> 512 in 2.0, 24 x 8192 -> 8192 in 15.6 (its MMAs 6.4): launch, one way from memory, the
// exchange; then expansions and the loads of x, with ALUs 30 % and the tensor pipe 40 % active.
//
// Dense weights: memory bounds it.  A warp has 16 rows x 128 elements (4 KB) on their way while it works on the 4 KB before, 16 warps an
// SM; lane t takes 16 bytes of every 64 of a row.  1 x 4096 -> 4096 in 8.2 us (4.1 TB/s), 1 x 4096 -> 16384 in 24.3 (5.5 TB/s, 0.85 of the
// copy rate); x asked for when it is needed instead of a piece ahead, 11.5 and 40.
#pragma once
#include "linear_umma.cuh"

namespace tcbnn {
namespace linear {

// Most warps of a block: fewer where a warp's sums and operands need more than 128 registers
__host__ __device__ constexpr int small_warps(int rt, int groups) { return rt * groups >= 8 ? 12 : 16; }
__host__ __device__ constexpr size_t small_bytes(int rt, int groups, int warps) { return (size_t)warps * 8 * groups * (rt * 16 + 4) * 4; }

__device__ __forceinline__ void mma_16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, bool bf16) {
    if (bf16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
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

// Sums of a block's warps, [warp][token][output] with rows of ROWS + 4, so that a warp's stores meet different banks
template <int ROWS, int TOKENS>
__device__ __forceinline__ void finish_small(const Args& a, const float* sums, int n0, int m0, int warps) {
    for (int i = threadIdx.x; i < ROWS * TOKENS; i += blockDim.x) {
        const int token = i / ROWS, o = i - token * ROWS, n = n0 + o, m = m0 + token;
        if (m >= a.M || n >= a.N) continue;
        float z = 0.f;
#pragma unroll 4
        for (int v = 0; v < warps; v++) z += sums[(v * TOKENS + token) * (ROWS + 4) + o];
        z = fmaf(z, a.scale ? ld_dep(a.scale + n) : 1.f, a.bias ? load(a.bias, n, a.bias_type) : 0.f);
        z = activate(z, a.activation);
        if (a.residual) z += load(a.residual, m * a.ldr + n, a.out_type);
        store(a.out, m * a.ldo + n, a.out_type, z);
    }
}

template <int RT, int T, bool BF>
__device__ __forceinline__ void bit_linear_small(const Args& a, float* sums) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, pieces = (a.K + 127) >> 7;
    const int warps = min((int)blockDim.x >> 5, pieces), n0 = blockIdx.x * RT * 16, m0 = blockIdx.y * T * 8;
    const bool wide = ((reinterpret_cast<uintptr_t>(a.x) | (uintptr_t)(a.M > 1 ? a.ldx * 2 : 0)) & 15) == 0, eights = (a.K & 7) == 0;
    // (factors that the compiler cannot know: one logic operation takes one constant, and a multiplication stays one)
    const uint32_t shift[3] = {4u * blockDim.z, 16u * blockDim.z, 64u * blockDim.z}, minus = (BF ? 0xBF80BF80u : 0xBC00BC00u) * blockDim.z;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    float acc[RT][T][4] = {};
    // (rows behind the last: the last again, whose sums nobody stores)
    const uint32_t* w_row[RT][2];
#pragma unroll
    for (int i = 0; i < RT; i++)
#pragma unroll
        for (int h = 0; h < 2; h++) w_row[i][h] = reinterpret_cast<const uint32_t*>(a.W) + (long long)min(n0 + i * 16 + h * 8 + g, a.N - 1) * a.ldw;
    const uint16_t* x_row[T];
#pragma unroll
    for (int j = 0; j < T; j++) x_row[j] = reinterpret_cast<const uint16_t*>(a.x) + (long long)min(m0 + j * 8 + g, a.M - 1) * a.ldx + 8 * t;
    auto words = [&](uint4 (&w)[RT][2], int p) {
#pragma unroll
        for (int i = 0; i < RT; i++)
#pragma unroll
            for (int h = 0; h < 2; h++) w[i][h] = ld_dep(reinterpret_cast<const uint4*>(w_row[i][h] + p * 4));
    };
    auto elements = [&](uint4 (&x)[T], int p, int s) {   // eight of a lane's 32
        const int k = p * 128 + 32 * s;
        if (wide && (eights || p * 128 + 128 <= a.K)) {
#pragma unroll
            for (int j = 0; j < T; j++) x[j] = k + 8 * t < a.K ? ld_dep(reinterpret_cast<const uint4*>(x_row[j] + k)) : make_uint4(0, 0, 0, 0);
        } else {
#pragma unroll
            for (int j = 0; j < T; j++) x[j] = eight_anywhere(x_row[j] + k, a.K - k - 8 * t);
        }
    };
    constexpr int AHEAD = T <= 2 ? 4 : 2;                // eights of x on their way
    const uint32_t mine = (3 - t) << 4 | (7 - t);        // a lane's byte of two words
    uint4 w[RT][2], x[AHEAD][T];
    if (warp < pieces) {
        words(w, warp);
#pragma unroll
        for (int s = 0; s < AHEAD; s++) elements(x[s], warp, s);
    }
    for (int p = warp; p < pieces; p += warps) {
        const bool more = p + warps < pieces;
        uint32_t v[RT][2];                               // a lane's bytes of the four words, the first on top
#pragma unroll
        for (int i = 0; i < RT; i++)
#pragma unroll
            for (int h = 0; h < 2; h++) v[i][h] = __byte_perm(__byte_perm(w[i][h].z, w[i][h].w, mine), __byte_perm(w[i][h].x, w[i][h].y, mine), 0x5410);
        if (more) words(w, p + warps);
#pragma unroll
        for (int s = 0; s < 4; s++) {                    // 32 elements of K, two MMAs a tile, expanded as in expand_signs
#pragma unroll
            for (int i = 0; i < RT; i++) {
                uint32_t f[2][4];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const uint32_t z = __byte_perm(v[i][h], v[i][h] << 1, (7 - s) << 12 | (3 - s) << 4 | (7 - s) << 8 | (3 - s));
#pragma unroll
                    for (int c = 0; c < 4; c++) f[c >> 1][2 * (c & 1) + h] = ((c ? z * shift[c - 1] : z) & 0x80008000u) ^ minus;
                }
#pragma unroll
                for (int j = 0; j < T; j++) mma_16(acc[i][j], f[0], x[s % AHEAD][j].x, x[s % AHEAD][j].y, BF);
#pragma unroll
                for (int j = 0; j < T; j++) mma_16(acc[i][j], f[1], x[s % AHEAD][j].z, x[s % AHEAD][j].w, BF);
            }
            if (s + AHEAD < 4) elements(x[s % AHEAD], p, s + AHEAD);
            else if (more) elements(x[s % AHEAD], p + warps, s + AHEAD - 4);
        }
    }
    constexpr int PITCH = RT * 16 + 4;
#pragma unroll
    for (int i = 0; i < RT; i++)
#pragma unroll
        for (int j = 0; j < T; j++)
#pragma unroll
            for (int c = 0; c < 4; c++) if (warp < warps) sums[((warp * T + j) * 8 + 2 * t + (c & 1)) * PITCH + i * 16 + g + 8 * (c >> 1)] = acc[i][j][c];
    __syncthreads();
    finish_small<RT * 16, 8 * T>(a, sums, n0, m0, warps);
}

// ---- dense weights ----------------------------------------------------------------------------------
constexpr int kDenseWarps = 8, kDensePiece = 128;
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
    float* mine = sums + (warp * 8 + 2 * t) * 20 + g;      // a thread's four sums
    auto add_up = [&]() {
#pragma unroll
        for (int c = 0; c < 4; c++) {
            mine[(c & 1) * 20 + 8 * (c >> 1)] += acc[c];
            acc[c] = 0.f;
        }
    };
#pragma unroll
    for (int c = 0; c < 4; c++) mine[(c & 1) * 20 + 8 * (c >> 1)] = 0.f;
    uint4 v[2][4][3];
    if (warp < pieces) ask(v[0], warp);
    for (int p = warp, turn = 0; p < pieces; p += 2 * kDenseWarps) {
        if (turn++ == 3) { add_up(); turn = 1; }               // (chains of 768 of K: see linear_umma.cuh)
        if (p + kDenseWarps < pieces) ask(v[1], p + kDenseWarps);
        work(v[0]);
        if (p + kDenseWarps >= pieces) break;
        if (p + 2 * kDenseWarps < pieces) ask(v[0], p + 2 * kDenseWarps);
        work(v[1]);
    }
    add_up();
    __syncthreads();
    finish_small<16, 8>(a, sums, n0, m0, kDenseWarps);
}

}  // namespace linear
}  // namespace tcbnn
