// Products of real-valued rows on tcgen05 (kind::f16, fp32 accumulators in tensor memory):
// y[m][n] = act(s[n] * sum_k x[m][k] w[n][k] + b[n]) + r[m][n].
//
// The MMA's 128 rows are rows of W (outputs), its columns rows of x (tokens): one token costs 16 columns, a prompt 256,
// by the same kernel, and what belongs to an output -- scale, bias, where it is stored -- belongs to a lane.
//
//   warps 0-7   epilogue  : 32 outputs x 32 tokens at a time
//   warp  8     loader W  : tensor copies of 128 rows x 64 (dense) or 128 rows x 512 bits (packed)
//   warp  9     loader x  : tensor copies of `cols` rows x 64
//   warp  10    MMA       : converged, elected lane; four MMAs of K = 16 per 64
//   warps 12-15 expanders : (packed) signs to +-1 in tensor memory, where the MMA reads its W operand
//
// Tensor copies fill rows and elements past the end with zeros, so no size needs a case of its own.
//
// Packed weights cost a sixteenth of the bytes, and expanded in tensor memory they take nothing of the shared-memory port, which rows
// of x fill.  An MMA takes 100 clocks that way at least, whatever its columns, and a block of 64 of K 400 to 570 with what the
// expanders wait for: few tokens are another kernel's (linear_small.cuh).  Expanded in shared memory instead, 475 clocks; two groups of
// expanders, no faster at 256 columns (472 us against 466, below); blocks handed over in twos and fours, 420 clocks, but
// 680 at 256 columns; pairs of SMs, 429 us against 410: all taken back.
//
// Where tiles of 128 x cols leave SMs idle, K is cut over a cluster's CTAs (SPLIT), whose sums meet in shared memory, in rank
// order: the same result every time.  Where there are enough, pairs of SMs own tiles of 256 outputs (PAIR): each CTA holds its
// 128 rows of W and half of the tokens' rows, the leader issues MMAs that read both (cta_group::2), so that rows of x
// come from L2 and out of shared memory half as often.
//
// What bounds it: large products the GPU's power.  4096 x 16384 x 4096 over a second takes 400 us in pairs (1374 TFLOP/s, 1.3 GHz, 0.98 of
// cuBLAS in the same minute), 437 without pairs, with gelu 417, fp32 results 436 and 493; packed weights 408, with gelu 453, as two sets of
// 256 columns do not fit beside the expanded weights and half of an epilogue shows.  In a burst 350 (0.95 of the measured GEMM rate).  Few tokens: W's way from
// memory, 16 x 9216 -> 4096 16.2 us for 75 MB (0.72 of the copy rate).  Between them a CTA's bytes from L2, 72 per clock, and
// set-up and epilogue, 3 us of a launch.
#pragma once
#include "bconv_umma_pre.cuh"
#include "linear.cuh"

namespace tcbnn {
namespace linear {

constexpr int kThreadsDense = 11 * 32, kThreadsBits = 16 * 32;
constexpr int kMaxCols = 256, kMaxStages = 12, kMaxRing = 8, kRawStages = 3;
constexpr uint32_t kWStage = 128 * 128, kRawStage = 128 * 64;            // 128 rows of 64 elements, of 512 bits

// 32 tokens x 32 outputs of 16 bits that an epilogue warp turns: rows of 64 bytes, 80 apart, so that eight of them meet different banks
constexpr uint32_t kTurnPitch = 80, kTurn = 32 * kTurnPitch;
enum Form { ALONE = 0, SPLIT = 1, PAIR = 2 };
struct Plan {
    int bits, form, cols, splits;                      // tokens per tile (a multiple of 16), CTAs that share K
    int tiles_m, tiles_n, band;                        // tiles of tokens and of outputs; token tiles worked on together
    int kblocks, per;                                  // of 64; of a CTA
    int stages, ring, accumulators;                    // of x (and dense W), of expanded W, of sums
    int columns;                                       // of tensor memory
    int chained;                                       // the sets of sums take turns by chains of kChain blocks
};
// The tensor cores cut an fp32 sum off at every 16 of K, always towards zero: 4.7e-7 of the result after 512 of K, 1.0e-6 after 1024, 4.4e-6
// after 4096, 1.9e-5 after 16384 (fp32 multiply-adds: 6e-7 and 1.5e-6 at the last two).  16-bit results round that away.  For fp32
// results of dense weights a set of sums takes chains of at most kChain blocks, and the epilogue adds the chains up in registers: 5e-7 to
// 7e-7 at any K (fp16, whose products are longer, 6e-7 to 9.6e-7; sums that only grow 1.5e-6 and 4.3e-6).  The sets take turns as they
// otherwise do by tiles, or a cluster's CTA has a set for each of its chains.  4096 x 4096 -> 16384 368 -> 378 us, with gelu 391 -> 422;
// smaller ones as fast on average.  Sums of +-1 times x lose 5e-7 after 16384 and are left in one chain.
constexpr int kChain = 12, kChainCols = 64;            // columns of a cluster's CTA whose sets take turns: its registers hold no more
// rows of x that a CTA holds of a tile
__host__ __device__ inline int own_cols(const Plan& p) { return p.form == PAIR ? p.cols / 2 : p.cols; }
__host__ __device__ inline uint32_t stage_bytes(const Plan& p) { return (p.bits ? 0u : kWStage) + (uint32_t)own_cols(p) * 128u; }
// ring (where the cluster's sums go afterwards), raw bits, barriers; 1 KB for its alignment
__host__ __device__ inline size_t ring_bytes(const Plan& p) {
    const size_t ring = (size_t)p.stages * stage_bytes(p), sums = p.splits > 1 ? (size_t)p.cols * 512 : 0;
    return ((ring > sums ? ring : sums) + 1023) & ~(size_t)1023;
}
__host__ __device__ inline size_t smem_bytes(const Plan& p) {
    return ring_bytes(p) + (p.bits ? kRawStages * kRawStage : 0) + (p.form != SPLIT ? 8 * kTurn : 0) + 64 * 8 + 1024;
}

__device__ __forceinline__ void tensor_g2s(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
// the same to the calling CTA of a pair, completing on the leader's barrier (no multicast)
__device__ __forceinline__ void tensor_g2s_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t leader_bar) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(leader_bar) : "memory");
}
// rows of 128 bytes, 128-byte swizzle, eight rows 1 KB apart from the next
__device__ __forceinline__ uint64_t swizzled_desc(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
// fp16 or bf16 operands, both K-major, fp32 sums
__device__ __forceinline__ uint32_t idesc_16(int type, int m, int n) {
    const uint32_t f = type == BF16 ? 1u : 0u;
    return (1u << 4) | (f << 7) | (f << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// Four MMAs over 64 elements of K: both operands 32 bytes (two 16-byte units of the descriptor) on each time, or A
// eight columns of tensor memory.  The commits of a pair arrive in both CTAs.
// As one block with the tests of the barriers of the next stage (and, TS, of the next W operand) in front and their answers read
// behind: a test takes 150-200 clocks to return while the MMAs keep the shared-memory port busy, and the tensor pipe queues no more
// than two or three instructions.  Then the commits of the stage, of the operand and (bar_c != 0) of the sums.
// a: descriptor (low half) of W in shared memory, or its address in tensor memory (TS).  Bit 0 / 1 of the result: phase par0 / par1
// of bar0 / bar1 is complete.
#define TCBNN_MMA_SS(G, PRED)                                                                        \
    "mov.b64 da, {xa, %5};\n\tmov.b64 db, {xb, %5};\n\t"                                            \
    "@pl tcgen05.mma.cta_group::" G ".kind::f16 [%2], da, db, %6, " PRED ";\n\tadd.u32 xa, xa, 2;\n\tadd.u32 xb, xb, 2;\n\t"
#define TCBNN_MMA_TS(G, PRED)                                                                        \
    "mov.b64 db, {xb, %5};\n\t"                                                                     \
    "@pl tcgen05.mma.cta_group::" G ".kind::f16 [%2], [xa], db, %6, " PRED ";\n\tadd.u32 xa, xa, 8;\n\tadd.u32 xb, xb, 2;\n\t"
#define TCBNN_MMA_RUN(OP, SECOND, G, Q, W, B)                                                        \
    asm volatile("{\n\t.reg .pred p0, p1, pa, pt, pl, pc, ps;\n\t.reg .b64 da, db;\n\t.reg .b32 xa, xb, r1;\n\t.reg .b16 both;\n\tmov.b16 both, 3;\n\t" \
                 "mbarrier.test_wait.parity" Q ".shared::cta.b64 p0, [%8], %9;\n\t"                  \
                 "setp.ne.b32 p1, %1, %1;\n\t" SECOND("mbarrier.test_wait.parity" Q ".shared::cta.b64 p1, [%10], %11;\n\t") \
                 "setp.ne.b32 pa, %7, 0;\n\tsetp.ne.b32 pl, %1, 0;\n\tsetp.eq.b32 pt, %1, %1;\n\tsetp.ne.and.b32 pc, %14, 0, pl;\n\t" \
                 "mov.u32 xa, %3;\n\tmov.u32 xb, %4;\n\t" OP(G, "pa") OP(G, "pt") OP(G, "pt") OP(G, "pt") \
                 "@pl tcgen05.commit.cta_group::" G ".mbarrier::arrive::one.shared::cluster" W ".b64 [%12]" B ";\n\t" \
                 SECOND("@pl tcgen05.commit.cta_group::" G ".mbarrier::arrive::one.shared::cluster" W ".b64 [%13]" B ";\n\t") \
                 "@pc tcgen05.commit.cta_group::" G ".mbarrier::arrive::one.shared::cluster" W ".b64 [%14]" B ";\n\t" \
                 "selp.u32 %0, 1, 0, p0;\n\tselp.u32 r1, 2, 0, p1;\n\tor.b32 %0, %0, r1;\n\t}"      \
                 : "=&r"(ok) : "r"(leader), "r"(d), "r"(a), "r"(b_lo), "r"(hi), "r"(idesc), "r"(acc), "r"(bar0), "r"(par0), "r"(bar1), \
                   "r"(par1), "r"(bar_e), "r"(bar_r), "r"(bar_c) : "memory")
#define TCBNN_YES(X) X
#define TCBNN_NO(X) ""
template <bool TS, bool PAIR>
__device__ __forceinline__ uint32_t mma_64(uint32_t leader, uint32_t d, uint32_t a, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t acc,
                                           uint32_t bar0, uint32_t par0, uint32_t bar1, uint32_t par1, uint32_t bar_e, uint32_t bar_r, uint32_t bar_c) {
    uint32_t ok;
    if constexpr (TS && PAIR) TCBNN_MMA_RUN(TCBNN_MMA_TS, TCBNN_YES, "2", ".acquire.cluster", ".multicast::cluster", ", both");
    else if constexpr (TS) TCBNN_MMA_RUN(TCBNN_MMA_TS, TCBNN_YES, "1", "", "", "");
    else if constexpr (PAIR) TCBNN_MMA_RUN(TCBNN_MMA_SS, TCBNN_NO, "2", ".acquire.cluster", ".multicast::cluster", ", both");
    else TCBNN_MMA_RUN(TCBNN_MMA_SS, TCBNN_NO, "1", "", "", "");
    return ok;
}
#undef TCBNN_YES
#undef TCBNN_NO
#undef TCBNN_MMA_RUN
#undef TCBNN_MMA_TS
#undef TCBNN_MMA_SS
// 32 signs as 16 pairs of +-1: register i holds elements 2i (low half) and 2i + 1, which are bits 31 - 2i and 30 - 2i.  `minus`:
// -1 twice, whose signs a set bit turns.  The word is laid out once so that a shift brings both bits to their places; half of the shifts are
// multiplications, which another pipe takes (`four`, unknown to the compiler: 1001 x 2049 -> 5000 30.5 -> 29.3 us).
__device__ __forceinline__ void expand_signs(uint32_t w, uint32_t minus, uint32_t four, uint32_t* r) {
    const uint32_t a = __byte_perm(w, w << 1, 0x7632);
    uint32_t b = __byte_perm(w, w << 1, 0x5410);
#pragma unroll
    for (int i = 0; i < 8; i++) {
        r[i] = ((a << (2 * i)) & 0x80008000u) ^ minus;
        r[8 + i] = (b & 0x80008000u) ^ minus;
        b *= four;
    }
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&e)[32]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
                 "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
                 ::"r"(taddr), "r"(e[0]), "r"(e[1]), "r"(e[2]), "r"(e[3]), "r"(e[4]), "r"(e[5]), "r"(e[6]), "r"(e[7]), "r"(e[8]), "r"(e[9]),
                   "r"(e[10]), "r"(e[11]), "r"(e[12]), "r"(e[13]), "r"(e[14]), "r"(e[15]), "r"(e[16]), "r"(e[17]), "r"(e[18]), "r"(e[19]),
                   "r"(e[20]), "r"(e[21]), "r"(e[22]), "r"(e[23]), "r"(e[24]), "r"(e[25]), "r"(e[26]), "r"(e[27]), "r"(e[28]), "r"(e[29]),
                   "r"(e[30]), "r"(e[31]) : "memory");
}
__device__ __forceinline__ float4 ld_peer4(uint32_t shared, uint32_t rank) {
    uint32_t p;
    float4 v;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(p) : "r"(shared), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(p) : "memory");
    return v;
}

template <bool SHORT, int COUNT>
__device__ __forceinline__ void activate_all(float (&v)[COUNT], int activation) {
    switch (activation) {
    case RELU:
#pragma unroll
        for (int j = 0; j < COUNT; j++) v[j] = activate<SHORT>(v[j], RELU);
        break;
    case GELU:
#pragma unroll
        for (int j = 0; j < COUNT; j++) v[j] = activate<SHORT>(v[j], GELU);
        break;
    case GELU_TANH:
#pragma unroll
        for (int j = 0; j < COUNT; j++) v[j] = activate<SHORT>(v[j], GELU_TANH);
        break;
    case SILU:
#pragma unroll
        for (int j = 0; j < COUNT; j++) v[j] = activate<SHORT>(v[j], SILU);
        break;
    }
}
// Results of fp32, and the few of a cluster's CTA: a lane has its output's scale and bias, and stores token by token, a warp 128
// (64) consecutive bytes.
template <bool F32>
struct Output {
    const Args& a;
    int n;
    float scale, bias;
    __device__ __forceinline__ Output(const Args& a_, int n_) : a(a_), n(n_), scale(1.f), bias(0.f) {
        if (n >= a.N) return;
        if (a.scale) scale = ld_dep(a.scale + n);
        if (a.bias) bias = load(a.bias, n, a.bias_type);
    }
    template <int COUNT>
    __device__ __forceinline__ void finish(float (&v)[COUNT], int m0, int rows) const {
#pragma unroll
        for (int j = 0; j < COUNT; j++) v[j] = fmaf(v[j], scale, bias);
        activate_all<false>(v, a.activation);
        if (n >= a.N) return;
        const int type = F32 ? (int)FP32 : a.out_type;
        if (a.residual) {
            long long at = m0 * a.ldr + n;
#pragma unroll
            for (int j = 0; j < COUNT; j++, at += a.ldr)
                if (j < rows) v[j] += load(a.residual, at, type);
        }
        long long at = m0 * a.ldo + n;
#pragma unroll
        for (int j = 0; j < COUNT; j++, at += a.ldo)
            if (j < rows) store(a.out, at, type, v[j]);
    }
};
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t pack16(float lo, float hi, int type) {
    uint32_t w;
    if (type == BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
    return w;
}
__device__ __forceinline__ float2 unpack16(uint32_t w, int type) {
    if (type == BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
// Results of 16 bits.  The sums come in pieces of 8 outputs x 8 tokens spread over a warp like an MMA's fragments, which stmatrix
// stores turned, a token's eight outputs together; 16 bytes of a row are then a lane's, and a residual goes the other way.
// (Two-byte stores, a lane an output: 16,000 clocks for 128 x 256.)
struct Output16 {
    const Args& a;
    uint32_t turn;                                     // this warp's buffer
    int n0;                                            // first of the warp's 32 outputs
    bool wide_out, wide_res;                           // rows of 16-byte pieces
    float scale[4], bias[4];                           // of outputs n0 + 8 i + lane / 4
    __device__ __forceinline__ Output16(const Args& a_, uint32_t turn_, int n0_) : a(a_), turn(turn_), n0(n0_) {
        wide_out = ((reinterpret_cast<uintptr_t>(a.out) | (uintptr_t)(a.ldo * 2)) & 15) == 0;
        wide_res = ((reinterpret_cast<uintptr_t>(a.residual) | (uintptr_t)(a.ldr * 2)) & 15) == 0;
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int n = n0 + 8 * i + (lane >> 2);
            scale[i] = a.scale && n < a.N ? ld_dep(a.scale + n) : 1.f;
            bias[i] = a.bias && n < a.N ? load(a.bias, n, a.bias_type) : 0.f;
        }
    }
    // piece i of a lane: token m0 + 8 i + lane / 4, outputs n + 0..7
    __device__ __forceinline__ void ask(uint4 (&r)[4], int m0, int rows) const {
        const int lane = threadIdx.x & 31, n = n0 + 8 * (lane & 3);
        const uint16_t* p = reinterpret_cast<const uint16_t*>(a.residual) + n;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int j = 8 * i + (lane >> 2);
            const uint16_t* q = p + (m0 + j) * a.ldr;
            r[i] = make_uint4(0, 0, 0, 0);
            if (j >= rows) continue;
            if (wide_res && n + 8 <= a.N) {
                r[i] = ld_dep(reinterpret_cast<const uint4*>(q));
            } else {
                uint32_t w[8];
#pragma unroll
                for (int e = 0; e < 8; e++) w[e] = n + e < a.N ? q[e] : 0u;
                r[i] = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
            }
        }
    }
    // sums of 16 lanes (outputs) each as tmem_ld_16x256b_x4 gives them
    __device__ __forceinline__ void finish(const int (&lo)[16], const int (&hi)[16], const uint4 (&r)[4], int m0, int rows) const {
        const int lane = threadIdx.x & 31;
        float v[32];
#pragma unroll
        for (int k = 0; k < 16; k++) {                   // register 4n + 2s + e: eight outputs s, token 8n + 2 (lane % 4) + e
            const int s = (k >> 1) & 1;
            v[k] = fmaf(__int_as_float(lo[k]), scale[s], bias[s]);
            v[16 + k] = fmaf(__int_as_float(hi[k]), scale[2 + s], bias[2 + s]);
        }
        activate_all<true>(v, a.activation);
        const uint32_t piece = turn + (lane >> 2) * kTurnPitch + (lane & 3) * 16;       // a lane's 16 bytes
        const uint32_t row = turn + (lane & 7) * kTurnPitch + (lane >> 3) * 16;          // a fragment's row
        if (a.residual) {
#pragma unroll
            for (int i = 0; i < 4; i++)
                asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(piece + i * 8 * kTurnPitch), "r"(r[i].x), "r"(r[i].y), "r"(r[i].z), "r"(r[i].w) : "memory");
            __syncwarp();
#pragma unroll
            for (int n = 0; n < 4; n++) {
                uint32_t w[4];
                asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                             : "r"(row + n * 8 * kTurnPitch) : "memory");
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float2 f = unpack16(w[i], a.out_type);
                    v[(i >> 1) * 16 + 4 * n + 2 * (i & 1)] += f.x;
                    v[(i >> 1) * 16 + 4 * n + 2 * (i & 1) + 1] += f.y;
                }
            }
            __syncwarp();
        }
#pragma unroll
        for (int n = 0; n < 4; n++)
            asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(row + n * 8 * kTurnPitch),
                         "r"(pack16(v[4 * n], v[4 * n + 1], a.out_type)), "r"(pack16(v[4 * n + 2], v[4 * n + 3], a.out_type)),
                         "r"(pack16(v[16 + 4 * n], v[16 + 4 * n + 1], a.out_type)), "r"(pack16(v[16 + 4 * n + 2], v[16 + 4 * n + 3], a.out_type)) : "memory");
        __syncwarp();
        const int n = n0 + 8 * (lane & 3);
        uint16_t* p = reinterpret_cast<uint16_t*>(a.out) + n;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int j = 8 * i + (lane >> 2);
            if (j >= rows || n >= a.N) continue;
            uint16_t* q = p + (m0 + j) * a.ldo;
            const uint4 w = lds128(piece + i * 8 * kTurnPitch);
            if (wide_out && n + 8 <= a.N) {
                *reinterpret_cast<uint4*>(q) = w;
            } else {
                const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (n + e < a.N) q[e] = (uint16_t)(x[e >> 1] >> (16 * (e & 1)));
            }
        }
        __syncwarp();                                    // (the buffer is read)
    }
};

// CHAINED: for results of fp32
template <bool BITS, int FORM, bool CHAINED>
__device__ __forceinline__ void umma_cta(const Args& a, const Plan& p, const CUtensorMap* map_w, const CUtensorMap* map_x, int* status,
                                         unsigned char* smem0) {
    using namespace umma;
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem0) + 1023) & ~(uintptr_t)1023);
    constexpr bool CLUSTER = FORM == SPLIT, PAIRED = FORM == PAIR;
    static_assert(!BITS || !PAIRED, "no pairs with packed weights: they were no faster");
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t nctas = CLUSTER ? [] { uint32_t n; asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(n)); return n; }() : 1u;
    const uint32_t rank = CLUSTER || PAIRED ? [] { uint32_t r; asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }() : 0u;
    const uint32_t stage = stage_bytes(p);
    unsigned char* sRaw = smem + ring_bytes(p);
    unsigned char* sTurn = sRaw + (BITS ? kRawStages * kRawStage : 0);
    uint64_t* sBar = reinterpret_cast<uint64_t*>(sTurn + (CLUSTER ? 0 : 8 * kTurn));
    // barriers: full[12] | empty[12] | ring full[8] | ring empty[8] | raw full[3] | raw empty[3] | sums full[2] | sums empty[2] | drain
    uint32_t* sTmem = reinterpret_cast<uint32_t*>(sBar + 51);
    volatile int* sAbort = reinterpret_cast<volatile int*>(sTmem + 1);
    const uint32_t bar0 = smem_u32(sBar);
    auto FULL = [&](int s) { return bar0 + 8u * s; };
    auto EMPTY = [&](int s) { return bar0 + 8u * (12 + s); };
    auto RFULL = [&](int s) { return bar0 + 8u * (24 + s); };
    auto REMPTY = [&](int s) { return bar0 + 8u * (32 + s); };
    auto RAWFULL = [&](int s) { return bar0 + 8u * (40 + s); };
    auto RAWEMPTY = [&](int s) { return bar0 + 8u * (43 + s); };
    auto SFULL = [&](int b) { return bar0 + 8u * (46 + b); };
    auto SEMPTY = [&](int b) { return bar0 + 8u * (48 + b); };
    const uint32_t DRAIN = bar0 + 8u * 50;

    // (a pair walks over the tiles together)
    const int team = CLUSTER ? (int)nctas : PAIRED ? 2 : 1;
    const int t_first = (int)blockIdx.x / team, t_step = (int)gridDim.x / team;
    const int ntiles = p.tiles_m * p.tiles_n;
    const int kb0 = CLUSTER ? (int)rank * p.per : 0, nkb = max(0, min(p.per, p.kblocks - kb0));     // this CTA's blocks of K
    const int n_of = PAIRED ? 256 : 128, n_own = PAIRED ? (int)rank * 128 : 0, own = own_cols(p);
    // bands of token tiles, in a band the tokens fastest: what runs together shares rows of both operands
    auto tile = [&](int t, int& tm, int& tn) {
        const int full = p.band * p.tiles_n, b = t / full, r = t - b * full, w = min(p.band, p.tiles_m - b * p.band);
        tn = r / w;
        tm = b * p.band + r - tn * w;
    };

    if (warp == 8 && lane == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(map_w) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(map_x) : "memory");
    }
    if (tid == 0) {
        for (int s = 0; s < kMaxStages; s++) { mbar_init(FULL(s), BITS ? 1 : 2); mbar_init(EMPTY(s), 1); }
        for (int s = 0; s < kMaxRing; s++) { mbar_init(RFULL(s), 4); mbar_init(REMPTY(s), 1); }
        for (int s = 0; s < kRawStages; s++) { mbar_init(RAWFULL(s), 1); mbar_init(RAWEMPTY(s), 4); }
        for (int b = 0; b < 2; b++) { mbar_init(SFULL(b), 1); mbar_init(SEMPTY(b), PAIRED ? 16 : 8); }
        mbar_init(DRAIN, 1);
        *sAbort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 10) {
        if constexpr (PAIRED) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(sTmem)), "r"(p.columns) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            tmem_alloc(smem_u32(sTmem), p.columns);
        }
    }
    fence_proxy_async();
    tc_fence_before();
    __syncthreads();
    if constexpr (PAIRED) cluster_sync();                // the partner's barriers and tensor memory are set up as well
    tc_fence_after();
    const uint32_t tmem = *sTmem;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // (not before the allocation: see bconv_umma_pre.cuh)
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const typename std::conditional<PAIRED, PairWait, WsWait>::type wait{sAbort, status};
    const uint32_t ring_col = (uint32_t)(p.accumulators * p.cols);
    // (one tile per cluster: its sets of sums, where there are several, are a chain each)
    const int chains = CHAINED ? (nkb + kChain - 1) / kChain : CLUSTER ? p.accumulators : 1, chain = nkb > 0 ? (nkb + chains - 1) / chains : 0;

    if (warp == 8 || warp == 9) {
        // =============================== loaders ============================================
        if (lane == 0 && nkb > 0) {
            const bool isw = warp == 8;
            const int step = BITS && isw ? 8 : 1, slots = BITS && isw ? kRawStages : p.stages;
            int s = 0, issued = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (int t = t_first; t < ntiles && ok; t += t_step) {
                int tm, tn;
                tile(t, tm, tn);
                for (int kb = 0; kb < nkb; kb += step) {
                    ok = wait(BITS && isw ? RAWEMPTY(s) : EMPTY(s), ph ^ 1);
                    if (!ok) break;
                    if (BITS && isw) {
                        mbar_expect_tx(RAWFULL(s), kRawStage);
                        tensor_g2s(smem_u32(sRaw) + s * kRawStage, map_w, (kb0 + kb) * 2, tn * n_of + n_own, RAWFULL(s));
                    } else {
                        const uint32_t bytes = isw ? kWStage : (uint32_t)own * 128u, dst = smem_u32(smem) + s * stage + (isw || BITS ? 0u : kWStage);
                        const int y = isw ? tn * n_of + n_own : tm * p.cols + (PAIRED ? (int)rank * own : 0);
                        if constexpr (PAIRED) {          // (rows past the end arrive as zeros, and count)
                            if (rank == 0) mbar_expect_tx(FULL(s), 2 * bytes);
                            tensor_g2s_pair(dst, isw ? map_w : map_x, (kb0 + kb) * 64, y, leader_address(FULL(s)));
                        } else {
                            mbar_expect_tx(FULL(s), bytes);
                            tensor_g2s(dst, isw ? map_w : map_x, (kb0 + kb) * 64, y, FULL(s));
                        }
                    }
                    issued++;
                    if (++s == slots) { s = 0; ph ^= 1; }
                }
            }
            if (!ok) {
                // giving up: wait (bounded) for the copies still in flight before the CTA exits (the second CTA of a pair,
                // whose copies complete on the other's barriers, lets the time of any copy pass)
                const bool here = !PAIRED || rank == 0 || (BITS && isw);
                for (int s2 = 0; s2 < slots; s2++) {
                    const bool this_pass = s2 < s;
                    if (!this_pass && issued < slots) continue;
                    for (int i = 0; i < (1 << 16); i++) {
                        if (here && mbar_try_wait(BITS && isw ? RAWFULL(s2) : FULL(s2), this_pass ? ph : ph ^ 1)) break;
                        __nanosleep(20);
                    }
                }
            }
        }
        __syncwarp();
    } else if (PAIRED && warp == 10 && rank == 1) {
        __syncwarp();                                    // (the leader issues for both)
    } else if (warp == 10) {
        // =============================== MMA issuer =========================================
        const uint32_t leader = elect_one() ? 1u : 0u;
        const uint32_t idesc = idesc_16(a.type, PAIRED ? 256 : 128, p.cols);
        const uint64_t desc0 = swizzled_desc(smem_u32(smem));
        const uint32_t hi = (uint32_t)(desc0 >> 32), lo0 = (uint32_t)desc0;
        int s = 0, r = 0, b = 0;
        uint32_t ph = 0, rph = 0, bph = 0, ready = 0;
        bool ok = true;
        if (nkb > 0)
            for (int t = t_first; t < ntiles && ok; t += t_step) {
                for (int k0 = 0; k0 < nkb && ok; k0 += chain) {          // (one turn where sums are not chained)
                    if (CHAINED || !CLUSTER) ok = wait.spin(SEMPTY(b), bph ^ 1);
                    if (!ok) break;
                    const uint32_t d = tmem + b * p.cols;
                    const int k1 = min(nkb, k0 + chain);
                    for (int kb = k0; kb < k1; kb++) {
                        if (BITS && !(ready & 2u)) ok = wait.spin(RFULL(r), rph);
                        if (ok && !(ready & 1u)) ok = wait.spin(FULL(s), ph);
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t lo = lo0 + (s * stage >> 4), x = BITS ? tmem + ring_col + r * 32 : lo;
                        const uint32_t bar_e = EMPTY(s), bar_r = REMPTY(r), bar_c = kb + 1 != k1 ? 0u : CHAINED || !CLUSTER ? SFULL(b) : k1 == nkb ? SFULL(0) : 0u;
                        if (++s == p.stages) { s = 0; ph ^= 1; }
                        if (BITS && ++r == p.ring) { r = 0; rph ^= 1; }
                        ready = mma_64<BITS, PAIRED>(leader, d, x, BITS ? lo : lo + (kWStage >> 4), hi, idesc, kb > k0, FULL(s), ph, RFULL(r), rph,
                                                     bar_e, bar_r, bar_c);
                    }
                    if (++b == p.accumulators) { b = 0; bph ^= 1; }
                }
            }
        if (!ok && leader) {
            // giving up: the MMAs already issued must have finished before tensor memory is freed
            if constexpr (PAIRED)
                asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(DRAIN) : "memory");
            else
                mma_commit(DRAIN);
            for (int i = 0; i < (1 << 20); i++)
                if (PAIRED ? mbar_test_cluster(DRAIN, 0) : mbar_try_wait(DRAIN, 0)) break;
        }
        __syncwarp();
    } else if (BITS && warp >= 12) {
        // =============================== expanders ==========================================
        const int quad = warp & 3, row = quad * 32 + lane;
        const uint32_t minus = a.type == BF16 ? 0xBF80BF80u : 0xBC00BC00u, four = 4 * blockDim.z;
        const uint32_t dst0 = tmem + ((uint32_t)(quad * 32) << 16) + ring_col;
        int raw = 0, r = 0, before = -1;                 // before: the slot being stored
        uint32_t rawph = 0, rph = 0;
        bool ok = true;
        auto hand_over = [&]() {
            if (before < 0) return;
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(RFULL(before));
            before = -1;
        };
        if (nkb > 0)
            for (int t = t_first; t < ntiles && ok; t += t_step)
                for (int kb = 0; kb < nkb && ok; kb += 8) {
                    const int blocks = min(8, nkb - kb);
                    ok = wait(RAWFULL(raw), rawph);
                    if (!ok) break;
                    // (the copy's 64-byte swizzle: 16-byte pieces turned by the row)
                    const uint32_t src = smem_u32(sRaw) + raw * kRawStage + row * 64;
                    for (int j = 0; j < blocks; j++) {
                        uint32_t w0, w1, e[32];
                        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w0), "=r"(w1)
                                     : "r"(src + (((j >> 1) ^ ((row >> 1) & 3)) << 4) + (j & 1) * 8) : "memory");
                        expand_signs(w0, minus, four, e);      // (while the block in front is on its way)
                        expand_signs(w1, minus, four, e + 16);
                        hand_over();
                        ok = wait(REMPTY(r), rph ^ 1);
                        if (!ok) break;
                        tc_fence_after();
                        tmem_st32(dst0 + r * 32, e);
                        before = r;
                        if (++r == p.ring) { r = 0; rph ^= 1; }
                    }
                    hand_over();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(RAWEMPTY(raw));
                    if (++raw == kRawStages) { raw = 0; rawph ^= 1; }
                }
        __syncwarp();
    } else if (warp < 8) {
        // =============================== epilogue ===========================================
        const int quad = warp & 3, half = warp >> 2;
        int b = 0;
        uint32_t bph = 0;
        bool ok = true;
        auto give_back = [&](int of) {                   // this warp has what it needs of the sums
            tc_fence_before();
            __syncwarp();
            if (lane == 0) { if constexpr (PAIRED) mbar_arrive_leader(SEMPTY(of)); else mbar_arrive(SEMPTY(of)); }
        };
        auto put = [&](const auto& f, int c0, int quad) {    // sums for the cluster: [four columns][128 outputs][4]
            float4* dst = reinterpret_cast<float4*>(smem) + (size_t)(c0 >> 2) * 128 + quad * 32 + lane;
#pragma unroll
            for (int j = 0; j < (int)(sizeof(f) / 16); j++)
                if (c0 + 4 * j < p.cols) dst[j * 128] = make_float4(f[4 * j], f[4 * j + 1], f[4 * j + 2], f[4 * j + 3]);
        };
        for (int t = t_first; t < ntiles && ok; t += t_step) {
            int tm, tn;
            tile(t, tm, tn);
            const int n0 = tn * n_of + n_own + quad * 32;
            if constexpr (CHAINED) {
                // a warp's pieces of 16 tokens, two of every four (pieces of 32 spill)
                constexpr int PIECES = (CLUSTER ? kChainCols : kMaxCols) / 32;
                const Output<!CLUSTER> out(a, n0 + lane);
                const int cols = CLUSTER ? p.cols : min(p.cols, a.M - tm * p.cols);
                auto at = [&](int i) { return half * 32 + (i >> 1) * 64 + (i & 1) * 16; };
                float sum[PIECES][16];
#pragma unroll
                for (int i = 0; i < PIECES; i++)
#pragma unroll
                    for (int j = 0; j < 16; j++) sum[i][j] = 0.f;
                for (int k0 = 0; k0 < nkb; k0 += chain) {
                    ok = wait.relaxed(SFULL(b), bph);
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll
                    for (int i = 0; i < PIECES; i++) {
                        if (at(i) >= cols) break;
                        int v[16];
                        tmem_ld16(tmem + ((uint32_t)(quad * 32) << 16) + b * p.cols + at(i), v);
                        tmem_ld_wait16(v);
#pragma unroll
                        for (int j = 0; j < 16; j++) sum[i][j] += __int_as_float(v[j]);
                    }
                    give_back(b);
                    if (++b == p.accumulators) { b = 0; bph ^= 1; }
                }
                if (!ok) break;
#pragma unroll
                for (int i = 0; i < PIECES; i++) {
                    if (at(i) >= cols) break;
                    if constexpr (CLUSTER) put(sum[i], at(i), quad);
                    else out.finish(sum[i], tm * p.cols + at(i), min(16, cols - at(i)));
                }
                continue;
            }
            const uint32_t tcol = tmem + ((uint32_t)(quad * 32) << 16) + b * p.cols;
            if (!CLUSTER && a.out_type != FP32) {
                const Output16 out(a, smem_u32(sTurn) + warp * kTurn, n0);
                const int m0 = tm * p.cols, cols = min(p.cols, a.M - m0);
                const int n = (cols - half * 32 + 63) / 64;              // this warp's pieces of 32 tokens: every second one
                auto at = [&](int k) { return half * 32 + k * 64; };
                auto rows_of = [&](int k) { return min(32, cols - at(k)); };
                uint4 res[4];
                auto ask = [&](int k) { if (a.residual && k < n) out.ask(res, m0 + at(k), rows_of(k)); };
                ask(0);
                ok = wait.relaxed(SFULL(b), bph);
                if (!ok) break;
                tc_fence_after();
                if (n <= 0) give_back(b);
                for (int k = 0; k < n; k++) {
                    int lo[16], hi[16];
                    tmem_ld_16x256b_x4(tcol + at(k), lo);
                    tmem_ld_16x256b_x4(tcol + (16u << 16) + at(k), hi);
                    tmem_ld_wait();
                    if (k + 1 == n) give_back(b);        // (in front of the last piece's work)
                    out.finish(lo, hi, res, m0 + at(k), rows_of(k));
                    ask(k + 1);
                }
            } else {
                const Output<!CLUSTER> out(a, n0 + lane);
                if (nkb > 0) ok = wait.relaxed(SFULL(b), bph);
                if (!ok) break;
                tc_fence_after();
                for (int c0 = half * 32; c0 < p.cols; c0 += 64) {
                    const int m0 = tm * p.cols + c0;
                    if (!CLUSTER && m0 >= a.M) break;
                    int v[32];
                    tmem_ld32(tcol + c0, v);
                    tmem_ld_wait();
                    float f[32];
#pragma unroll
                    for (int j = 0; j < 32; j++) f[j] = nkb > 0 ? __int_as_float(v[j]) : 0.f;
                    if constexpr (CLUSTER) {
                        for (int i = 1; i * chain < nkb; i++)
#pragma unroll
                            for (int h = 0; h < 32; h += 16) {
                                int more[16];
                                tmem_ld16(tcol + i * p.cols + c0 + h, more);
                                tmem_ld_wait16(more);
#pragma unroll
                                for (int j = 0; j < 16; j++) f[h + j] += __int_as_float(more[j]);
                            }
                        put(f, c0, quad);
                    } else {
                        out.finish(f, m0, min(min(32, p.cols - c0), a.M - m0));
                    }
                }
            }
            if (CLUSTER || a.out_type == FP32) give_back(b);
            if (++b == p.accumulators) { b = 0; bph ^= 1; }
        }
    }
    tc_fence_before();
    if constexpr (CLUSTER) {
        // Tensor memory goes back before the CTAs wait for one another: one that holds some and waits for a peer that waits for some
        // on another SM, held by a kernel of another stream that does the same, could wait forever.
        __syncthreads();
        if (warp == 10) tmem_dealloc(tmem, p.columns);
        // One tile per cluster: every CTA finishes each nctas-th group of four columns.
        cluster_sync();
        if (warp < 8 && !*sAbort) {
            const int quad = warp & 3, half = warp >> 2;
            int tm, tn;
            tile(t_first, tm, tn);
            const Output<false> out(a, tn * 128 + quad * 32 + lane);
            const int cols = min(p.cols, a.M - tm * p.cols);
            const uint32_t src = smem_u32(smem) + (uint32_t)(quad * 32 + lane) * 16u;
            for (int c = 4 * ((int)rank + half * (int)nctas); c < cols; c += 8 * (int)nctas) {
                float4 part[8];
#pragma unroll
                for (uint32_t r = 0; r < 8; r++)
                    if (r < nctas) part[r] = ld_peer4(src + (uint32_t)c * 512u, r);
                float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (uint32_t r = 0; r < 8; r++)
                    if (r < nctas) { v[0] += part[r].x; v[1] += part[r].y; v[2] += part[r].z; v[3] += part[r].w; }
                out.finish(v, tm * p.cols + c, min(4, cols - c));
            }
            __syncwarp();
        }
        cluster_sync();                                  // nobody reads this CTA's sums any more
    }
    if constexpr (!CLUSTER) __syncthreads();
    if constexpr (PAIRED) {
        cluster_sync();                                  // nothing of the partner's reaches into this CTA any more
        if (warp == 10) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(p.columns) : "memory");
    } else if (!CLUSTER && warp == 10) {
        tmem_dealloc(tmem, p.columns);
    }
}

// Rows of K elements of 16 bits, any distance apart, copied to rows of a multiple of 8 elements (none where rows = 0)
struct Rows { const uint16_t* from; uint16_t* to; long long ld; int rows; };
__device__ __forceinline__ void repack(const Rows& x, const Rows& w, int K) {
    const int pieces = (K + 7) / 8;
    const long long of_x = (long long)x.rows * pieces, total = of_x + (long long)w.rows * pieces;
    for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < total; i += (long long)gridDim.x * blockDim.x) {
        const bool isw = i >= of_x;
        const long long j = isw ? i - of_x : i, r = j / pieces;
        const int k = (int)(j - r * pieces) * 8;
        const uint16_t* s = isw ? w.from + r * w.ld + k : x.from + r * x.ld + k;
        uint32_t v[4];
#pragma unroll
        for (int q = 0; q < 4; q++)
            v[q] = (k + 2 * q < K ? (uint32_t)s[2 * q] : 0u) | (k + 2 * q + 1 < K ? (uint32_t)s[2 * q + 1] << 16 : 0u);
        reinterpret_cast<uint4*>(isw ? w.to : x.to)[j] = make_uint4(v[0], v[1], v[2], v[3]);
    }
}

}  // namespace linear
}  // namespace tcbnn
