// Kernels and C ABI of the products of real-valued rows (linear.cuh) and of the scores (log_probs.cuh).
#include "../../include/tcbnn_b200.h"
#include <algorithm>
#include <cmath>
#include "host.cuh"
#include "bnn_layers.cuh"
#include "linear_small.cuh"
#include "log_probs.cuh"

using namespace tcbnn;

namespace {

__device__ int g_linear_status;      // 1 after a bounded wait inside k_linear gave up

template <bool BITS, int FORM, bool CHAINED>
__global__ void __launch_bounds__(BITS ? linear::kThreadsBits : linear::kThreadsDense, FORM == linear::SPLIT ? 2 : 1)
k_linear(linear::Args a, linear::Plan p, int* status, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x) {
    extern __shared__ __align__(128) unsigned char dyn_smem_linear[];
    linear::umma_cta<BITS, FORM, CHAINED>(a, p, &map_w, &map_x, status, dyn_smem_linear);
}
template <int RT, int T, bool BF>
__global__ void __launch_bounds__(32 * linear::small_warps(RT, T), 1) k_bit_linear_small(linear::Args a) {
    extern __shared__ __align__(16) float bit_linear_sums[];
    linear::bit_linear_small<RT, T, BF>(a, bit_linear_sums);
}
template <bool BF, bool WIDE>
__global__ void __launch_bounds__(32 * linear::kDenseWarps, 2) k_linear_small(linear::Args a) {
    __shared__ float sums[linear::kDenseWarps * 8 * 20];
    linear::linear_small<BF, WIDE>(a, sums);
}
__global__ void __launch_bounds__(256) k_repack(linear::Rows x, linear::Rows w, int K) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    linear::repack(x, w, K);
}

template <int TYPE, int NW, bool CLUSTER>
__global__ void __launch_bounds__(NW == 1 ? 256 : NW * 32, 32 / (NW == 1 ? 8 : NW)) k_log_probs(scores::Args a) {
    __shared__ scores::Shared<NW> shared[NW == 1 ? 8 : 1];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if constexpr (CLUSTER) {
        uint32_t n, r;
        asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(n));
        asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
        scores::row<TYPE, NW, true>(a, shared[0], blockIdx.x / n, r, n);
    } else {
        const int warp = NW == 1 ? threadIdx.x >> 5 : 0;
        const long long r = NW == 1 ? blockIdx.x * 8LL + warp : blockIdx.x;
        if (r < a.M) scores::row<TYPE, NW, false>(a, shared[warp], r, 0, 1);
    }
}

size_t type_bytes(int type) { return type == TCBNN_FP32 ? 4 : 2; }

// A matrix of `rows` rows of `width` bytes, `pitch` bytes apart
struct Block { uintptr_t at; long long rows, width, pitch; };
// whether two share no byte: neither their extents, nor, with rows equally far apart, their columns
bool apart(const Block& a, const Block& b) {
    const uintptr_t a_end = a.at + (a.rows - 1) * a.pitch + a.width, b_end = b.at + (b.rows - 1) * b.pitch + b.width;
    if (a_end <= b.at || b_end <= a.at) return true;
    if (a.pitch != b.pitch && a.rows > 1 && b.rows > 1) return false;
    const long long pitch = a.rows > 1 ? a.pitch : b.pitch;
    if (a.rows == 1 && b.rows == 1) return false;
    long long off = (long long)(b.at - a.at) % pitch;
    if (off < 0) off += pitch;
    return off >= a.width && off + b.width <= pitch;
}

int check_linear(const char* what, const linear::Args& a, bool bits) {
    if (a.M < 0 || a.N < 1 || a.K < 1) return fail("%s: M >= 0, N and K >= 1", what);
    // (the largest K keeps a tile's time far inside the waits' limits)
    if (a.M > 1 << 30 || a.N > 1 << 30 || a.K > 1 << 24) return fail("%s: M and N up to 2^30, K up to 2^24", what);
    const long long far = 1LL << 40;
    if (a.ldx > far || a.ldw > far || a.ldo > far || (a.residual && a.ldr > far)) return fail("%s: leading dimensions up to 2^40", what);
    if (a.type != TCBNN_FP16 && a.type != TCBNN_BF16) return fail("%s: x is fp16 or bf16", what);
    if (a.out_type != a.type && a.out_type != TCBNN_FP32) return fail("%s: the result is of x's type or fp32", what);
    if (a.bias_type != a.type && a.bias_type != TCBNN_FP32) return fail("%s: the bias is of x's type or fp32", what);
    if (a.activation < 0 || a.activation > TCBNN_SILU) return fail("%s: unknown activation %d", what, a.activation);
    if (!a.W || (a.M > 0 && (!a.x || !a.out))) return fail("%s: null pointer", what);
    if (a.ldx < a.K || a.ldo < a.N || (a.residual && a.ldr < a.N)) return fail("%s: rows closer together than they are long", what);
    const int eb = (int)type_bytes(a.type), ob = (int)type_bytes(a.out_type);
    if (bits) {
        if ((a.ldw & 3) || a.ldw * 32 < a.K) return fail("%s: ldw must be a multiple of 4 words and cover K", what);
        if ((uintptr_t)a.W & 15) return fail("%s: packed weights must be 16-byte aligned", what);
        if ((uintptr_t)a.scale & 3) return fail("%s: the scale is not aligned to its type", what);
    } else if (a.ldw < a.K) {
        return fail("%s: rows closer together than they are long", what);
    }
    if (((uintptr_t)a.x | (bits ? 0 : (uintptr_t)a.W)) % eb || ((uintptr_t)a.out | (uintptr_t)a.residual) % ob || (uintptr_t)a.bias % type_bytes(a.bias_type))
        return fail("%s: a pointer is not aligned to its type", what);
    if (a.M == 0) return 0;
    const Block x{(uintptr_t)a.x, a.M, (long long)a.K * eb, a.ldx * eb}, out{(uintptr_t)a.out, a.M, (long long)a.N * ob, a.ldo * ob};
    const Block w = bits ? Block{(uintptr_t)a.W, a.N, a.ldw * 4, a.ldw * 4} : Block{(uintptr_t)a.W, a.N, (long long)a.K * eb, a.ldw * eb};
    if (!apart(x, out) || !apart(w, out)) return fail("%s: the result overlaps x or the weights", what);
    if (a.bias && !apart(Block{(uintptr_t)a.bias, 1, (long long)(a.N * type_bytes(a.bias_type)), (long long)(a.N * type_bytes(a.bias_type))}, out))
        return fail("%s: the result overlaps the bias", what);
    if (a.scale && !apart(Block{(uintptr_t)a.scale, 1, 4LL * a.N, 4LL * a.N}, out)) return fail("%s: the result overlaps the scale", what);
    if (a.residual && !(a.residual == a.out && a.ldr == a.ldo) && !apart(Block{(uintptr_t)a.residual, a.M, (long long)a.N * ob, a.ldr * ob}, out))
        return fail("%s: the residual overlaps the result without being it", what);
    return 0;
}

// Operands that tensor copies can read: rows that start on multiples of 16 bytes (less than 2^40 bytes apart)
bool rows_fit(const void* p, long long ld, int rows) {
    return ((uintptr_t)p & 15) == 0 && (rows == 1 || ((ld & 7) == 0 && ld < (1LL << 39)));
}
double bytes_to_copy(const void* x, const void* W, int M, int N, int K, long long ldx, long long ldw) {
    return 2.0 * K * ((rows_fit(x, ldx, M) ? 0 : M) + (!W || rows_fit(W, ldw, N) ? 0 : N));
}
size_t packed_bytes(int rows, int K) { return ((size_t)rows * ((K + 7) & ~7) * 2 + 255) & ~(size_t)255; }

// What is copied is written while other operands are read and results stored.
int check_workspace(const char* what, const linear::Args& a, bool bits, const void* workspace) {
    const bool move_x = !rows_fit(a.x, a.ldx, a.M), move_w = !bits && !rows_fit(a.W, a.ldw, a.N);
    if (!workspace || (!move_x && !move_w)) return 0;
    const long long eb = (long long)type_bytes(a.type), ob = (long long)type_bytes(a.out_type), bb = (long long)type_bytes(a.bias_type);
    const long long used = (long long)((move_x ? packed_bytes(a.M, a.K) : 0) + (move_w ? packed_bytes(a.N, a.K) : 0));
    const Block room{(uintptr_t)workspace, 1, used, used};
    const Block of[] = {{(uintptr_t)a.x, a.M, a.K * eb, a.ldx * eb}, {(uintptr_t)a.W, a.N, bits ? a.ldw * 4 : a.K * eb, bits ? a.ldw * 4 : a.ldw * eb},
                        {(uintptr_t)a.bias, 1, a.N * bb, a.N * bb}, {(uintptr_t)a.scale, 1, 4LL * a.N, 4LL * a.N},
                        {(uintptr_t)a.residual, a.M, a.N * ob, a.ldr * ob}, {(uintptr_t)a.out, a.M, a.N * ob, a.ldo * ob}};
    for (const Block& b : of)
        if (b.at && !apart(b, room)) return fail("%s: the workspace overlaps an operand or the result", what);
    return 0;
}

int g_linear_cols = 0, g_linear_splits = 0;              // tcbnn_set_linear_plan: 0 = from the model

// What a plan takes, in us at 1.9 GHz, fitted to 1400 forced plans over 22 shapes: the set-up of a launch, of a cluster's exchange, of a
// pair; a wave of tiles, each its blocks of 64 of K -- MMAs of cols / 2 clocks, or the bytes that a CTA draws from L2, or its
// expanders -- and an epilogue that the next tile's blocks hide but for a share; no less than the operands' way from memory.
double plan_time(const linear::Plan& p, int M, int N, int K, int sms) {
    struct Fit { double start, split[4], pair, clocks, bytes, block, finish, column, shown, memory; };
    static const Fit of[2] = {{2.2, {0, 3.0, 2.0, 1.7}, 1.4, 1.03, 72, 0, 2590, 30, 0.36, 5800},
                              {3.6, {0, 2.2, 1.9, 1.5}, 0, 1.03, 59, 500, 1760, 24, 0.44, 4700}};
    const Fit& f = of[p.bits];
    const bool pair = p.form == linear::PAIR;
    const double tiles = (double)p.tiles_m * p.tiles_n, bytes = (p.bits ? 1024 : 16384) + linear::own_cols(p) * 128.0;
    double waves = ceil(tiles * p.splits / (pair ? sms / 2 : sms)), block = 2.0 * p.cols * f.clocks;
    if (block < bytes / f.bytes) block = bytes / f.bytes;
    if (p.splits > 1 && waves > 1) {                     // (two CTAs share an SM, but not each other's latency)
        block *= 2;
        waves = ceil(waves / 2);
    }
    if (block < f.block) block = f.block;
    const double finish = f.finish + f.column * p.cols, blocks = p.per < p.kblocks ? p.per : p.kblocks;
    const double clocks = waves * (blocks * block + finish * (p.accumulators == 1 ? 1 : f.shown)) + (p.accumulators == 1 ? 0 : finish);
    const double weight = p.bits ? N * (K / 8.0) : 2.0 * N * K;
    const double memory = (weight + 2.0 * M * K + 2.0 * M * N) / (f.memory * 1e3);
    return (clocks / 1900 > memory ? clocks / 1900 : memory) + f.start + (pair ? f.pair : f.split[p.splits == 8 ? 3 : p.splits / 2]);
}

// The plan that takes least.  exact: for fp32 results, whose sums are chained (dense weights)
linear::Plan make_plan(int M, int N, int K, bool bits, bool exact, int sms) {
    linear::Plan best = {};
    double least = 1e300;
    const int kblocks = (K + 63) / 64, unit = bits ? 8 : 1;
    for (int shape = 0; shape < (bits ? 4 : 5); shape++) {               // K in 1, 2, 4, 8; pairs of CTAs
        const bool pair = shape == 4;
        const int splits = pair ? 1 : 1 << shape;
        if (g_linear_splits && g_linear_splits != (pair ? -2 : splits)) continue;
        const int per = ((kblocks + splits - 1) / splits + unit - 1) / unit * unit;
        if (splits > 1 && (splits - 1) * per >= kblocks && !g_linear_splits) continue;       // (a CTA without work)
        for (int cols = pair ? 32 : 16; cols <= linear::kMaxCols; cols += pair ? 32 : 16) {
            linear::Plan p = {};
            p.bits = bits;
            p.form = pair ? linear::PAIR : splits > 1 ? linear::SPLIT : linear::ALONE;
            if (bits && splits > 1 && cols > 128) continue;
            p.cols = cols;
            p.splits = splits;
            p.tiles_m = (M + cols - 1) / cols;
            p.tiles_n = pair ? (N + 255) / 256 : (N + 127) / 128;
            const long long tiles = (long long)p.tiles_m * p.tiles_n;
            if (splits > 1 && tiles * splits > (g_linear_splits ? 1 << 20 : 3LL * sms)) continue;      // (as far as the times were fitted)
            if (g_linear_cols ? cols != g_linear_cols : cols > 32 && cols >= M + 32) continue;
            const int chains = exact && !bits ? (per + linear::kChain - 1) / linear::kChain : 1;
            const bool apart = splits > 1 && (chains - 1) * cols + ((cols + 31) & ~31) <= 256;         // (a set of sums for each)
            p.chained = chains > 1 && !apart;
            if (p.chained && splits > 1 && cols > linear::kChainCols) {      // (no such kernel)
                if (!g_linear_cols) continue;
                p.chained = 0;
            }
            p.kblocks = kblocks;
            p.per = per;
            p.band = cols >= 128 ? 8 : 1024 / cols;
            // a second set of sums where there is room, and a second tile or chain
            p.accumulators = apart ? chains : !p.chained && (tiles <= (pair ? sms / 2 : sms) || p.form == linear::SPLIT || (bits && cols > 192)) ? 1 : 2;
            p.ring = !bits ? 0 : ((p.form == linear::SPLIT ? 256 : 512) - p.accumulators * cols) / 32;
            if (p.ring > linear::kMaxRing) p.ring = linear::kMaxRing;
            // (the epilogue reads 32 columns at a time of each set, the last of an odd multiple of 16 with 16 behind it)
            const int used = p.accumulators * cols + 32 * p.ring, read = (p.accumulators - 1) * cols + ((cols + 31) & ~31);
            p.columns = 32;
            while (p.columns < used || p.columns < read) p.columns *= 2;
            // A CTA of a cluster leaves room for one of the launch behind it, which is set up meanwhile.
            const size_t room = (p.form == linear::SPLIT ? 113 : 227) * 1024;
            for (p.stages = linear::kMaxStages; p.stages > 2 && linear::smem_bytes(p) > room; p.stages--) {}
            // (two stages of 43 KB and more, or sums of 112 KB and more to exchange: 224 x 4096 -> 4096 33.5 us, with three stages 13.9; 566 x 3560
            // -> 1504 26.9 and 24.8)
            if (splits > 1 && p.stages < 3 && !g_linear_cols) continue;
            const double t = plan_time(p, M, N, K, sms);
            if (t < least) { least = t; best = p; }
        }
    }
    return best;
}

// (The last plans of this thread: the search takes a microsecond.)
const linear::Plan& plan_linear(int M, int N, int K, bool bits, bool exact, int sms) {
    struct Kept { int M, N, K, bits, exact, sms, cols, splits; linear::Plan plan; };
    static thread_local Kept kept[64];
    Kept& k = kept[((unsigned)M * 2654435761u ^ (unsigned)N * 40503u ^ (unsigned)K * 2246822519u ^ (unsigned)bits * 128 ^ (unsigned)exact * 256) >> 7 & 63];
    if (k.M != M || k.N != N || k.K != K || k.bits != (int)bits || k.exact != (int)exact || k.sms != sms || k.cols != g_linear_cols || k.splits != g_linear_splits)
        k = Kept{M, N, K, (int)bits, (int)exact, sms, g_linear_cols, g_linear_splits, make_plan(M, N, K, bits, exact, sms)};
    return k.plan;
}

// What the launch that copies operands in front of the product takes
double copy_time(double bytes) { return bytes > 0 ? 2.3 + bytes * 0.36e-6 : 0; }
// How k_bit_linear_small runs: 16 x rt outputs and 8 x groups rows per block, on that many warps.
struct SmallPlan { int rt, groups, warps; double us; };
// The plan of least estimated time, in us at 1.9 GHz; its numbers were fitted to 822 times over 20 weights and 1 to 128 rows, and its
// choice is 0.8 % from the best one on average (20 % at most).  A block whose SM has nothing else takes all the warps that fit, others
// half of those, two to an SM; a warp's piece of 128 elements is paid in expansions and MMAs per 16 outputs and loads per eight rows (more of
// them where rows start on any element), or waits for its words; then the block's sums meet.
SmallPlan small_plan(int M, int N, int K, bool anywhere, int sms) {
    static const int of[][2] = {{1, 1}, {1, 2}, {1, 3}, {2, 1}, {2, 2}, {2, 3}, {2, 4}, {4, 1}};
    SmallPlan best = {0, 0, 0, 1e300};
    const int rows = (M + 7) / 8, pieces = (K + 127) / 128;
    for (const auto& f : of) {
        const int rt = f[0], groups = f[1];
        if (groups > rows) continue;
        const int most = linear::small_warps(rt, groups);
        const long long blocks = (long long)((N + 16 * rt - 1) / (16 * rt)) * ((rows + groups - 1) / groups);
        const int warps = blocks <= sms ? most : 8, busy = warps < pieces ? warps : pieces, at_once = warps > 8 || most < 16 ? 1 : 2;
        const double piece = rt * (146 + 25.0 * groups) + groups * (anywhere ? 267 : 121) + 9;
        const double turns = (pieces + busy - 1) / busy, outputs = rt * groups * (4.0 * rt * groups > warps ? 4.0 * rt * groups / warps : 1) * busy / 16;
        const auto wave = [&](int resident) {
            const double clocks = resident * busy / 4.0 * piece;
            return 1594 + turns * (clocks > 642 ? clocks : 642) + 186 * resident * outputs;
        };
        const long long full = blocks / (sms * at_once), rest = blocks % (sms * at_once);
        const double us = (2357 + full * wave(at_once) + (rest ? wave(rest > sms ? 2 : 1) : 0)) / 1900;
        if (us < best.us) best = SmallPlan{rt, groups, warps, us};
    }
    return best;
}

// Few rows: whether the kernels on warp-level MMAs are the faster ones, by estimates of both.  Packed weights: 1 x 4096 -> 4096 4.0 us, the
// other kernel 8.7; 32 x 1000 -> 1000 2.6 and 7.3; 24 x 8192 -> 8192 15.6 and 17.1; 64 x 4096 -> 4096 15.0 and 11.1.  Dense ones: 2.1 us
// and their bytes at 5.7 TB/s for every eight rows, or a warp's pieces one after another, or 1.75 us for every wave of blocks (4096 x 4096
// for one row 8.3 us, 512 x 512 for 64 2.4, 4096 x 9216 for 16 25, 512 -> 50000 for one 20.4; the other kernel 9.4, 4.4, 16.4, 11.8); rows
// that start on any element at 2.6 TB/s (1 x 4097 -> 4096 15.0, 32 x 1001 -> 1000 5.1, copied first 22.5, 7.8).  copied: bytes that the
// other kernel needs copied.
bool small_pays(int M, int N, int K, bool bits, double copied, int sms) {
    if (M > 128 || g_linear_cols || g_linear_splits) return false;
    double us;
    if (bits) {
        us = small_plan(M, N, K, copied > 0 || (K & 7), sms).us;
    } else {
        const double bytes = (M + 7) / 8 * 2.0 * N * K * (copied > 0 ? 0.39e-6 : 0.175e-6), pieces = ceil(ceil(K / 128.0) / 8) * (copied > 0 ? 0.8 : 0.55);
        const double blocks = (N + 15) / 16 * (double)((M + 7) / 8), waves = blocks > 2 * sms ? 1.75 * blocks / (2 * sms) : 0;
        us = 2.1 + std::max(waves, std::max(bytes, pieces));
    }
    return us < plan_time(plan_linear(M, N, K, bits, false, sms), M, N, K, sms) + copy_time(copied);
}

// A launch of few rows' kernel: outputs x rows
int launch_small(void (*kernel)(linear::Args), const linear::Args& a, int outputs, int rows, int threads, size_t smem, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((a.N + outputs - 1) / outputs, (a.M + rows - 1) / rows);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
    return e != cudaSuccess ? fail("linear: %s", cudaGetErrorString(e)) : 0;
}

int linear_map(CUtensorMap* map, const void* base, CUtensorMapDataType type, int width, int rows, long long pitch_bytes, int box_x, int box_y,
               CUtensorMapSwizzle swizzle) {
    if (!tensor_encode()) return fail("linear: the driver has no cuTensorMapEncodeTiled");
    if (rows == 1) pitch_bytes = ((long long)width * (type == CU_TENSOR_MAP_DATA_TYPE_UINT32 ? 4 : 2) + 15) & ~15LL;
    const cuuint64_t dims[2] = {(cuuint64_t)width, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)pitch_bytes};
    const cuuint32_t box[2] = {(cuuint32_t)box_x, (cuuint32_t)box_y}, steps[2] = {1, 1};
    const CUresult e = tensor_encode()(map, type, 2, const_cast<void*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                                       CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (e != CUDA_SUCCESS) return fail("linear: tensor map of %d rows of %d: error %d", rows, width, (int)e);
    return 0;
}

int launch_linear(const linear::Args& a, const linear::Plan& p, int sms, const CUtensorMap& map_w, const CUtensorMap& map_x, cudaStream_t st) {
    using namespace linear;
    using Kernel = void (*)(Args, Plan, int*, CUtensorMap, CUtensorMap);
    static const struct { bool bits; int form; bool chained; Kernel kernel; } of[] = {
        {false, ALONE, false, k_linear<false, ALONE, false>}, {false, SPLIT, false, k_linear<false, SPLIT, false>},
        {false, PAIR, false, k_linear<false, PAIR, false>}, {false, ALONE, true, k_linear<false, ALONE, true>},
        {false, SPLIT, true, k_linear<false, SPLIT, true>}, {false, PAIR, true, k_linear<false, PAIR, true>},
        {true, ALONE, false, k_linear<true, ALONE, false>}, {true, SPLIT, false, k_linear<true, SPLIT, false>}};
    static bool done[64];
    static int* status_of[64];
    int dev = 0;
    cudaGetDevice(&dev);
    if (configure_once(done, [&] {
            cudaError_t e = cudaSuccess;
            for (const auto& k : of)
                if (e == cudaSuccess) e = cudaFuncSetAttribute(k.kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
            return e != cudaSuccess ? e : cudaGetSymbolAddress((void**)&status_of[dev & 63], g_linear_status);
        })) return 1;
    int i = 0;
    while (of[i].bits != (bool)p.bits || of[i].form != p.form || of[i].chained != (bool)p.chained) i++;
    const long long tiles = (long long)p.tiles_m * p.tiles_n;
    const int team = p.form == PAIR ? 2 : p.splits;
    const long long teams = p.form == SPLIT || tiles < sms / team ? tiles : sms / team;
    const cudaError_t e = launch_dependent_cluster(of[i].kernel, (unsigned)(teams * team), team > 1 ? team : 0, p.bits ? kThreadsBits : kThreadsDense, smem_bytes(p), st,
                                                   a, p, status_of[dev & 63], map_w, map_x);
    if (e != cudaSuccess) return fail("linear: %s", cudaGetErrorString(e));
    return 0;
}

int run_bit_linear_small(const linear::Args& a, int sms, cudaStream_t st) {
    using namespace linear;
    using Kernel = void (*)(Args);
    static const struct { int rt, groups; Kernel bf16, fp16; } of[] = {
#define TCBNN_SMALL(RT, T) {RT, T, k_bit_linear_small<RT, T, true>, k_bit_linear_small<RT, T, false>}
        TCBNN_SMALL(1, 1), TCBNN_SMALL(1, 2), TCBNN_SMALL(1, 3), TCBNN_SMALL(2, 1), TCBNN_SMALL(2, 2),
        TCBNN_SMALL(2, 3), TCBNN_SMALL(2, 4), TCBNN_SMALL(4, 1)};
#undef TCBNN_SMALL
    static bool done[64];
    if (configure_once(done, [] {
            cudaError_t e = cudaSuccess;
            for (const auto& k : of)
                for (Kernel f : {k.bf16, k.fp16})
                    if (e == cudaSuccess)
                        e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)small_bytes(k.rt, k.groups, small_warps(k.rt, k.groups)));
            return e;
        })) return 1;
    const SmallPlan p = small_plan(a.M, a.N, a.K, !rows_fit(a.x, a.ldx, a.M) || (a.K & 7), sms);
    int i = 0;
    while (of[i].rt != p.rt || of[i].groups != p.groups) i++;
    const int pieces = (a.K + 127) / 128;
    return launch_small(a.type == TCBNN_BF16 ? of[i].bf16 : of[i].fp16, a, 16 * p.rt, 8 * p.groups, 32 * p.warps,
                        small_bytes(p.rt, p.groups, pieces < p.warps ? pieces : p.warps), st);
}

int run_linear_small(const linear::Args& a, cudaStream_t st) {
    using namespace linear;
    const bool wide = rows_fit(a.x, a.ldx, a.M) && rows_fit(a.W, a.ldw, a.N);
    auto kernel = a.type == TCBNN_BF16 ? wide ? k_linear_small<true, true> : k_linear_small<true, false>
                                       : wide ? k_linear_small<false, true> : k_linear_small<false, false>;
    return launch_small(kernel, a, 16, 8, 32 * kDenseWarps, 0, st);
}

int run_linear(const char* what, linear::Args a, bool bits, void* workspace, size_t workspace_bytes, cudaStream_t st) {
    if (check_linear(what, a, bits)) return 1;
    if (a.M == 0) return 0;
    if (check_workspace(what, a, bits, workspace)) return 1;
    int sms;
    if (sm_count(&sms)) return 1;
    const double copied = bytes_to_copy(a.x, bits ? nullptr : a.W, a.M, a.N, a.K, a.ldx, a.ldw);
    if (small_pays(a.M, a.N, a.K, bits, copied, sms)) return bits ? run_bit_linear_small(a, sms, st) : run_linear_small(a, st);
    const size_t need = tcbnn_linear_workspace_bytes(a.x, bits ? nullptr : a.W, a.M, a.N, a.K, a.ldx, a.ldw);
    if (need) {
        if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 255))
            return fail("%s: these operands need %zu bytes of workspace, 256-byte aligned", what, need);
        char* room = (char*)workspace;
        linear::Rows moved[2] = {};
        long long units = 0;
        const auto move = [&](linear::Rows& m, const void** p, long long* ld, int rows) {
            m = linear::Rows{(const uint16_t*)*p, (uint16_t*)room, *ld, rows};
            *p = room;
            *ld = (a.K + 7) & ~7;
            room += packed_bytes(rows, a.K);
            units += (long long)rows * ((a.K + 7) / 8);
        };
        if (!rows_fit(a.x, a.ldx, a.M)) move(moved[0], &a.x, &a.ldx, a.M);
        if (!bits && !rows_fit(a.W, a.ldw, a.N)) move(moved[1], &a.W, &a.ldw, a.N);
        const long long blocks = (units + 255) / 256;
        const cudaError_t e = launch_dependent(k_repack, (unsigned)(blocks < 16LL * sms ? blocks : 16LL * sms), 256, 0, st, moved[0], moved[1], a.K);
        if (e != cudaSuccess) return fail("%s: %s", what, cudaGetErrorString(e));
    }
    const linear::Plan& p = plan_linear(a.M, a.N, a.K, bits, a.out_type == TCBNN_FP32, sms);
    if (!p.cols) return fail("%s: the forced plan does not exist for these operands", what);
    const CUtensorMapDataType type = a.type == TCBNN_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    CUtensorMap map_w, map_x;
    if (linear_map(&map_x, a.x, type, a.K, a.M, a.ldx * 2, 64, linear::own_cols(p), CU_TENSOR_MAP_SWIZZLE_128B)) return 1;
    if (bits ? linear_map(&map_w, a.W, CU_TENSOR_MAP_DATA_TYPE_UINT32, (a.K + 31) / 32, a.N, a.ldw * 4, 16, 128, CU_TENSOR_MAP_SWIZZLE_64B)
             : linear_map(&map_w, a.W, type, a.K, a.N, a.ldw * 2, 64, 128, CU_TENSOR_MAP_SWIZZLE_128B)) return 1;
    return launch_linear(a, p, sms, map_w, map_x, st);
}

int g_scores_warps = 0, g_scores_ctas = 0;               // tcbnn_set_log_probs_plan: 0 = from the sizes

// How many warps share a row.  As many as bring 32 to every SM, but no more than find a batch each; at least so many that a warp has
// eight batches at most, that the vectors read once more (the share top / threads of the row) stay few, and, for more than 16
// alternatives, that a bound from 32 maxima is not the least of them.  One warp, 2, 4, 8: 8192 x 1000 fp32 with 5 alternatives 13.4,
// 21, 30, 53 us, with 32 71, 30, 39, 69; 2000 x 8000 bf16 21.8, 16.1, 15.1, 18.9; 500 x 4000 fp32 11.5, 8.4, 7.0, 6.1; 4096 x 50001 bf16
// 168, 116, 91, 92.  Clusters of CTAs only where warps that find two batches are still wanted, as they cost 1 to 3 us: 256 x 50257 fp16
// 21.2 us alone, 16.7 in pairs, 22.2 in fours; 300 x 32000 fp32 12.9, 17.7, 21; 1 x 131072 bf16 15.1, 10.8, 7.7, 6.5 in eights.
template <int TYPE>
int run_log_probs(const scores::Args& a, int sms, cudaStream_t st) {
    const int per = 4 * scores::Element<TYPE>::kPer;
    const long long batches = (a.V + 32LL * per - 1) / (32 * per);
    const double want = 32.0 * sms / a.M, most = (double)batches;
    double need = want < most ? want : most;
    if (need < most / 8) need = most / 8;
    if (need < a.top * most / 64) need = a.top * most / 64;
    if (a.top > 16 && need < 2) need = 2;
    int warps = 1, ctas = 1;
    while (warps < 8 && warps < need) warps *= 2;
    while (warps == 8 && ctas < 8 && most >= 32.0 * ctas && want >= 16.0 * ctas) ctas *= 2;
    if (g_scores_warps) { warps = g_scores_warps; ctas = g_scores_ctas; }
    const auto go = [&](auto kernel) {
        const unsigned grid = warps == 1 ? (unsigned)((a.M + 7LL) / 8) : (unsigned)a.M * ctas, threads = warps == 1 ? 256 : 32 * warps;
        const cudaError_t e = launch_dependent_cluster(kernel, grid, ctas > 1 ? ctas : 0, threads, 0, st, a);
        return e != cudaSuccess ? fail("log_probs: %s", cudaGetErrorString(e)) : 0;
    };
    if (ctas > 1) return go(k_log_probs<TYPE, 8, true>);
    return warps == 1 ? go(k_log_probs<TYPE, 1, false>) : warps == 2 ? go(k_log_probs<TYPE, 2, false>)
         : warps == 4 ? go(k_log_probs<TYPE, 4, false>) : go(k_log_probs<TYPE, 8, false>);
}

}  // namespace

extern "C" {

size_t tcbnn_linear_workspace_bytes(const void* x, const void* W, int M, int N, int K, long long ldx, long long ldw) {
    int sms;
    if (M < 1 || N < 1 || K < 1) return 0;
    const double copied = bytes_to_copy(x, W, M, N, K, ldx, ldw);
    if (copied == 0 || (!sm_count(&sms) && small_pays(M, N, K, !W, copied, sms))) return 0;
    return (rows_fit(x, ldx, M) ? 0 : packed_bytes(M, K)) + (!W || rows_fit(W, ldw, N) ? 0 : packed_bytes(N, K));
}

int tcbnn_linear(const void* x, const void* W, const void* bias, const void* residual, void* out, int M, int N, int K, long long ldx,
                 long long ldw, long long ldr, long long ldo, int type, int out_type, int bias_type, int activation, void* workspace,
                 size_t workspace_bytes, void* stream) {
    const linear::Args a{x, W, nullptr, bias, residual, out, M, N, K, ldx, ldw, ldr, ldo, type, out_type, bias_type, activation};
    return run_linear("linear", a, false, workspace, workspace_bytes, (cudaStream_t)stream);
}

int tcbnn_set_linear_plan(int cols, int splits) {
    if (cols < 0 || cols > linear::kMaxCols || cols % (splits == -2 ? 32 : 16) || (splits != -2 && (splits < 0 || splits > 8 || (splits & (splits - 1)))))
        return fail("set_linear_plan: cols is 0 or a multiple of 16 up to 256, splits is 0, 1, 2, 4 or 8, or -2 (pairs; cols a multiple of 32)");
    g_linear_cols = cols;
    g_linear_splits = splits;
    return 0;
}

int tcbnn_linear_plan(int M, int N, int K, int packed, int out_type, int sms, int* plan) {
    if (M < 1 || N < 1 || K < 1 || M > 1 << 30 || N > 1 << 30 || K > 1 << 24 || sms < 2 || !plan) return fail("linear_plan: M, N, K >= 1, sms >= 2");
    const linear::Plan& p = plan_linear(M, N, K, packed != 0, out_type == TCBNN_FP32, sms);
    if (!p.cols) return fail("linear_plan: the forced plan does not exist for these sizes");
    const int of[9] = {small_pays(M, N, K, packed != 0, 0, sms), p.form, p.cols, p.splits, p.accumulators, p.columns, p.stages, (int)linear::smem_bytes(p), p.chained};
    std::copy(of, of + 9, plan);
    return 0;
}

int tcbnn_linear_status(int* status) {
    if (!status) return fail("linear_status: null pointer");
    CUDA_TRY(cudaDeviceSynchronize());
    CUDA_TRY(cudaMemcpyFromSymbol(status, g_linear_status, sizeof(int)));
    if (*status) {                                       // reading a failure clears it
        const int zero = 0;
        CUDA_TRY(cudaMemcpyToSymbol(g_linear_status, &zero, sizeof(int)));
    }
    return 0;
}

int tcbnn_bit_linear(const void* x, const uint32_t* W, const float* scale, const void* bias, const void* residual, void* out, int M, int N,
                     int K, long long ldx, long long ldw, long long ldr, long long ldo, int type, int out_type, int bias_type,
                     int activation, void* workspace, size_t workspace_bytes, void* stream) {
    const linear::Args a{x, W, scale, bias, residual, out, M, N, K, ldx, ldw, ldr, ldo, type, out_type, bias_type, activation};
    return run_linear("bit_linear", a, true, workspace, workspace_bytes, (cudaStream_t)stream);
}

int tcbnn_set_log_probs_plan(int warps, int ctas) {
    const bool alone = ctas <= 1 && (warps == 1 || warps == 2 || warps == 4 || warps == 8), shared = (ctas == 2 || ctas == 4 || ctas == 8) && warps == 8;
    if (warps && !alone && !shared) return fail("set_log_probs_plan: 1, 2, 4 or 8 warps, or 2, 4 or 8 CTAs of 8 warps");
    g_scores_warps = warps;
    g_scores_ctas = ctas < 1 ? 1 : ctas;
    return 0;
}

int tcbnn_log_probs(const void* logits, int type, int M, int V, long long ld, const void* targets, int target_bytes, float temperature,
                    int top, float* logp, float* entropy, int64_t* top_ids, float* top_logp, void* stream) {
    if (M < 0 || V < 1 || V > 1 << 30) return fail("log_probs: M >= 0 and V >= 1, up to 2^30");
    if (type != TCBNN_FP32 && type != TCBNN_FP16 && type != TCBNN_BF16) return fail("log_probs: logits are fp32, fp16 or bf16");
    if (ld < V) return fail("log_probs: rows closer together than they are long");
    if (ld > 1LL << 40) return fail("log_probs: ld up to 2^40");
    if (targets && target_bytes != 4 && target_bytes != 8) return fail("log_probs: targets are int32 or int64");
    if (!(temperature >= 1e-30f && temperature <= 1e30f)) return fail("log_probs: the temperature must be between 1e-30 and 1e30");
    if (top < 0 || top > scores::kMaxTop || top > V) return fail("log_probs: top must be between 0 and %d and at most V", scores::kMaxTop);
    if (M == 0) return 0;
    if (!logits || (top && (!top_ids || !top_logp)) || (targets && !logp)) return fail("log_probs: null pointer");
    if ((uintptr_t)logits % type_bytes(type) || (targets && (uintptr_t)targets % target_bytes) || (((uintptr_t)logp | (uintptr_t)entropy) & 3) ||
        (top && (((uintptr_t)top_ids & 7) || ((uintptr_t)top_logp & 3))))
        return fail("log_probs: a pointer is not aligned to its type");
    const auto vector = [](const void* p, long long bytes) { return Block{(uintptr_t)p, 1, bytes, bytes}; };
    const Block of[] = {{(uintptr_t)logits, M, V * (long long)type_bytes(type), ld * (long long)type_bytes(type)}, vector(targets, (long long)M * target_bytes),
                        vector(targets ? logp : nullptr, 4LL * M), vector(entropy, 4LL * M), vector(top ? top_ids : nullptr, 8LL * M * top),
                        vector(top ? top_logp : nullptr, 4LL * M * top)};
    for (int i = 2; i < 6; i++)
        for (int j = 0; j < i; j++)
            if (of[i].at && of[j].at && !apart(of[j], of[i])) return fail("log_probs: results overlap the logits, the targets or one another");
    const scores::Args a{logits, targets, M, V, type, target_bytes, top, ld, 1.f / temperature, targets ? logp : nullptr, entropy,
                         (long long*)top_ids, top_logp};
    int sms;
    if (sm_count(&sms)) return 1;
    return type == TCBNN_FP32 ? run_log_probs<linear::FP32>(a, sms, (cudaStream_t)stream)
         : type == TCBNN_FP16 ? run_log_probs<linear::FP16>(a, sms, (cudaStream_t)stream)
                              : run_log_probs<linear::BF16>(a, sms, (cudaStream_t)stream);
}

}  // extern "C"
