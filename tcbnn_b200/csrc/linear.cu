// Kernels and C ABI of the products of real-valued rows (linear.cuh) and of the scores (log_probs.cuh).
#include "../../include/tcbnn_b200.h"
#include <cmath>
#include "host.cuh"
#include "bnn_layers.cuh"
#include "linear_umma.cuh"
#include "log_probs.cuh"

using namespace tcbnn;

namespace {

__device__ int g_linear_status;      // 1 after a bounded wait inside k_linear gave up

template <bool BITS, int FORM>
__global__ void __launch_bounds__(BITS ? linear::kThreadsBits : linear::kThreadsDense, FORM == linear::SPLIT ? 2 : 1)
k_linear(linear::Args a, linear::Plan p, int* status, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x) {
    extern __shared__ __align__(128) unsigned char dyn_smem_linear[];
    linear::umma_cta<BITS, FORM>(a, p, &map_w, &map_x, status, dyn_smem_linear);
}
__global__ void __launch_bounds__(256) k_repack(const uint16_t* src, long long ld, int rows, int K, int pitch, uint16_t* dst) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // (the product waits before it reads)
    linear::repack(src, ld, rows, K, pitch, dst);
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
size_t packed_bytes(int rows, int K) { return ((size_t)rows * ((K + 7) & ~7) * 2 + 255) & ~(size_t)255; }

int g_linear_cols = 0, g_linear_splits = 0;              // tcbnn_set_linear_plan: 0 = from the model

// The plan with the least clocks.  A block of 64 of K costs a CTA its MMAs (cols / 2 each), its bytes from L2, or, with packed
// weights, the expanders' time; a tile its set-up and what of the epilogue shows; a cluster its exchange.
linear::Plan make_plan(int M, int N, int K, bool bits, int sms) {
    linear::Plan best = {};
    double least = 1e300;
    const int kblocks = (K + 63) / 64, unit = bits ? 8 : 1;
    for (int shape = 0; shape < 5; shape++) {
        const bool pair = shape == 4;
        const int splits = pair ? 1 : 1 << shape;
        if (g_linear_splits && g_linear_splits != (pair ? -2 : splits)) continue;
        const int per = ((kblocks + splits - 1) / splits + unit - 1) / unit * unit;
        if (splits > 1 && (splits - 1) * per >= kblocks && !g_linear_splits) continue;       // (a CTA without work)
        const int teams = pair || splits == 2 ? sms / 2 : splits == 1 ? sms : splits == 4 ? sms * 33 / 148 : sms * 15 / 148;
        for (int cols = pair ? 32 : 16; cols <= linear::kMaxCols; cols += pair ? 32 : 16) {
            linear::Plan p = {};
            p.form = pair ? linear::PAIR : splits > 1 ? linear::SPLIT : linear::ALONE;
            p.cols = cols;
            p.splits = splits;
            p.tiles_m = (M + cols - 1) / cols;
            p.tiles_n = pair ? (N + 255) / 256 : (N + 127) / 128;
            const long long tiles = (long long)p.tiles_m * p.tiles_n;
            if (splits > 1 && tiles * splits > (1 << 20)) continue;
            if (g_linear_cols ? cols != g_linear_cols : cols > 32 && cols >= M + 32) continue;
            p.kblocks = kblocks;
            p.per = per;
            p.band = cols >= 128 ? 8 : 1024 / cols;
            p.accumulators = tiles <= teams || (bits && cols > 192) ? 1 : 2;
            // A CTA of a cluster leaves room for one of the launch behind it, which is set up meanwhile.
            const bool half = p.form == linear::SPLIT;
            p.ring = (half ? 256 - cols > 128 ? 256 - cols : 128 : 512 - p.accumulators * cols) / 32;
            if (p.ring > linear::kMaxRing) p.ring = linear::kMaxRing;
            p.columns = 32;
            while (p.columns < p.accumulators * cols + (bits ? 32 * p.ring : 0)) p.columns *= 2;
            const int room = (half ? 113 : 227) * 1024;
            p.stages = (room - 2048 - 8 * (int)linear::kTurn - (bits ? linear::kRawStages * (int)linear::kRawStage : 0)) / (int)linear::stage_bytes(p, bits);
            if (p.stages > linear::kMaxStages) p.stages = linear::kMaxStages;
            if (p.stages < 2) p.stages = 2;
            while (p.stages > 2 && linear::smem_bytes(p, bits) > (size_t)room) p.stages--;
            if (linear::smem_bytes(p, bits) > 227 * 1024) continue;
            const double mma = 2.0 * cols, bytes = (bits ? 1024 : 16384) + linear::own_cols(p) * 128.0;
            double block = bytes / 72 > mma ? bytes / 72 : mma;
            if (bits && block < 130) block = 130;
            const double finish = 400 + cols * 12.0, waves = (double)((tiles + teams - 1) / teams);
            const double clocks = waves * (p.per * block + (p.accumulators == 1 ? finish : 200)) + finish + 2500 + (splits > 1 || pair ? 2000 : 0);
            if (clocks < least) { least = clocks; best = p; }
        }
    }
    return best;
}

// (The last plans of this thread: the search takes a microsecond.)
const linear::Plan& plan_linear(int M, int N, int K, bool bits, int sms) {
    struct Kept { int M, N, K, bits, sms, cols, splits; linear::Plan plan; };
    static thread_local Kept kept[64];
    Kept& k = kept[((unsigned)M * 2654435761u ^ (unsigned)N * 40503u ^ (unsigned)K * 2246822519u ^ (unsigned)bits) >> 7 & 63];
    if (k.M != M || k.N != N || k.K != K || k.bits != (int)bits || k.sms != sms || k.cols != g_linear_cols || k.splits != g_linear_splits)
        k = Kept{M, N, K, (int)bits, sms, g_linear_cols, g_linear_splits, make_plan(M, N, K, bits, sms)};
    return k.plan;
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

template <bool BITS>
int launch_linear(const linear::Args& a, const linear::Plan& p, int sms, const CUtensorMap& map_w, const CUtensorMap& map_x, cudaStream_t st) {
    static bool done[64];
    if (configure_once(done, [] {
            cudaError_t e = cudaFuncSetAttribute(k_linear<BITS, linear::ALONE>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
            if (e == cudaSuccess) e = cudaFuncSetAttribute(k_linear<BITS, linear::SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
            return e != cudaSuccess ? e : cudaFuncSetAttribute(k_linear<BITS, linear::PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
        })) return 1;
    void* status = nullptr;
    CUDA_TRY(cudaGetSymbolAddress(&status, g_linear_status));
    const long long tiles = (long long)p.tiles_m * p.tiles_n;
    const int threads = BITS ? linear::kThreadsBits : linear::kThreadsDense;
    const size_t smem = linear::smem_bytes(p, BITS);
    const int team = p.form == linear::PAIR ? 2 : p.splits;
    const long long teams = p.form == linear::SPLIT || tiles < sms / team ? tiles : sms / team;
    auto kernel = p.form == linear::ALONE ? k_linear<BITS, linear::ALONE> : p.form == linear::SPLIT ? k_linear<BITS, linear::SPLIT>
                                                                                                    : k_linear<BITS, linear::PAIR>;
    const cudaError_t e = launch_dependent_cluster(kernel, (unsigned)(teams * team), team > 1 ? team : 0, threads, smem, st, a, p, (int*)status,
                                                   map_w, map_x);
    if (e != cudaSuccess) return fail("linear: %s", cudaGetErrorString(e));
    return 0;
}

int run_linear(const char* what, linear::Args a, bool bits, void* workspace, size_t workspace_bytes, cudaStream_t st) {
    if (check_linear(what, a, bits)) return 1;
    if (a.M == 0) return 0;
    int sms;
    if (sm_count(&sms)) return 1;
    const size_t need = tcbnn_linear_workspace_bytes(a.x, bits ? nullptr : a.W, a.M, a.N, a.K, a.ldx, a.ldw);
    if (need) {
        if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 255))
            return fail("%s: these operands need %zu bytes of workspace, 256-byte aligned", what, need);
        char* room = (char*)workspace;
        const int pitch = (a.K + 7) & ~7;
        auto repack = [&](const void** p, long long* ld, int rows) {
            const long long units = (long long)rows * (pitch / 8), blocks = (units + 255) / 256;
            k_repack<<<(unsigned)(blocks < 16LL * sms ? blocks : 16LL * sms), 256, 0, st>>>((const uint16_t*)*p, *ld, rows, a.K, pitch, (uint16_t*)room);
            *p = room;
            *ld = pitch;
            room += packed_bytes(rows, a.K);
        };
        if (!rows_fit(a.x, a.ldx, a.M)) repack(&a.x, &a.ldx, a.M);
        if (!bits && !rows_fit(a.W, a.ldw, a.N)) repack(&a.W, &a.ldw, a.N);
        if (launch_check(what)) return 1;
    }
    const linear::Plan& p = plan_linear(a.M, a.N, a.K, bits, sms);
    const CUtensorMapDataType type = a.type == TCBNN_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    CUtensorMap map_w, map_x;
    if (linear_map(&map_x, a.x, type, a.K, a.M, a.ldx * 2, 64, linear::own_cols(p), CU_TENSOR_MAP_SWIZZLE_128B)) return 1;
    if (bits ? linear_map(&map_w, a.W, CU_TENSOR_MAP_DATA_TYPE_UINT32, (a.K + 31) / 32, a.N, a.ldw * 4, 16, 128, CU_TENSOR_MAP_SWIZZLE_64B)
             : linear_map(&map_w, a.W, type, a.K, a.N, a.ldw * 2, 64, 128, CU_TENSOR_MAP_SWIZZLE_128B)) return 1;
    return bits ? launch_linear<true>(a, p, sms, map_w, map_x, st) : launch_linear<false>(a, p, sms, map_w, map_x, st);
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
    if (M < 1 || N < 1 || K < 1) return 0;
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
    if (M < 0 || V < 1) return fail("log_probs: M >= 0 and V >= 1");
    if (type != TCBNN_FP32 && type != TCBNN_FP16 && type != TCBNN_BF16) return fail("log_probs: logits are fp32, fp16 or bf16");
    if (ld < V) return fail("log_probs: rows closer together than they are long");
    if (targets && target_bytes != 4 && target_bytes != 8) return fail("log_probs: targets are int32 or int64");
    if (!(temperature >= 1e-30f && temperature <= 1e30f)) return fail("log_probs: the temperature must be between 1e-30 and 1e30");
    if (top < 0 || top > scores::kMaxTop || top > V) return fail("log_probs: top must be between 0 and %d and at most V", scores::kMaxTop);
    if (M == 0) return 0;
    if (!logits || (top && (!top_ids || !top_logp)) || (targets && !logp)) return fail("log_probs: null pointer");
    if ((uintptr_t)logits % type_bytes(type) || (targets && (uintptr_t)targets % target_bytes) || (((uintptr_t)logp | (uintptr_t)entropy) & 3) ||
        (top && (((uintptr_t)top_ids & 7) || ((uintptr_t)top_logp & 3))))
        return fail("log_probs: a pointer is not aligned to its type");
    const scores::Args a{logits, targets, M, V, type, target_bytes, top, ld, 1.f / temperature, targets ? logp : nullptr, entropy,
                         (long long*)top_ids, top_logp};
    int sms;
    if (sm_count(&sms)) return 1;
    return type == TCBNN_FP32 ? run_log_probs<linear::FP32>(a, sms, (cudaStream_t)stream)
         : type == TCBNN_FP16 ? run_log_probs<linear::FP16>(a, sms, (cudaStream_t)stream)
                              : run_log_probs<linear::BF16>(a, sms, (cudaStream_t)stream);
}

}  // extern "C"
