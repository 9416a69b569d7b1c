// Kernels and C ABI of the products of real-valued rows (linear.cuh) and of the scores (log_probs.cuh).
#include "../../include/tcbnn_b200.h"
#include "host.cuh"
#include "linear.cuh"
#include "log_probs.cuh"

using namespace tcbnn;

namespace {

template <bool BITS>
__global__ void __launch_bounds__(256) k_linear_64(linear::Args a) { linear::tile_64<BITS>(a); }
__global__ void __launch_bounds__(256) k_log_probs_row(scores::Args a) { scores::row(a); }

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

int run_linear(const char* what, const linear::Args& a, bool bits, void* workspace, size_t workspace_bytes, cudaStream_t st) {
    if (check_linear(what, a, bits)) return 1;
    if (a.M == 0) return 0;
    const dim3 grid((a.N + 63) / 64, (a.M + 63) / 64);
    if (bits) k_linear_64<true><<<grid, 256, 0, st>>>(a);
    else k_linear_64<false><<<grid, 256, 0, st>>>(a);
    return launch_check(what);
}

}  // namespace

extern "C" {

size_t tcbnn_linear_workspace_bytes(const void* x, const void* W, int M, int N, int K, long long ldx, long long ldw) {
    (void)x; (void)W; (void)M; (void)N; (void)K; (void)ldx; (void)ldw;
    return 0;
}

int tcbnn_linear(const void* x, const void* W, const void* bias, const void* residual, void* out, int M, int N, int K, long long ldx,
                 long long ldw, long long ldr, long long ldo, int type, int out_type, int bias_type, int activation, void* workspace,
                 size_t workspace_bytes, void* stream) {
    const linear::Args a{x, W, nullptr, bias, residual, out, M, N, K, ldx, ldw, ldr, ldo, type, out_type, bias_type, activation};
    return run_linear("linear", a, false, workspace, workspace_bytes, (cudaStream_t)stream);
}

int tcbnn_bit_linear(const void* x, const uint32_t* W, const float* scale, const void* bias, const void* residual, void* out, int M, int N,
                     int K, long long ldx, long long ldw, long long ldr, long long ldo, int type, int out_type, int bias_type,
                     int activation, void* workspace, size_t workspace_bytes, void* stream) {
    const linear::Args a{x, W, scale, bias, residual, out, M, N, K, ldx, ldw, ldr, ldo, type, out_type, bias_type, activation};
    return run_linear("bit_linear", a, true, workspace, workspace_bytes, (cudaStream_t)stream);
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
    k_log_probs_row<<<M, 256, 0, (cudaStream_t)stream>>>(a);
    return launch_check("log_probs");
}

}  // extern "C"
