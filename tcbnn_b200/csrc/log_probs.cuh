// Log probabilities from logits.  With d = (x - max x) / T and S = sum e^d over a row of V logits:
//   logp(target) = d(target) - ln S,   entropy = ln S - sum(e^d d) / S,   the `top` largest logits and their logp.
// A token of logit -inf is ruled out: probability 0, no alternative.  A row that rules out everything has logp
// -inf and entropy 0; one that holds NaN or +inf has NaN for both.  Alternatives are ordered by (logit, lowest token),
// NaN taking no part.
//
// This form reads a row once per block for the sums and once for every alternative.
#pragma once
#include "linear.cuh"

namespace tcbnn {
namespace scores {

constexpr int kMaxTop = 32;

struct Args {
    const void* logits; const void* targets;
    int M, V, type, target_bytes, top;
    long long ld;
    float inv_t;
    float* logp; float* entropy; long long* top_ids; float* top_logp;
};

// Order of the alternatives as one number: the larger, the earlier; 0: no alternative.
__device__ __forceinline__ unsigned long long key_of(float x, int token) {
    if (!(x > -INFINITY)) return 0ull;                 // ruled out, or NaN
    uint32_t u = __float_as_uint(x + 0.f);             // (-0 is 0)
    u ^= (u >> 31) ? 0xFFFFFFFFu : 0x80000000u;
    return ((unsigned long long)u << 32) | (0xFFFFFFFFu - (uint32_t)token);
}
__device__ __forceinline__ float logit_of(unsigned long long key) {
    uint32_t u = (uint32_t)(key >> 32);
    u ^= (u >> 31) ? 0x80000000u : 0xFFFFFFFFu;
    return __uint_as_float(u);
}
__device__ __forceinline__ int token_of(unsigned long long key) { return (int)(0xFFFFFFFFu - (uint32_t)key); }

// max m, sum e^{(x-m)/T} and sum e^{(x-m)/T} (x-m) of part of a row
struct Sums { float m, s, t; };
__device__ __forceinline__ void add(Sums& a, const Sums& b, float inv_t) {
    const float m = fmaxf(a.m, b.m);
    if (m == -INFINITY) { a.s += b.s; a.t += b.t; return; }              // (0, or NaN)
    // a part far below m has nothing to add, whatever its distance times its sums comes to (fp32's lowest as a mask)
    const float da = a.m - m, db = b.m - m, ea = expf(da * inv_t), eb = expf(db * inv_t);
    a.t = (ea == 0.f ? 0.f : ea * fmaf(a.s, da, a.t)) + (eb == 0.f ? 0.f : eb * fmaf(b.s, db, b.t));
    a.s = ea * a.s + eb * b.s;
    a.m = m;
}

__device__ __forceinline__ void row(const Args& a) {
    __shared__ Sums ss[256];
    __shared__ unsigned long long sk[256];
    const int r = blockIdx.x, t = threadIdx.x;
    const long long base = r * a.ld;
    Sums q{-INFINITY, 0.f, 0.f};
    for (int i = t; i < a.V; i += 256) {
        const float x = linear::load(a.logits, base + i, a.type);
        if (x != -INFINITY) add(q, Sums{x, x == x && x != INFINITY ? 1.f : NAN, 0.f}, a.inv_t);
    }
    ss[t] = q;
    __syncthreads();
    for (int h = 128; h; h >>= 1) {
        if (t < h) add(ss[t], ss[t + h], a.inv_t);
        __syncthreads();
    }
    const Sums all = ss[0];
    const float lse = logf(all.s);
    auto logp = [&](float x) { return x == -INFINITY ? (all.s == all.s ? -INFINITY : NAN) : fmaf(x - all.m, a.inv_t, -lse); };
    if (t == 0) {
        const bool none = all.m == -INFINITY && all.s == 0.f;
        if (a.logp) {
            const long long y = !a.targets ? -1 : a.target_bytes == 8 ? reinterpret_cast<const long long*>(a.targets)[r] : reinterpret_cast<const int*>(a.targets)[r];
            a.logp[r] = y < 0 ? 0.f : y >= a.V ? NAN : logp(linear::load(a.logits, base + y, a.type));
        }
        if (a.entropy) a.entropy[r] = none ? 0.f : lse - all.t / all.s * a.inv_t;
    }
    unsigned long long last = ~0ull;
    for (int k = 0; k < a.top; k++) {
        unsigned long long best = 0;
        for (int i = t; i < a.V; i += 256) {
            const unsigned long long key = key_of(linear::load(a.logits, base + i, a.type), i);
            if (key < last && key > best) best = key;
        }
        __syncthreads();
        sk[t] = best;
        __syncthreads();
        for (int h = 128; h; h >>= 1) {
            if (t < h && sk[t + h] > sk[t]) sk[t] = sk[t + h];
            __syncthreads();
        }
        last = sk[0];
        if (t == 0) {
            a.top_ids[(long long)r * a.top + k] = last ? token_of(last) : -1;
            a.top_logp[(long long)r * a.top + k] = logp(last ? logit_of(last) : -INFINITY);
        }
    }
}

}  // namespace scores
}  // namespace tcbnn
