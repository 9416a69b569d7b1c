// Log probabilities from logits.  With d = (x - max x) / T and S = sum e^d over a row of V logits:
//   logp(target) = d(target) - ln S,   entropy = ln S - sum(e^d d) / S,   the `top` largest logits and their logp.
// A token of logit -inf is ruled out: probability 0, no alternative.  A row that rules out everything has logp
// -inf and entropy 0; one that holds NaN or +inf has NaN for both.  Alternatives are ordered by (logit, lowest token),
// NaN taking no part.
//
// One pass over the row.  With c = log2(e) / T and R = max(x) c rounded to a whole number, so that fma(x, c, -R) is rounded once, a
// thread keeps the maximum m, R, s = sum 2^{xc - R} and t = sum 2^{xc - R} (xc - R) of what it has seen; a batch of 64 bytes that
// raises R rescales both once.  R is at least -2^28, and logits below -1e30 (fp16: the lowest, -65504), masks among them, are
// raised to that in front of the sums, two at a time in 16 bits: their terms are 0, and no product 0 * inf arises.  Rows for which
// that does not hold -- |max(x) c| beyond 2^28, a maximum near -65504 in fp16, temperatures beyond 1e6 -- are summed again as they
// are, from their maximum.
//
// Alternatives cost the pass nothing but the threads' maxima: at its end the top-th largest of them (of the best few per warp) is a
// bound that at least `top` logits reach, hardly more when they come in random order; the few threads whose maximum reaches it have
// their vectors read once more, by their whole warp, and what reaches the bound goes to a list in shared memory, which is
// sorted, 32 keys to a warp, and merged.  (A threshold from the first 64 bytes of every thread, tested in the loop: 178 us against
// 83 without alternatives at 4096 x 50001.)  Where the list overflows -- more ties than it holds -- the row is read again, the
// list cut to its best `top` as often as it fills.
//
// One to eight warps share a row, or the CTAs of a cluster, whose parts meet in the first one's shared memory.  (A thread's share depends
// on where the row starts modulo 16 bytes, and with it the order of the sums, not the values that are compared.)
//
// What bounds it: long rows the issue slots, 2.75 instructions a clock of 4 while 0.55 of the special-function units' slots and 0.70 of
// HBM's copy rate are used (4096 x 50001 bf16, 410 MB: 90.5 us with eight alternatives, 75.0 without); few or short rows the chain
// load, sums, bound, second look, sort (8 x 1000 fp32 4.0 us, 1 x 131072 bf16 6.4, of which a launch is 2).  24 warps an SM instead of
// 32, 107 us; 40 warps with 32 bytes a thread, 94.5; the row that follows fetched into L2 ahead, 97 to 127.
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

// maximum, R and the two sums of part of a row
struct Sums { float m, ref, s, t; };
constexpr float kLeastRef = -268435456.f;              // -2^28

__host__ __device__ constexpr int list_of(int warps) { return warps < 8 ? 256 * warps : 2048; }      // keys that a row's list holds
constexpr uint32_t kAll = 0xffffffffu;

using linear::ex2;
// order of finite values and infinities as unsigned numbers, NaN and -inf lowest
__device__ __forceinline__ uint32_t order_of(float x) { return (uint32_t)(key_of(x, 0) >> 32); }

__device__ __forceinline__ uint4 load16(const void* p) {
    uint4 v;
    asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
// what logits are raised to in front of the sums
__host__ __device__ constexpr float lowest_of(int type) { return type == linear::FP16 ? -65504.f : -0x1.92p+99f; }      // (about -1e30)
template <int TYPE>
struct Element {
    static constexpr int kBytes = TYPE == linear::FP32 ? 4 : 2, kPer = 16 / kBytes;
    static __device__ __forceinline__ uint32_t raise(uint32_t w) {           // (NaN stays)
        uint32_t r;
        if constexpr (TYPE == linear::FP32) asm("max.NaN.f32 %0, %1, %2;" : "=r"(r) : "r"(w), "r"(0xF1490000u));
        else if constexpr (TYPE == linear::BF16) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(w), "r"(0xF149F149u));
        else asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(w), "r"(0xFBFFFBFFu));
        return r;
    }
    static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {      // (of NaN and a number the number)
        uint32_t r;
        if constexpr (TYPE == linear::FP32) asm("max.f32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        else if constexpr (TYPE == linear::BF16) asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        else asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ float low(uint32_t w) {
        if constexpr (TYPE == linear::FP32) return __uint_as_float(w);
        else if constexpr (TYPE == linear::BF16) return __uint_as_float(w << 16);
        else return __half2float(__ushort_as_half((unsigned short)(w & 0xFFFFu)));
    }
    static __device__ __forceinline__ float high(uint32_t w) {
        if constexpr (TYPE == linear::BF16) return __uint_as_float(w & 0xFFFF0000u);
        else return __half2float(__ushort_as_half((unsigned short)(w >> 16)));
    }
    static __device__ __forceinline__ float most(uint32_t w) {                // of a word
        if constexpr (TYPE == linear::FP32) return __uint_as_float(w);
        else return fmaxf(low(w), high(w));
    }
    // element j of a vector
    static __device__ __forceinline__ float get(const uint4& v, int j) {
        if constexpr (TYPE == linear::FP32) {
            return __uint_as_float(j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w);
        } else {
            const uint32_t w = j < 2 ? v.x : j < 4 ? v.y : j < 6 ? v.z : v.w;
            if constexpr (TYPE == linear::BF16) return __uint_as_float(j & 1 ? w & 0xFFFF0000u : w << 16);
            else return __half2float(__ushort_as_half((unsigned short)(j & 1 ? w >> 16 : w & 0xFFFFu)));
        }
    }
};

// ---- sorted lists of 32 keys, one per lane, falling -------------------------------------------------
__device__ __forceinline__ void exchange(unsigned long long& key, int distance, bool larger) {
    const unsigned long long o = __shfl_xor_sync(kAll, key, distance);
    if ((o > key) == larger) key = o;
}
__device__ __forceinline__ unsigned long long sort32(unsigned long long key) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int size = 2; size <= 32; size *= 2)
#pragma unroll
        for (int d = size / 2; d; d /= 2) exchange(key, d, ((lane & d) == 0) == ((lane & size) == 0));
    return key;
}
__device__ __forceinline__ uint32_t sort32(uint32_t v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int size = 2; size <= 32; size *= 2)
#pragma unroll
        for (int d = size / 2; d; d /= 2) {
            const uint32_t o = __shfl_xor_sync(kAll, v, d);
            v = ((lane & d) == 0) == ((lane & size) == 0) ? max(v, o) : min(v, o);
        }
    return v;
}
// the 32 best of two falling lists (`other` given in rising order)
__device__ __forceinline__ unsigned long long merge32(unsigned long long key, unsigned long long other) {
    const int lane = threadIdx.x & 31;
    if (other > key) key = other;
#pragma unroll
    for (int d = 16; d; d /= 2) exchange(key, d, (lane & d) == 0);
    return key;
}

template <int NW>
struct Shared {
    unsigned long long list[list_of(NW)];
    unsigned long long best[NW][32];     // per warp; [0]: the row's
    Sums sums[NW + 1];                                 // per warp; [NW]: of the CTA, for the cluster
    uint32_t maxima[32];
    unsigned char hot[NW][32];                         // per warp: lanes whose maximum reaches the bound
    int count;
    unsigned long long cut;                            // of the second reading: what does not exceed it is out
};
template <int NW>
__device__ __forceinline__ void meet() {
    if constexpr (NW == 1) __syncwarp();
    else __syncthreads();
}

// the 32 best of the first `n` of the list, falling, in the lanes of warp 0
template <int NW>
__device__ __forceinline__ unsigned long long best_of_list(Shared<NW>& s, int n, int warp, int lane) {
    if (n <= 32) {                                     // by counting: an eighth of the instructions of sorting six
        if (warp == 0) {
            const unsigned long long mine = lane < n ? s.list[lane] : 0ull;
            int rank = 0;
            for (int i = 0; i < n; i++) rank += s.list[i] > mine;
            __syncwarp();
            s.best[0][lane] = 0;
            __syncwarp();
            if (lane < n) s.best[0][rank] = mine;
            __syncwarp();
            return s.best[0][lane];
        }
        return 0ull;
    }
    unsigned long long key = 0;
    for (int i = warp * 32; i < n; i += NW * 32) {
        const unsigned long long other = sort32(i + lane < n ? s.list[i + lane] : 0ull);
        key = merge32(key, __shfl_xor_sync(kAll, other, 31));
    }
    if constexpr (NW > 1) {
        const int lists = min(NW, (n + 31) >> 5);
        s.best[warp][lane] = key;
        __syncthreads();
        for (int h = NW / 2; h; h /= 2) {
            if (warp < h && warp + h < lists) s.best[warp][lane] = key = merge32(key, s.best[warp + h][31 - lane]);
            __syncthreads();
        }
    }
    return key;
}

__device__ __forceinline__ float most_of_warp(float x) {                   // (-inf where nothing else is)
    const uint32_t o = __reduce_max_sync(kAll, order_of(x));
    return o ? logit_of((unsigned long long)o << 32) : -INFINITY;
}
__device__ __forceinline__ float ref_of(float m, float c) { return fmaxf(rintf(m * c), kLeastRef); }
__device__ __forceinline__ void reduce(Sums& q, float c) {                // over a warp
    q.m = most_of_warp(q.m);
    const float ref = ref_of(q.m, c), d = q.ref - ref, f = ex2(d);
    q.t = f * fmaf(q.s, d, q.t);
    q.s = f * q.s;
    q.ref = ref;
#pragma unroll
    for (int h = 16; h; h /= 2) {
        q.s += __shfl_xor_sync(kAll, q.s, h);
        q.t += __shfl_xor_sync(kAll, q.t, h);
    }
}
// The sums of a warp's threads, into shared memory where several share the row; behind a barrier finish_row() gives the row's.
template <int NW>
__device__ __forceinline__ void reduce_warps(Sums& q, Shared<NW>& s, float c, int warp, int lane) {
    reduce(q, c);
    if (NW > 1 && lane == 0) s.sums[warp] = q;
}
template <int NW>
__device__ __forceinline__ void finish_row(Sums& q, Shared<NW>& s, float c, int lane) {
    if constexpr (NW > 1) {
        q = lane < NW ? s.sums[lane] : Sums{-INFINITY, kLeastRef, 0.f, 0.f};
        reduce(q, c);
    }
}
// The sums of a whole row as they are defined, from its maximum: R = 0 stands for mc.
template <int TYPE, int NW>
__device__ __forceinline__ void sum_again(const Args& a, Shared<NW>& s, const char* base, float c, int tid, int warp, int lane, Sums& q) {
    constexpr int THREADS = NW * 32;
    float m = -INFINITY;
    for (int i = tid; i < a.V; i += THREADS) m = fmaxf(m, linear::load(base, i, TYPE));
    q = Sums{m, 0.f, 0.f, 0.f};
    meet<NW>();                                        // (s.sums is free)
    reduce_warps<NW>(q, s, 0.f, warp, lane);
    meet<NW>();
    finish_row<NW>(q, s, 0.f, lane);
    m = q.m;
    q = Sums{0.f, 0.f, 0.f, 0.f};
    for (int i = tid; i < a.V; i += THREADS) {
        const float x = linear::load(base, i, TYPE), y = (x - m) * c, e = x == -INFINITY ? 0.f : ex2(y);
        q.s += e;
        q.t = fmaf(e, fmaxf(y, -3.0e38f), q.t);
    }
    meet<NW>();
    reduce_warps<NW>(q, s, 0.f, warp, lane);
    meet<NW>();
    finish_row<NW>(q, s, 0.f, lane);
    q.m = m;
}

template <int TYPE, int NW, bool CLUSTER>
__device__ __forceinline__ void row(const Args& a, Shared<NW>& s, long long r, uint32_t rank, uint32_t nctas) {
    using E = Element<TYPE>;
    constexpr int THREADS = NW * 32, PER = E::kPer, U = 4, LIST = list_of(NW);
    const int tid = NW == 1 ? threadIdx.x & 31 : threadIdx.x, lane = tid & 31, warp = NW == 1 ? 0 : tid >> 5;
    const char* base = reinterpret_cast<const char*>(a.logits) + r * a.ld * E::kBytes;
    // elements in front of the first 16-byte boundary, vectors, elements behind them
    const int head = min(a.V, (int)((16 - (reinterpret_cast<uintptr_t>(base) & 15)) & 15) / E::kBytes);
    const int vectors = (a.V - head) / PER, tail = a.V - head - vectors * PER;
    const char* body = base + head * E::kBytes;
    const int v0 = CLUSTER ? (int)((long long)vectors * rank / nctas) : 0, v1 = CLUSTER ? (int)((long long)vectors * (rank + 1) / nctas) : vectors;
    const bool first = rank == 0, last = rank + 1 == nctas;
    const float c = a.inv_t * 1.44269504088896341f;    // log2 e / T

    if (tid == 0) { s.count = 0; s.cut = 0; }
    Sums q{-INFINITY, kLeastRef, 0.f, 0.f};
    auto raise_to = [&](float bm) {                    // a batch's maximum
        if (bm > q.m) {
            q.m = bm;
            const float ref = ref_of(bm, c);
            if (ref > q.ref) {
                const float d = q.ref - ref, f = ex2(d);
                q.t = f * fmaf(q.s, d, q.t);
                q.s *= f;
                q.ref = ref;
            }
        }
    };
    auto add = [&](float x) {
        const float y = fmaf(x, c, -q.ref), e = ex2(y);
        q.s += e;
        q.t = fmaf(e, y, q.t);
    };
    auto push = [&](float x, int token) {
        const unsigned long long key = key_of(x, token);
        if (key) {
            const int at = atomicAdd(&s.count, 1);
            if (at < LIST) s.list[at] = key;
        }
    };
    auto batch = [&](const uint4 (&v)[U]) {
        uint32_t r[U][4], most = E::raise(v[0].x);
#pragma unroll
        for (int u = 0; u < U; u++) {
            r[u][0] = E::raise(v[u].x); r[u][1] = E::raise(v[u].y); r[u][2] = E::raise(v[u].z); r[u][3] = E::raise(v[u].w);
            most = E::larger(most, E::larger(E::larger(r[u][0], r[u][1]), E::larger(r[u][2], r[u][3])));
        }
        raise_to(E::most(most));
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                add(E::low(r[u][j]));
                if constexpr (E::kPer == 8) add(E::high(r[u][j]));
            }
    };
    // (-inf: no part in anything)
    const uint32_t fill = TYPE == linear::FP32 ? 0xFF800000u : TYPE == linear::BF16 ? 0xFF80FF80u : 0xFC00FC00u;
    // of a thread, U vectors THREADS apart each: so many batches that every thread has in full, and one more that some have in part
    const int i0 = v0 + tid, full = (v1 - v0) / (U * THREADS), batches = (v1 - v0 + U * THREADS - 1) / (U * THREADS);
    const char* at_v = body + (long long)i0 * 16;
    auto load = [&](uint4 (&v)[U], int b) {
        if (b < full) {
#pragma unroll
            for (int u = 0; u < U; u++) v[u] = load16(at_v + u * THREADS * 16);
        } else if (b < batches) {
#pragma unroll
            for (int u = 0; u < U; u++)
                v[u] = i0 + (b * U + u) * THREADS < v1 ? load16(at_v + u * THREADS * 16) : make_uint4(fill, fill, fill, fill);
        }
        at_v += U * THREADS * 16;
    };
    uint4 cur[U], next[U];
    load(cur, 0);
    // the ends: a thread each
    int at = -1;
    float end = -INFINITY;
    if (first && tid < head) at = tid;
    else if (last && tid >= 16 && tid - 16 < tail) at = head + vectors * PER + tid - 16;
    if (at >= 0) end = linear::load(base, at, TYPE);
    long long target = -1;
    float given = 0.f;
    if (a.logp && tid == 0 && first) {                 // (under way while the row is read)
        target = a.target_bytes == 8 ? reinterpret_cast<const long long*>(a.targets)[r] : reinterpret_cast<const int*>(a.targets)[r];
        if (target >= 0 && target < a.V) given = linear::load(base, target, TYPE);
    }
    for (int b = 0; b < batches; b++) {
        load(next, b + 1);
        if (b < full || i0 - lane + b * U * THREADS < v1) batch(cur);    // (of the warp)
#pragma unroll
        for (int u = 0; u < U; u++) cur[u] = next[u];
    }
    const float most = q.m;                            // of the vectors
    if (at >= 0) {
        const float raised = end < lowest_of(TYPE) ? lowest_of(TYPE) : end;
        raise_to(raised);
        add(raised);
    }
    if (a.top) {
        reduce_warps<NW>(q, s, c, warp, lane);
        uint32_t o = most > lowest_of(TYPE) ? order_of(most) : 0u;
        if constexpr (NW > 1) {
            constexpr int BEST = 32 / NW;              // per warp
            for (int i = 0; i < BEST; i++) {
                const uint32_t largest = __reduce_max_sync(kAll, o);
                if (lane == 0) s.maxima[warp * BEST + i] = largest;
                if (lane == __ffs(__ballot_sync(kAll, o == largest)) - 1) o = 0;
            }
            __syncthreads();
            o = s.maxima[lane];
        }
        o = __shfl_sync(kAll, sort32(o), a.top - 1);
        const float bound = o ? logit_of((unsigned long long)o << 32) : -INFINITY;
        if (NW == 1) __syncwarp();                     // (the count is 0)
        // the vectors of the threads that reach it, over the lanes of their warp
        const uint32_t hot = __ballot_sync(kAll, most >= bound);
        if (most >= bound) s.hot[warp][__popc(hot & ((1u << lane) - 1))] = (unsigned char)lane;
        __syncwarp();
        const int each = (v1 - v0 - (tid - lane) + THREADS - 1) / THREADS, vs = each > 0 ? __popc(hot) * each : 0;      // (each: the first lane's)
        const float per = 1.f / (float)each;
        for (int p = lane; p < vs; p += 32) {
            // (p / each: exact in fp32, as p + 1/2 is half of 1 / each off the next whole number at least, and p < 2^18; others divide)
            const int h = vs <= 1 << 18 ? (int)(((float)p + 0.5f) * per) : p / each;
            const int i = v0 + tid - lane + s.hot[warp][h] + (p - h * each) * THREADS;
            if (i >= v1) continue;
            const uint4 v = load16(body + (long long)i * 16);
            uint32_t over = 0;
#pragma unroll
            for (int j = 0; j < PER; j++) over |= E::get(v, j) >= bound ? 1u << j : 0u;
            for (; over; over &= over - 1) {
                const int e = head + i * PER + __ffs(over) - 1;
                push(linear::load(base, e, TYPE), e);
            }
        }
        if (end >= bound && at >= 0) push(end, at);
    }
    if (!a.top) reduce_warps<NW>(q, s, c, warp, lane);
    meet<NW>();
    finish_row<NW>(q, s, c, lane);
    // alternatives
    unsigned long long key = 0;
    if (a.top) {
        const int n = s.count;
        if (n <= LIST) {
            key = best_of_list<NW>(s, n, warp, lane);
        } else {
            // again, in short steps behind each of which the list has room for the next
            const int from = first ? 0 : head + v0 * PER, to = last ? a.V : head + v1 * PER;
            meet<NW>();
            if (tid == 0) { s.count = 0; s.cut = 0; }
            meet<NW>();
            for (int e0 = from; e0 < to; e0 += 2 * THREADS) {
                const unsigned long long cut = s.cut;
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const int e = e0 + j * THREADS + tid;
                    const unsigned long long k = e < to ? key_of(linear::load(base, e, TYPE), e) : 0ull;
                    if (k > cut) s.list[atomicAdd(&s.count, 1)] = k;
                }
                meet<NW>();
                const int have = s.count;
                meet<NW>();                            // (everybody has read it before it changes)
                if (have > LIST - 2 * THREADS || e0 + 2 * THREADS >= to) {
                    key = best_of_list<NW>(s, have, warp, lane);
                    meet<NW>();
                    if (warp == 0) {
                        if (lane < a.top) s.list[lane] = key;
                        if (lane == a.top - 1) s.cut = key;
                        if (lane == 0) s.count = min(have, a.top);
                    }
                    meet<NW>();
                }
            }
        }
    }
    if constexpr (CLUSTER) {
        // the first CTA's first warp takes the others' parts
        if (warp == 0) {
            s.best[0][lane] = key;
            if (lane == 0) s.sums[NW] = q;
        }
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (first) {
            auto peer = [&](const void* p, uint32_t of) {
                uint32_t x;
                asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(x) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(of));
                return x;
            };
            auto ld = [&](uint32_t at) {
                float v;
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
                return v;
            };
            q = Sums{-INFINITY, kLeastRef, 0.f, 0.f};
            if ((uint32_t)lane < nctas) {
                const uint32_t at = peer(&s.sums[NW], lane);
                q = Sums{ld(at), ld(at + 4), ld(at + 8), ld(at + 12)};
            }
            reduce(q, c);
            if (a.top) {                               // warp w has the list of CTA w
                if (warp > 0 && (uint32_t)warp < nctas)
                    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(key) : "r"(peer(&s.best[0][lane], warp)) : "memory");
                if ((uint32_t)warp < nctas) s.best[warp][lane] = key;
                __syncthreads();
                for (int h = (int)nctas / 2; h; h /= 2) {
                    if (warp < h) s.best[warp][lane] = key = merge32(key, s.best[warp + h][31 - lane]);
                    __syncthreads();
                }
            }
        }
        __syncwarp();
        // (nobody leaves before its part is read)
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (!first) return;
    }
    // terms of raised logits are 0, and what R was rounded by is at most 16
    const bool right = a.inv_t >= 1e-6f && a.inv_t <= 1e6f && (q.m - lowest_of(TYPE)) * c > 150.f && fabsf(q.m * c) < -kLeastRef - 256.f;
    if (!right) sum_again<TYPE, NW>(a, s, base, c, tid, warp, lane, q);
    if (warp == 0) {
        // ln sum e^{(x - m)/T}
        const float lse = logf(q.s) - (right ? fmaf(q.m, c, -q.ref) * 0.693147180559945309f : 0.f);
        auto logp = [&](float x) { return x == -INFINITY ? (q.s == q.s ? -INFINITY : q.s) : fmaf(x - q.m, a.inv_t, -lse); };
        if (lane == 0) {
            if (a.logp) a.logp[r] = target < 0 ? 0.f : target >= a.V ? NAN : logp(given);
            if (a.entropy) a.entropy[r] = q.m == -INFINITY && q.s == 0.f ? 0.f : logf(q.s) - q.t / q.s * 0.693147180559945309f;
        }
        if (lane < a.top) {
            a.top_ids[r * a.top + lane] = key ? token_of(key) : -1;
            a.top_logp[r * a.top + lane] = logp(key ? logit_of(key) : -INFINITY);
        }
    }
}

}  // namespace scores
}  // namespace tcbnn
