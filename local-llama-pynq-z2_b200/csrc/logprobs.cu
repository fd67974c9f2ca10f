// Log probabilities of given tokens, the entropy and the most probable tokens of rows of logits (mvb_logprobs).
//
//     lse = m + ln z,  m = max x,  z = sum exp(x - m);   logp[id] = (x[id] - m) - ln z
//     entropy = -sum p ln p = ln z - (sum (x - m) exp(x - m)) / z
//     top: the `top` largest logits by (value, lowest index first), with their log probabilities
//
// One pass over the logits: each thread keeps (m, z, w = sum (x - m) exp(x - m)) of its elements (m starts as its warp's
// first maximum and moves only when it is 4 behind), and for the top tokens only the maximum of each 4 vectors (one
// shared-memory word per 16 or 32 elements), so that the streaming loop has no candidate lists and no barriers. Afterwards
// the top-th largest of the threads' own maxima (its 16 leading bits) is a lower bound of the top-th largest element; the
// few groups whose maximum reaches it are listed, their vectors read again (from L2), a thread each, and their elements
// that reach it ranked. Rows with more such elements than the list holds (a vocabulary masked to a few tokens: the rest
// all equal) take the elements above the bound, then those equal to it in the order of their index; where even the former
// overflow, `top` rounds of an arg max.
// A few rows: a row is split over a cluster of up to 16 CTAs, joined through distributed shared memory in rank order.
// Bound: the logits are read once; the exponentials (one a logit, 16 per clock and SM) come close for 16-bit types.
// 2000 rows of 151,936 bf16 logits, top 20: 119 us in a burst (5.1 TB/s), 130 for a second on end, where the power limit
// takes a tenth of the clock; 1000 rows in fp32: 121 us; one row: 9 us.
#include <cooperative_groups.h>
#include <limits.h>
#include <math.h>

#include <atomic>

#include "../../include/matvec_b200.h"
#include "mvb_runtime.h"
#include "rows.cuh"

namespace mvb {
namespace logp {

using namespace rows;
namespace cg = cooperative_groups;

static __device__ int g_logp_error;

constexpr int kVecs = 4;      // 16-byte vectors a thread has in flight (a group: one maximum)
constexpr int kList = 2048;   // candidates
constexpr int kMostTop = 64;
constexpr int kGroups = 512;    // groups that are read again, listed; more are scanned by their own threads
constexpr float kBehind = 4.0f;
constexpr float kLog2e = 1.44269504088896341f;

struct Params {
    const void *x;
    const int *ids;
    float *logp, *entropy, *top_logp;
    int *top_ids;
    long long stride;
    int rows, vocab, nids, top, splits, iters;
};

// (value, ~index) in one integer: larger values first, then the lower index; NaN behind everything, -0 with +0.
__device__ __forceinline__ unsigned long long key_of(float v, int i) {
    const float c = v == 0.0f ? 0.0f : v;
    const uint32_t b = __float_as_uint(c);
    const uint32_t o = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return ((unsigned long long)(v == v ? o : 0u) << 32) | (uint32_t)~(uint32_t)i;
}
__device__ __forceinline__ float value_of(unsigned long long key) {
    const uint32_t o = (uint32_t)(key >> 32);
    if (!o) return __int_as_float(0x7FC00000);
    return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);
}

struct Sums {
    float m, z, w;  // maximum, sum of exp(x - m), sum of (x - m) exp(x - m)
};

__device__ __forceinline__ float exp_fast(float d) {  // exp(d), d <= 0 or NaN
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(__fmul_rn(d, kLog2e)));
    return y;
}

// x - m, at least -1e30 (so that exp(-inf) * -inf is 0), NaN kept
__device__ __forceinline__ float below(float x, float base) {
    float d = __fsub_rn(x, base);
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(d) : "f"(-1e30f));
    return d;
}

__device__ __forceinline__ void move_to(Sums &s, float m) {  // m >= s.m
    if (m == s.m || s.m == -INFINITY) {
        s.m = m;  // nothing summed yet (or the same): a thread that only saw -inf has z = w = 0
        return;
    }
    const float d = below(s.m, m), e = exp_fast(d);
    s.w = e * __fmaf_rn(d, s.z, s.w);
    s.z *= e;
    s.m = m;
}

__device__ __forceinline__ Sums joined(Sums a, Sums b) {
    const float m = fmaxf(a.m, b.m);
    move_to(a, m);
    move_to(b, m);
    return Sums{m, a.z + b.z, a.w + b.w};
}

template <typename T> struct Vec { static constexpr int kN = 16 / sizeof(T); };

// Two fp32 lanes in one register pair: Blackwell's packed adds and multiply-adds, half the instructions.
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 halves(uint64_t p) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p));
    return f;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// Words of a vector (one fp32 or two 16-bit elements): the larger of two without regard to NaN; not below a floor, NaN
// kept; and the fp32 values. The floor stands for elements whose exponential is zero as long as the maximum is above
// kSane: it keeps -inf out of (x - m) exp(x - m).
template <typename T> struct Word;
template <> struct Word<float> {
    static constexpr float kSane = -1e29f;
    static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
        return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    }
    static __device__ __forceinline__ uint32_t floored(uint32_t a) {
        asm("max.NaN.f32 %0, %0, %1;" : "+r"(a) : "r"(0xF149F2CAu));  // -1e30
        return a;
    }
    static __device__ __forceinline__ float first(uint32_t a) { return __uint_as_float(a); }
    static __device__ __forceinline__ float second(uint32_t) { return -INFINITY; }
};
template <> struct Word<__nv_bfloat16> {
    static constexpr float kSane = -1e29f;
    static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ uint32_t floored(uint32_t a) {
        asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(a) : "r"(0xF14AF14Au));  // -1.0004e30
        return a;
    }
    static __device__ __forceinline__ float first(uint32_t a) { return __uint_as_float(a << 16); }
    static __device__ __forceinline__ float second(uint32_t a) { return __uint_as_float(a & 0xFFFF0000u); }
};
template <> struct Word<__half> {
    static constexpr float kSane = -60000.0f;
    static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ uint32_t floored(uint32_t a) {
        asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(a) : "r"(0xFBFFFBFFu));  // -65504
        return a;
    }
    static __device__ __forceinline__ float first(uint32_t a) { return __low2float(*reinterpret_cast<__half2 *>(&a)); }
    static __device__ __forceinline__ float second(uint32_t a) { return __high2float(*reinterpret_cast<__half2 *>(&a)); }
};

template <typename T>
__device__ __forceinline__ void unpack(const uint4 &u, float (&f)[Vec<T>::kN]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (sizeof(T) == 4) {
            f[i] = __uint_as_float(w[i]);
        } else {
            f[2 * i] = Word<T>::first(w[i]);
            f[2 * i + 1] = Word<T>::second(w[i]);
        }
    }
}

__device__ __forceinline__ uint4 load_stream(const uint4 *p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}

template <typename T, bool TOP, int kThreads>
__global__ void __launch_bounds__(kThreads, 768 / kThreads) logprobs_kernel(const Params p) {
    constexpr int N = Vec<T>::kN;
    // turns of the streaming loop that share a maximum: 32 elements of a thread (with 16 for fp32 the maxima of a 151,936
    // word vocabulary take 38 KB and two thirds of the threads fit)
    constexpr int kTurns = sizeof(T) / 2, kGroupVecs = kVecs * kTurns;
    extern __shared__ __align__(16) float group_max[];  // [iters][kThreads], TOP only
    __shared__ Sums parts[kThreads / 32];
    __shared__ Sums cta_sums;
    __shared__ __align__(16) float thread_max[kThreads];
    __shared__ unsigned long long list[TOP ? kList : 1], best[TOP ? kMostTop : 1];
    __shared__ unsigned long long round_best[kThreads / 32];
    __shared__ float bound;
    __shared__ int count, above, taken, listed, warp_count[kThreads / 32];
    __shared__ uint16_t groups[TOP ? kGroups : 1];

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row = blockIdx.x / p.splits, split = blockIdx.x - row * p.splits;
    const T *x = static_cast<const T *>(p.x) + (size_t)row * p.stride;
    // elements before the first 16-byte boundary, whole vectors, the rest
    int head = (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T);
    head = min(head, p.vocab);
    const int nvec = (p.vocab - head) / N, edge = p.vocab - nvec * N;  // edge: elements outside the vectors, < 2 N
    const int v0 = (int)((long long)nvec * split / p.splits), v1 = (int)((long long)nvec * (split + 1) / p.splits);
    const uint4 *vec = reinterpret_cast<const uint4 *>(x + head);
    auto edge_at = [&](int i) { return i < head ? i : head + nvec * N + (i - head); };

    Sums s = {-INFINITY, 0.0f, 0.0f};
    float mine = -INFINITY;  // this thread's largest element of the vectors
    int seen = 0;
    int v = v0 + tid;
    // whole groups of kVecs vectors, the same number for every thread
    const int whole = (v1 - v0) / (kVecs * kThreads);
    uint4 next[kVecs];  // the group after this one, on its way
    if (whole > 0) {
#pragma unroll
        for (int k = 0; k < kVecs; k++) next[k] = load_stream(vec + v + k * kThreads);
    }
    for (; seen < whole; v += kVecs * kThreads, seen++) {
        uint32_t u[4 * kVecs];
#pragma unroll
        for (int k = 0; k < kVecs; k++) {
            u[4 * k] = next[k].x;
            u[4 * k + 1] = next[k].y;
            u[4 * k + 2] = next[k].z;
            u[4 * k + 3] = next[k].w;
        }
        if (seen + 1 < whole) {
#pragma unroll
            for (int k = 0; k < kVecs; k++) next[k] = load_stream(vec + v + (kVecs + k) * kThreads);
        }
        uint32_t gm[2] = {u[0], u[1]};
#pragma unroll
        for (int k = 2; k < 4 * kVecs; k++) gm[k & 1] = Word<T>::larger(gm[k & 1], u[k]);
        gm[0] = Word<T>::larger(gm[0], gm[1]);
        const float g = fmaxf(fmaxf(Word<T>::first(gm[0]), Word<T>::second(gm[0])), -INFINITY);
        if (TOP) {
            float &gm_at = group_max[seen / kTurns * kThreads + tid];
            gm_at = seen % kTurns ? fmaxf(gm_at, g) : g;
        }
        mine = fmaxf(mine, g);
        if (seen == 0) {
            float first = g;
#pragma unroll
            for (int o = 16; o; o >>= 1) first = fmaxf(first, __shfl_xor_sync(0xffffffffu, first, o));
            s.m = first;
        }
        if (g > s.m + kBehind) move_to(s, g);
        if (s.m > Word<T>::kSane) {
            const uint64_t base = pair(-s.m, -s.m), l2e = pair(kLog2e, kLog2e);
            uint64_t z[2] = {0, 0}, w[2] = {0, 0};
#pragma unroll
            for (int k = 0; k < 4 * kVecs; k += sizeof(T) / 2) {
                uint64_t x;
                if constexpr (sizeof(T) == 4) {
                    x = pair(Word<T>::first(Word<T>::floored(u[k])), Word<T>::first(Word<T>::floored(u[k + 1])));
                } else {
                    const uint32_t f = Word<T>::floored(u[k]);
                    x = pair(Word<T>::first(f), Word<T>::second(f));
                }
                const int a = (k / (sizeof(T) / 2)) & 1;
                const uint64_t d = add2(x, base);
                const float2 t = halves(mul2(d, l2e));
                float2 e;
                asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(t.x));
                asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(t.y));
                const uint64_t e2 = pair(e.x, e.y);
                z[a] = add2(z[a], e2);
                w[a] = fma2(d, e2, w[a]);
            }
            const float2 zz = halves(add2(z[0], z[1])), ww = halves(add2(w[0], w[1]));
            s.z += zz.x + zz.y;
            s.w += ww.x + ww.y;
        } else {  // only masks so far: element by element
            const float base = s.m == -INFINITY ? 0.0f : s.m;
#pragma unroll
            for (int k = 0; k < 4 * kVecs; k++) {
                for (int h = 0; h < 4 / (int)sizeof(T); h++) {
                    const float d = below(h ? Word<T>::second(u[k]) : Word<T>::first(u[k]), base), e = exp_fast(d);
                    s.z += e;
                    s.w = __fmaf_rn(d, e, s.w);
                }
            }
        }
    }
    if (v < v1) {  // the last, partial group
        float g = -INFINITY;
        for (int k = 0; k < kVecs && v + k * kThreads < v1; k++) {
            float f[N];
            unpack<T>(load_stream(vec + v + k * kThreads), f);
            float gv = f[0];
#pragma unroll
            for (int i = 1; i < N; i++) gv = fmaxf(gv, f[i]);
            g = fmaxf(g, gv);
            if (gv > s.m + kBehind) move_to(s, gv);
            const float base = s.m == -INFINITY ? 0.0f : s.m;
#pragma unroll
            for (int i = 0; i < N; i++) {
                const float d = below(f[i], base), e = exp_fast(d);
                s.z += e;
                s.w = __fmaf_rn(d, e, s.w);
            }
        }
        if (TOP) {
            float &gm_at = group_max[seen / kTurns * kThreads + tid];
            gm_at = seen % kTurns ? fmaxf(gm_at, g) : g;
        }
        mine = fmaxf(mine, g);
        seen++;
    }
    if (split == 0 && tid < edge) {
        const float f = to_f32(x[edge_at(tid)]);
        if (f > s.m + kBehind) move_to(s, f);
        const float d = below(f, s.m == -INFINITY ? 0.0f : s.m), e = exp_fast(d);
        s.z += e;
        s.w = __fmaf_rn(d, e, s.w);
    }
    // the given tokens' logits, on their way while the rest is joined
    float given = 0.0f;
    int id = -1;
    if (split == 0 && tid < p.nids) {
        id = p.ids[(size_t)row * p.nids + tid];
        if ((unsigned)id < (unsigned)p.vocab) given = to_f32(x[id]);
    }
    {  // the warp's sums: one move to its maximum, then plain sums
        float m = s.m;
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        move_to(s, m);
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            s.z += __shfl_xor_sync(0xffffffffu, s.z, o);
            s.w += __shfl_xor_sync(0xffffffffu, s.w, o);
        }
        if (lane == 0) parts[warp] = s;
    }
    if (TOP) thread_max[tid] = mine;
    if (tid == 0) {
        bound = -INFINITY;
        count = above = taken = listed = 0;
    }
    if (TOP && tid < kMostTop) best[tid] = 0;
    __syncthreads();
    if (warp == 1 && lane == 0) {
        Sums t = parts[0];
#pragma unroll
        for (int w = 1; w < kThreads / 32; w++) t = joined(t, parts[w]);
        cta_sums = t;
    }
    if (TOP) {
        // A lower bound of the top-th largest of the threads' maxima, and so of the top-th largest element: the largest
        // value of 16 leading bits that `top` maxima reach (exact for bf16). One warp, a binary search of 16 votes.
        if (warp == 0) {
            uint32_t o[kThreads / 32];
#pragma unroll
            for (int i = 0; i < kThreads / 32; i++) o[i] = (uint32_t)(key_of(thread_max[i * 32 + lane], 0) >> 48);
            uint32_t found = 0;
#pragma unroll
            for (uint32_t bit = 0x8000u; bit; bit >>= 1) {
                int n = 0;
#pragma unroll
                for (int i = 0; i < kThreads / 32; i++) n += o[i] >= (found | bit);
                if (__reduce_add_sync(0xffffffffu, n) >= p.top) found |= bit;
            }
            // (-inf and what lies below its 16 bits: everything is a candidate)
            if (lane == 0) bound = found <= 0x007Fu ? -INFINITY : value_of((unsigned long long)found << 48);
        }
        __syncthreads();
        const float bd = bound;
        // the elements that reach it, into the list while it has room; count counts them all
        auto offer = [&](float v, int i) {
            const int at = atomicAdd(&count, 1);
            if (at < kList) list[at] = key_of(v, i);
            if (v > bd) atomicAdd(&above, 1);
        };
        if (split == 0 && tid < edge) {
            const float v = to_f32(x[edge_at(tid)]);
            if (v >= bd) offer(v, edge_at(tid));
        }
        const int entries = (seen + kTurns - 1) / kTurns;
        if (mine >= bd) {
#pragma unroll 8
            for (int it = 0; it < entries; it++)
                if (group_max[it * kThreads + tid] >= bd) {
                    const int at = atomicAdd(&listed, 1);
                    if (at < kGroups) groups[at] = (uint16_t)(it * kThreads + tid);
                }
        }
        __syncthreads();
        const int ng = listed;
        if (ng <= kGroups) {  // the groups' vectors, a thread each
            for (int i = tid; i < ng * kGroupVecs; i += kThreads) {
                const int g = groups[i / kGroupVecs];
                const int v = v0 + g % kThreads + ((g / kThreads) * kGroupVecs + i % kGroupVecs) * kThreads;
                if (v >= v1) continue;
                float f[N];
                unpack<T>(vec[v], f);
#pragma unroll
                for (int e = 0; e < N; e++)
                    if (f[e] >= bd) offer(f[e], head + v * N + e);
            }
        } else for (int it = 0; it < entries; it++) {
            if (!(group_max[it * kThreads + tid] >= bd)) continue;
            if (*(volatile int *)&count > kList) {  // only the number above the bound matters now
                if (!(group_max[it * kThreads + tid] > bd)) continue;
            }
            const int v = v0 + tid + it * kGroupVecs * kThreads;
            for (int k = 0; k < kGroupVecs && v + k * kThreads < v1; k++) {
                float f[N];
                unpack<T>(vec[v + k * kThreads], f);
#pragma unroll
                for (int i = 0; i < N; i++)
                    if (f[i] >= bd) offer(f[i], head + (v + k * kThreads) * N + i);
            }
        }
        __syncthreads();
        const int elements = (v1 - v0) * N + (split == 0 ? edge : 0), want = min(p.top, elements);
        int n = count;
        const int n_above = above;
        __syncthreads();
        if (n > kList && n_above <= kList - kMostTop - 2 * N) {
            // too many equal to the bound: the list again with those above it, then the lowest indices equal to it
            if (tid == 0) count = 0;
            __syncthreads();
            auto above_only = [&](float v, int i) {
                if (v > bd) list[atomicAdd(&count, 1)] = key_of(v, i);
            };
            if (split == 0 && tid < edge) above_only(to_f32(x[edge_at(tid)]), edge_at(tid));
            for (int it = 0; it < entries; it++) {
                if (!(group_max[it * kThreads + tid] > bd)) continue;
                const int v = v0 + tid + it * kGroupVecs * kThreads;
                for (int k = 0; k < kGroupVecs && v + k * kThreads < v1; k++) {
                    float f[N];
                    unpack<T>(vec[v + k * kThreads], f);
#pragma unroll
                    for (int i = 0; i < N; i++) above_only(f[i], head + (v + k * kThreads) * N + i);
                }
            }
            __syncthreads();
            // in order of index: the edge before the vectors, the vectors 256 at a time, the edge behind them
            const int need = want - n_above;
            const int b0 = split == 0 ? 0 : head + v0 * N, b1 = split == 0 && p.splits == 1 ? p.vocab : head + v1 * N;
            for (int i0 = b0; taken < need; i0 += kThreads) {
                if (i0 >= b1) break;
                const int i = i0 + tid;
                const bool equal = i < b1 && to_f32(x[i]) == bd;
                const unsigned vote = __ballot_sync(0xffffffffu, equal);
                if (lane == 0) warp_count[warp] = __popc(vote);
                const int had = taken;
                __syncthreads();
                int before = had + __popc(vote & ((1u << lane) - 1)), total = 0;
                for (int w = 0; w < kThreads / 32; w++) {
                    if (w < warp) before += warp_count[w];
                    total += warp_count[w];
                }
                if (equal && before < need) list[n_above + before] = key_of(bd, i);
                __syncthreads();
                if (tid == 0) taken = had + total;
                __syncthreads();
            }
            n = n_above + max(0, min(need, taken));
            if (split == 0 && p.splits > 1) {  // a split row's last elements are split 0's too: candidates as well
                if (tid == 0) count = n;
                __syncthreads();
                if (tid < edge - head && to_f32(x[edge_at(head + tid)]) == bd)
                    list[atomicAdd(&count, 1)] = key_of(bd, edge_at(head + tid));
                __syncthreads();
                n = count;
            }
        }
        if (n >= want && n <= kList) {
            __syncthreads();
            for (int i = tid; i < n; i += kThreads) {
                const unsigned long long key = list[i];
                int above_me = 0;
                for (int j = 0; j < n; j++) above_me += list[j] > key;
                if (above_me < p.top) best[above_me] = key;
            }
            __syncthreads();
        } else {
            // one arg max after another, below the last
            unsigned long long last = ~0ull;
            for (int k = 0; k < want; k++) {
                unsigned long long b = 0;
                auto see = [&](float v, int i) {
                    const unsigned long long key = key_of(v, i);
                    if (key < last && key > b) b = key;
                };
                for (int v = v0 + tid; v < v1; v += kThreads) {
                    float f[N];
                    unpack<T>(vec[v], f);
#pragma unroll
                    for (int i = 0; i < N; i++) see(f[i], head + v * N + i);
                }
                if (split == 0 && tid < edge) see(to_f32(x[edge_at(tid)]), edge_at(tid));
#pragma unroll
                for (int o = 16; o; o >>= 1) {
                    const unsigned long long t = __shfl_xor_sync(0xffffffffu, b, o);
                    b = t > b ? t : b;
                }
                if (lane == 0) round_best[warp] = b;
                __syncthreads();
                for (int w = 0; w < kThreads / 32; w++) b = round_best[w] > b ? round_best[w] : b;
                if (tid == 0) best[k] = b;
                last = b;
                __syncthreads();
            }
        }
    }
    __syncthreads();
    Sums all = cta_sums;
    if (p.splits > 1) {
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        if (split == 0) {
            if (tid == 0) {
                Sums t = all;
                for (int w = 1; w < p.splits; w++) t = joined(t, *cluster.map_shared_rank(&cta_sums, w));
                parts[0] = t;
            }
            if (TOP) {  // the sisters' best, ranked together (splits * top <= 1024 entries)
                const int n = p.splits * p.top;
                for (int i = tid; i < n; i += kThreads) list[i] = *cluster.map_shared_rank(&best[i % p.top], i / p.top);
                __syncthreads();
                for (int i = tid; i < n; i += kThreads) {
                    const unsigned long long key = list[i];
                    int above_me = 0;
                    for (int j = 0; j < n; j++) above_me += list[j] > key;
                    if (key && above_me < p.top) best[above_me] = key;
                }
            }
        }
        cluster.sync();  // no CTA leaves while rank 0 reads it
        if (split) return;
        all = parts[0];
    }
    // a row without a finite logit has no distribution
    const float logz = all.z > 0.0f ? logf(all.z) : __int_as_float(0x7FC00000);
    if (tid == 0 && p.entropy) p.entropy[row] = logz - all.w / all.z;
    for (int i = tid; i < p.nids; i += kThreads) {
        if (i != tid) {  // more tokens than threads
            id = p.ids[(size_t)row * p.nids + i];
            if ((unsigned)id < (unsigned)p.vocab) given = to_f32(x[id]);
        }
        float r = 0.0f;  // -1: no token
        if (id != -1) {
            r = (given - all.m) - logz;
            if ((unsigned)id >= (unsigned)p.vocab) {
                r = __int_as_float(0x7FC00000);
                note(&g_logp_error, kBadToken);
            }
        }
        p.logp[(size_t)row * p.nids + i] = r;
    }
    if (TOP && tid < p.top) {
        const unsigned long long key = best[tid];
        p.top_ids[(size_t)row * p.top + tid] = (int)~(uint32_t)key;
        p.top_logp[(size_t)row * p.top + tid] = (value_of(key) - all.m) - logz;
    }
}

template <typename T, bool TOP, int kThreads>
static cudaError_t launch_threads(Params p, cudaStream_t stream) {
    constexpr int kChunk = kThreads * 32;  // elements of a row of maxima: 32 a thread
    auto kernel = logprobs_kernel<T, TOP, kThreads>;
    // a row over more CTAs while the grid leaves SMs idle and each CTA still has a chunk, or where its maxima would not
    // fit in shared memory
    // (200 rows of fp32: 34 us whole, 27 us in halves that run at once; 148 rows in quarters: 33 us, in halves 25)
    int splits = 1;
    while (splits < 16 && (((long long)p.rows * splits * 2 <= (splits == 1 ? 148 * 3 : 148 * 2) &&
                            (long long)kChunk * splits * 2 <= p.vocab) ||
                           (TOP && (long long)p.vocab / splits / kChunk >= 150)))
        splits *= 2;
    p.splits = splits;
    p.iters = (int)(((long long)p.vocab / splits + kChunk) / kChunk) + 1;
    const size_t smem = TOP ? (size_t)p.iters * kThreads * 4 : 0;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess && smem > 16 * 1024)
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(p.rows * splits));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = splits;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, p);
}

// The rows that whole waves hold, one row a CTA: the time of p.rows rows goes with it, since rows are alike.
template <typename T, bool TOP, int kThreads>
static long long rows_of_waves(const Params &p) {
    static std::atomic<size_t> known{0};
    size_t fixed = known.load(std::memory_order_relaxed);
    if (!fixed) {  // (a query that failed is not kept)
        cudaFuncAttributes a = {};
        if (cudaFuncGetAttributes(&a, logprobs_kernel<T, TOP, kThreads>) == cudaSuccess) known.store(fixed = a.sharedSizeBytes);
        else cudaGetLastError();
    }
    const size_t smem = TOP ? ((size_t)p.vocab / (kThreads * 32) + 2) * kThreads * 4 : 0;
    const long long fit = 228 * 1024 / (long long)(fixed + smem + 1024), most = 768 / kThreads;
    const long long slots = 148 * (fit < 1 ? 1 : fit < most ? fit : most);
    return (p.rows + slots - 1) / slots * slots;
}

template <typename T, bool TOP>
static cudaError_t launch(const Params &p, cudaStream_t stream) {
    // 128 threads a row and more rows an SM, so that the ends of rows (joins, candidates) of some stand beside the streaming
    // of others, unless 256 fill their waves better (bf16, top 20, 128 | 256: 740 rows 49 | 55 us, 888 rows 74 | 60, 1,500
    // rows 112 | 102, 2,000 rows 119 | 128)
    if (rows_of_waves<T, TOP, 128>(p) <= rows_of_waves<T, TOP, 256>(p)) return launch_threads<T, TOP, 128>(p, stream);
    return launch_threads<T, TOP, 256>(p, stream);
}

int *logp_error_word() {
    void *p = nullptr;
    return cudaGetSymbolAddress(&p, g_logp_error) == cudaSuccess ? static_cast<int *>(p) : nullptr;
}

}  // namespace logp

namespace rows {
int *rope_error_word();
int *kv_error_word();
}  // namespace rows
namespace attn {
int *attn_error_word();
int *tc_error_word();
}

// The current device's error words (each source file's own), read and cleared at once: a note that falls between a read and
// a clearing store of two callers would be lost, or one note be told twice.
struct ErrorWords {
    int *at[5];
};
__global__ void take_errors_kernel(const ErrorWords w, int *out) {
    if (threadIdx.x < 5) out[threadIdx.x] = atomicExch(w.at[threadIdx.x], rows::kOk);
}
// Five words of host memory that the device writes, a thread's own.
struct HostWords {
    int *p = nullptr;
    ~HostWords() {
        if (p) cudaFreeHost(p);
    }
};
}  // namespace mvb

using namespace mvb;

extern "C" int mvb_logprobs(const void *x, long long stride, int dtype, int rows, int vocab, const int *ids, int nids,
                            float *logp, float *entropy, int top, int *top_ids, float *top_logp, void *stream) {
    const char *who = "mvb_logprobs";
    if (!rows::known_type(dtype)) {
        set_error("%s: unknown type %d", who, dtype);
        return -1;
    }
    if (rows < 0 || vocab <= 0 || vocab > (1 << 21) || nids < 0 || top < 0 || top > logp::kMostTop || top > vocab ||
        rows > INT_MAX / 16) {
        set_error("%s: unsupported rows=%d vocab=%d ids=%d top=%d (need vocab <= 2097152, top <= min(%d, vocab))", who,
                  rows, vocab, nids, top, logp::kMostTop);
        return -1;
    }
    if (!rows) return 0;
    if (!x || ((uintptr_t)x & (rows::type_bytes(dtype) - 1)) || (nids && (!ids || !logp)) ||
        (top && (!top_ids || !top_logp)) || ((uintptr_t)ids & 3) || ((uintptr_t)logp & 3) || ((uintptr_t)entropy & 3) ||
        ((uintptr_t)top_ids & 3) || ((uintptr_t)top_logp & 3)) {
        set_error("%s: null or misaligned pointer", who);
        return -1;
    }
    logp::Params p = {};
    p.x = x;
    p.stride = stride;
    p.rows = rows;
    p.vocab = vocab;
    p.ids = ids;
    p.nids = nids;
    p.logp = logp;
    p.entropy = entropy;
    p.top = top;
    p.top_ids = top_ids;
    p.top_logp = top_logp;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (dtype == rows::kF32) e = top ? logp::launch<float, true>(p, s) : logp::launch<float, false>(p, s);
    else if (dtype == rows::kBF16)
        e = top ? logp::launch<__nv_bfloat16, true>(p, s) : logp::launch<__nv_bfloat16, false>(p, s);
    else e = top ? logp::launch<__half, true>(p, s) : logp::launch<__half, false>(p, s);
    if (e != cudaSuccess) {
        set_error("%s: launch failed: %s", who, cudaGetErrorString(e));
        return -1;
    }
    return 0;
}

// Synchronizes `stream`; the first bad index that a serving operator met on the device since the last call (and clears it).
extern "C" int mvb_serve_status(void *stream) {
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    static thread_local HostWords host;
    const ErrorWords w = {{rows::rope_error_word(), rows::kv_error_word(), attn::attn_error_word(), attn::tc_error_word(),
                           logp::logp_error_word()}};
    cudaError_t e = w.at[0] && w.at[1] && w.at[2] && w.at[3] && w.at[4] ? cudaSuccess : cudaErrorInvalidSymbol;
    if (e == cudaSuccess && !host.p) e = cudaHostAlloc(&host.p, 5 * sizeof(int), cudaHostAllocPortable | cudaHostAllocMapped);
    if (e == cudaSuccess) {
        take_errors_kernel<<<1, 32, 0, s>>>(w, host.p);
        e = cudaGetLastError();
    }
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    if (e != cudaSuccess) {
        set_error("mvb_serve_status: the stream failed: %s", cudaGetErrorString(e));
        return -1;
    }
    for (int i = 0; i < 5; i++)
        if (host.p[i]) return host.p[i];
    return 0;
}
