// Log probabilities of given tokens, the entropy and the most probable tokens of rows of logits (mvb_logprobs).
//
//     lse = m + ln z,  m = max x,  z = sum exp(x - m);   logp[id] = (x[id] - m) - ln z
//     entropy = -sum p ln p = ln z - (sum (x - m) exp(x - m)) / z
//     top: the `top` largest logits by (value, lowest index first), with their log probabilities
//
// One pass over the logits: each thread keeps (m, z, w = sum (x - m) exp(x - m)) of its elements, moved to a new maximum
// once per 4 vectors, and for the top tokens only the maximum of those 4 vectors (one shared-memory word per 16 or 32
// elements), so that the streaming loop has no candidate lists and no barriers. Afterwards the top-th largest of the
// threads' own maxima is a lower bound of the top-th largest element; the few vectors whose maximum reaches it are read
// again (from L2) and their elements that reach it ranked. Rows with more such elements than the list holds (a
// vocabulary masked to a few tokens: the rest all equal) take the elements above the bound, then those equal to it in
// the order of their index; where even the former overflow, `top` rounds of an arg max.
// A few rows: a row is split over a cluster of up to 16 CTAs, joined through distributed shared memory in rank order.
// Bound: the logits are read once; the exponentials (one a logit, 16 per clock and SM) come close for 16-bit types.
#include <cooperative_groups.h>
#include <limits.h>
#include <math.h>

#include "../../include/matvec_b200.h"
#include "mvb_runtime.h"
#include "rows.cuh"

namespace mvb {
namespace logp {

using namespace rows;
namespace cg = cooperative_groups;

static __device__ int g_logp_error;

constexpr int kThreads = 256;
constexpr int kVecs = 4;      // 16-byte vectors a thread has in flight (a group: one maximum)
constexpr int kList = 2048;   // candidates
constexpr int kMostTop = 64;
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

template <typename T>
__device__ __forceinline__ void unpack(const uint4 &u, float (&f)[Vec<T>::kN]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (sizeof(T) == 4) {
            f[i] = __uint_as_float(w[i]);
        } else if constexpr (Type<T>::kId == kBF16) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        } else {
            const float2 h = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            f[2 * i] = h.x;
            f[2 * i + 1] = h.y;
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

template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads, 4) logprobs_kernel(const Params p) {
    constexpr int N = Vec<T>::kN;
    extern __shared__ __align__(16) float group_max[];  // [iters][kThreads], TOP only
    __shared__ Sums parts[kThreads / 32];
    __shared__ Sums cta_sums;
    __shared__ __align__(16) float thread_max[kThreads];
    __shared__ unsigned long long list[TOP ? kList : 1], best[TOP ? kMostTop : 1];
    __shared__ unsigned long long round_best[kThreads / 32];
    __shared__ float bound;
    __shared__ int count, above, taken, warp_count[kThreads / 32];

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
    for (int it = 0, v = v0 + tid; v < v1; it++, v += kVecs * kThreads) {
        uint4 u[kVecs];
        const int left = (v1 - v + kThreads - 1) / kThreads;  // vectors of this thread from here on
#pragma unroll
        for (int k = 0; k < kVecs; k++)
            if (k < left) u[k] = load_stream(vec + v + k * kThreads);
        float f[kVecs][N];
        float g = -INFINITY;
#pragma unroll
        for (int k = 0; k < kVecs; k++) {
            if (k < left) {
                unpack<T>(u[k], f[k]);
            } else {
#pragma unroll
                for (int i = 0; i < N; i++) f[k][i] = -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < N; i++) g = fmaxf(g, f[k][i]);
        }
        if (TOP) group_max[it * kThreads + tid] = g;
        seen = it + 1;
        mine = fmaxf(mine, g);
        if (g > s.m) move_to(s, g);
        const float base = s.m == -INFINITY ? 0.0f : s.m;
        float z = 0.0f, w = 0.0f;
#pragma unroll
        for (int k = 0; k < kVecs; k++)
#pragma unroll
            for (int i = 0; i < N; i++) {
                const float d = below(f[k][i], base), e = exp_fast(d);
                z += e;
                w = __fmaf_rn(d, e, w);
            }
        s.z += z;
        s.w += w;
    }
    if (split == 0 && tid < edge) {
        const float f = to_f32(x[edge_at(tid)]);
        if (f > s.m) move_to(s, f);
        const float d = below(f, s.m == -INFINITY ? 0.0f : s.m), e = exp_fast(d);
        s.z += e;
        s.w = __fmaf_rn(d, e, s.w);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const Sums t = {__shfl_xor_sync(0xffffffffu, s.m, o), __shfl_xor_sync(0xffffffffu, s.z, o),
                        __shfl_xor_sync(0xffffffffu, s.w, o)};
        s = joined(s, t);
    }
    if (lane == 0) parts[warp] = s;
    if (TOP) thread_max[tid] = mine;
    if (tid == 0) {
        bound = -INFINITY;
        count = above = taken = 0;
    }
    if (TOP && tid < kMostTop) best[tid] = 0;
    __syncthreads();
    if (tid == 0) {
        Sums t = parts[0];
#pragma unroll
        for (int w = 1; w < kThreads / 32; w++) t = joined(t, parts[w]);
        cta_sums = t;
    }
    if (TOP) {
        // the top-th largest of the threads' maxima
        int rank = 0;
        for (int i = 0; i < kThreads / 4; i++) {
            const float4 o = reinterpret_cast<const float4 *>(thread_max)[i];
            rank += (o.x > mine || (o.x == mine && 4 * i < tid)) + (o.y > mine || (o.y == mine && 4 * i + 1 < tid)) +
                    (o.z > mine || (o.z == mine && 4 * i + 2 < tid)) + (o.w > mine || (o.w == mine && 4 * i + 3 < tid));
        }
        if (rank == p.top - 1) bound = mine;
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
        for (int it = 0; it < seen; it++) {
            if (!(group_max[it * kThreads + tid] >= bd)) continue;
            if (*(volatile int *)&count > kList) {  // only the number above the bound matters now
                if (!(group_max[it * kThreads + tid] > bd)) continue;
            }
            const int v = v0 + tid + it * kVecs * kThreads;
            for (int k = 0; k < kVecs && v + k * kThreads < v1; k++) {
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
            for (int it = 0; it < seen; it++) {
                if (!(group_max[it * kThreads + tid] > bd)) continue;
                const int v = v0 + tid + it * kVecs * kThreads;
                for (int k = 0; k < kVecs && v + k * kThreads < v1; k++) {
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
        const int id = p.ids[(size_t)row * p.nids + i];
        float r = 0.0f;  // -1: no token
        if (id != -1) {
            if ((unsigned)id < (unsigned)p.vocab) {
                r = (to_f32(x[id]) - all.m) - logz;
            } else {
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

template <typename T, bool TOP>
static cudaError_t launch(Params p, cudaStream_t stream) {
    constexpr int N = Vec<T>::kN, kChunk = kThreads * kVecs * N;
    auto kernel = logprobs_kernel<T, TOP>;
    // a row over more CTAs while the grid leaves SMs idle and each CTA still has a chunk, or where its maxima would not
    // fit in shared memory
    int splits = 1;
    while (splits < 16 && (((long long)p.rows * splits * 2 <= 148 * 2 && (long long)kChunk * splits * 2 <= p.vocab) ||
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

int logp_take_error(cudaStream_t s) {
    int v = 0;
    if (cudaMemcpyFromSymbolAsync(&v, g_logp_error, sizeof v, 0, cudaMemcpyDeviceToHost, s) != cudaSuccess ||
        cudaStreamSynchronize(s) != cudaSuccess)
        return -1;
    const int z = 0;
    if (v && (cudaMemcpyToSymbolAsync(g_logp_error, &z, sizeof z, 0, cudaMemcpyHostToDevice, s) != cudaSuccess ||
              cudaStreamSynchronize(s) != cudaSuccess))
        return -1;
    return v;
}

}  // namespace logp

namespace rows {
int rope_take_error(cudaStream_t s);
int kv_take_error(cudaStream_t s);
}  // namespace rows
namespace attn {
int attn_take_error(cudaStream_t s);
}
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

// Synchronizes `stream`; the first bad index that a serving operator met since the last call (and clears it).
extern "C" int mvb_serve_status(void *stream) {
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    int first = 0;
    for (auto take : {rows::rope_take_error, rows::kv_take_error, attn::attn_take_error, logp::logp_take_error}) {
        const int v = take(s);
        if (v < 0) {
            set_error("mvb_serve_status: the stream failed: %s", cudaGetErrorString(cudaGetLastError()));
            return -1;
        }
        if (!first) first = v;
    }
    return first;
}
