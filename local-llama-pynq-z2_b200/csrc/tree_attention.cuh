// Shared by the two kernels of mvb_tree_attention (tree_attention.cu: few query rows; tree_attention_tc.cu: many).
#pragma once
#include "rows.cuh"

namespace mvb {
namespace attn {

struct AttnParams {
    const void *q;
    void *out;
    float *lse;  // or null
    const uint8_t *kq, *vq;
    const float *ks, *vs;
    rows::Batch bt;
    const unsigned long long *tree;  // or null: each new token sees those before it and itself
    long long q_stride, out_stride;
    float scale_log2;  // the softmax scale times log2(e)
    int words, rows, heads, kv_heads, group, head, max_new, qtiles;
    // A sequence's keys lie over `splits` CTAs of a cluster (blockIdx.x % splits), joined there, and, where few sequences leave
    // SMs idle that clusters do not reach, over `supers` such clusters (blockIdx.x / splits), whose results go to `work`
    // and are joined by a second kernel: [supers][rows][heads] x head fp32, then [supers][rows][heads] x (max, sum).
    int splits, supers;
    float *work;
    size_t work_bytes;
};

__device__ __forceinline__ float2 *work_ml(const AttnParams &p) {
    return reinterpret_cast<float2 *>(p.work + (size_t)p.supers * p.rows * p.heads * p.head);
}
inline size_t work_need(const AttnParams &p, int supers) {
    return (size_t)supers * p.rows * p.heads * (p.head + 2) * 4;
}
// The second kernel: p.supers parts of every row joined into p.out and p.lse.
cudaError_t launch_join(const AttnParams &p, int dtype, cudaStream_t s);

// One sequence of the batch, its index arrays checked (a value out of range is noted and clamped: no access leaves
// the arrays, and mvb_serve_status tells).
struct Sequence {
    int row0, n, ctx, len;  // first row, new tokens, cached positions before them, ctx + n
};

__device__ __forceinline__ Sequence sequence_at(const AttnParams &p, int b, int *error) {
    Sequence s;
    s.row0 = p.bt.cu[b];
    const int end = p.bt.cu[b + 1];
    s.ctx = p.bt.lens[b];
    bool ok = s.row0 >= 0 && end >= s.row0 && end <= p.rows && end - s.row0 <= p.max_new && s.ctx >= 0;
    s.n = ok ? end - s.row0 : 0;
    const long long most = (long long)p.bt.table_cols << p.bt.page_log2;
    if (ok && (long long)s.ctx + s.n > most) ok = false, s.n = 0;
    if (!ok) rows::note(error, rows::kBadLength);
    s.len = s.ctx + s.n;
    return s;
}

// A page that the table names: page 0 with the error noted where there is none.
__device__ __forceinline__ int checked_page(const AttnParams &p, int pg, int *error) {
    if ((unsigned)pg < (unsigned)p.bt.pages) return pg;
    rows::note(error, rows::kBadPage);
    return 0;
}
// The page of position pos (in range of the table).
__device__ __forceinline__ int page_of(const AttnParams &p, int b, int pos, int *error) {
    return checked_page(p, p.bt.table[(size_t)b * p.bt.table_cols + (pos >> p.bt.page_log2)], error);
}

// Whether new token i of the sequence may see position t.
__device__ __forceinline__ bool allowed(const AttnParams &p, const Sequence &s, int i, int t) {
    if (t < s.ctx) return true;
    const int j = t - s.ctx;
    if (j >= s.n || i >= s.n) return false;
    if (!p.tree) return j <= i;
    if ((j >> 6) >= p.words) return false;
    return (p.tree[(size_t)(s.row0 + i) * p.words + (j >> 6)] >> (j & 63)) & 1;
}

__device__ __forceinline__ float exp2_fast(float x) {  // 2 ulp; exp2(-inf) = 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 2^k as fp32 for k in [-126, 127].
__device__ __forceinline__ float pow2(int k) { return __int_as_float((k + 127) << 23); }

// The same of an integer-valued float of that range.
__device__ __forceinline__ float pow2_of(float k) {
    return __int_as_float(__float_as_int(__fadd_rn(k, 12582912.0f + 127.0f)) << 23);
}

// Biased exponent of |x| (0 for zero and subnormals, 255 for infinities and NaN).
__device__ __forceinline__ int exponent_of(float x) { return (__float_as_int(x) >> 23) & 255; }

// The unit of a row's sums: l = sum of 2^(s + b) over its scores s (log2), O = sum of P' v with P' = 2^(s + b) vs in fp16. b
// keeps every P' below 2^kTop (and every weight below 2^kSumTop); when it has to fall, the row's largest P' so far comes near
// 2^(kTop - lazy). fp16's steps below 2^-14 are 2^-24, so no weight is off by more than 2^(lazy - 40) of the row's largest
// weight times value scale. Only weights and scales that the row sees count: a key that the mask hides from it leaves b
// where it is, and so does one that stands far above the rest while its value is near zero. b is a whole number, so that O and
// l change by exact factors (of scores above 2^24, whose spacing leaves nothing else, minus the score); infinite while the
// row has seen none.
__host__ __device__ constexpr float lazy(int parts) { return parts == 2 ? 9.0f : 13.0f; }
constexpr float kTop = 15.99f, kSumTop = 100.0f;
// What the largest score plus b may reach beside value scales up to vmax before `moved` has to be asked.
__device__ __forceinline__ float unit_limit(float vmax) { return fminf(kSumTop, (kTop - 0.005f) - __log2f(vmax)); }
// log2 of a value scale, for scores plus that: nothing where the scale is infinite.
__device__ __forceinline__ float log_scale(float vs) { return fabsf(vs) < INFINITY ? __log2f(fabsf(vs)) : -INFINITY; }
// 2^(s - t) vs for the row's largest score t; nothing where the scale is infinite or the score hidden.
__device__ __forceinline__ float product_of(float s, float rf, float t, float vs) {
    const float w = __fmul_rn(exp2_fast(__fmaf_rn(s, rf, -t)), fabsf(vs));
    return w < INFINITY ? w : 0.0f;
}
// b where the row meets scores up to t and products up to 2^top (rounded at a score's spacing, of which whole numbers are
// multiples: where b stays, no product reaches 2^16).
template <int PP>  // parts of P'
__device__ __forceinline__ float moved(float b, float t, float top) {
    float to = b;
    if (t + b > kSumTop) to = floorf(__fsub_rd(kSumTop - 4.0f, t));
    if (top + b > kTop) to = fminf(to, floorf(__fsub_rd(16.0f - lazy(PP), top)));
    // (value scales above 2^100: rather a weight below 2^-122 lost than all of them)
    return to < b ? fminf(b, fmaxf(to, ceilf(-122.0f - t))) : b;
}
// The factor of l and O; what has seen nothing is zero.
__device__ __forceinline__ float unit_factor(float b, float to) {
    const float k = to - b;
    return b == INFINITY ? 1.0f : k >= -126.0f ? pow2_of(k) : 0.0f;
}
__device__ __forceinline__ float or_zero(float b) { return b == INFINITY ? 0.0f : b; }
// A sum l in b's unit as (max, sum in its unit): 2^max * sum with sum in [1, 2).
__device__ __forceinline__ float2 normal_sum(float b, float l) {
    const float k = (float)(exponent_of(l) - 127);
    return l == 0.0f ? make_float2(-INFINITY, 0.0f) : make_float2(k - b, l * pow2_of(-k));
}

// Bytes 0 and 2 of a word (int8) as an exact half2: the byte with its sign bit flipped in the low mantissa of 1024 is
// 1024 + (v + 128). One logic operation takes the bytes out, flips the signs and puts the exponents in.
__device__ __forceinline__ uint32_t bytes_to_half2(uint32_t x) {
    uint32_t h = (x & 0x00FF00FFu) ^ 0x64806480u;
    const uint32_t bias = 0x64806480u;  // 1152
    asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(h) : "r"(bias));
    return h;
}

// Nibbles k and k + 4 of a word (int4) as an exact half2: 1024 + (v + 8).
__device__ __forceinline__ uint32_t nibbles_to_half2(uint32_t x, int k) {
    uint32_t h = ((x >> (4 * k)) & 0x000F000Fu) ^ 0x64086408u;
    const uint32_t bias = 0x64086408u;  // 1032
    asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(h) : "r"(bias));
    return h;
}

// Tiles of `tile` query rows of a sequence with max_new new tokens into p.qtiles; false where a grid cannot hold them.
inline bool tiles_fit(AttnParams &p, int tile) {
    const long long n = ((long long)p.max_new * p.group + tile - 1) / tile;
    p.qtiles = (int)n;
    return n * p.kv_heads <= 65535;
}
constexpr cudaError_t kTooManyRows = cudaErrorInvalidConfiguration;

constexpr int kMaxSplits = 16, kMaxSupers = 8;
int most_supers(const AttnParams &p);

// CTAs of `kernel` in clusters of n that the current device holds at once (0 where none fits). Looked up once a kernel,
// size and device: clusters live inside a GPC, so that sizes which do not divide its SMs leave some idle.
int cluster_slots(const void *kernel, int n, int threads, size_t smem);

// Over how many CTAs of a cluster (splits) and how many clusters (supers, at most most_supers) a sequence's keys are split,
// so that the estimated time is least: `base` jobs without a split, `steps` units of work each for the longest sequence,
// `fixed` units to start, fill and join a CTA (`more` where the CTAs exceed one wave), `each` for every CTA of the cluster
// that it is joined with, and `join` for a second kernel, at least `least` units a CTA. All in one wave: whole units. More,
// of one sequence: its jobs are alike and run in whole waves. Several: three quarters of the longest on average, in no
// order, and the last jobs end a third of a job apart.
struct Split {
    int splits, supers;
};
template <typename F>
inline Split choose_splits(long long base, int batch, double steps, double fixed, double more, double each,
                           double join, double least, int most_supers, const F &slots_of) {
    Split best = {1, 1};
    double best_time = 1e300;
    for (int n = 1; n <= kMaxSplits; n++) {
        if (n > 1 && steps < least * n) break;
        const int slots = slots_of(n);
        if (slots < n) continue;
        for (int m = 1; m <= most_supers; m++) {
            if (m > 1 && steps < least * n * m) break;
            const double fill = (double)base * n * m / slots, units = steps / (n * m);
            const double job = (fill > 1.0 ? units + more : ceil(units) + fixed) + n * each;
            if (each > 0.0 && fill <= 1.0 && (n & (n - 1))) continue;  // clusters of 6 or 12 take longer than of 8 or 16
            double time = job;
            if (fill > 1.0) time = batch == 1 ? (double)((base * n * m + slots - 1) / slots) * job
                                              : (0.75 * fill > 1.0 ? 0.75 * fill : 1.0) * job + job / 3;
            if (m > 1) time += join;
            if (time < best_time * 0.999) best_time = time, best = Split{n, m};
            if (fill > 2.0) break;
        }
    }
    return best;
}

// The kernel for many query rows; returns the CUDA error of its launch.
cudaError_t launch_tc(const AttnParams &p, int dtype, int bits, int max_len, cudaStream_t s);

}  // namespace attn
}  // namespace mvb
