// A paged key/value cache held in 8 or 4 bits: quantized as it is written (mvb_kv_append), read back (mvb_kv_read).
//
// Format: the integers of a (page, kv head) are page x head contiguous bytes (head / 2 for 4 bits, two's complement
// nibbles with element 2i low, the .qwb order), the scales page fp32 values. One scale covers one token's head: it then
// factors out of q.k and folds into the softmax weight of v, so that an attention can multiply the integers themselves,
// which 16-bit tensor-core operands hold exactly (per group of 32, as the weights have it, the keys' products would
// have to be scaled group by group).
//     scale = fl32(max |x| / Q), Q = 127 or 7;   integer = rint(x / scale), ties to even;   value = integer * scale
// x is the rotated key in fp64 (the products of an fp32 element with an fp32 cosine are exact there, so each element is
// rounded once), or the value itself: an integer next to a border comes out the same for every order of evaluation. The
// work is done in fp32 all the same: only the elements that may hold the row's maximum, and those within 1e-4 of a border
// (1 in 5,000), are computed in fp64. A row that has an infinity or a NaN (after the rotation in fp32) gets the scale NaN
// and reads back as NaN. All-zero rows have scale 0.
#include <limits.h>

#include "../../include/matvec_b200.h"
#include "mvb_runtime.h"
#include "rope_rows.cuh"

namespace mvb {
namespace rows {

static __device__ int g_kv_error;

struct KvParams {
    uint8_t *kq, *vq;
    float *ks, *vs;
    Batch bt;
    int rows, kv_heads, head;
    // append
    const void *q, *k, *v;
    void *q_out;
    const int *pos;
    const float *rope;
    long long q_stride, k_stride, v_stride, q_out_stride;
    int heads, rot, table_rows, pairs;
    int kv_chunks, q_per, chunks;
    // read
    void *k_out, *v_out;
    long long k_out_stride, v_out_stride;
    int tokens_per_block;
};

// rint(x / scale) in fp64, at most MOST.
template <int MOST>
__device__ __noinline__ float quotient(double x, float scale) {
    if (!(scale > 0.0f)) return 0.0f;
    return (float)fmin(fmax(rint(__ddiv_rn(x, (double)scale)), -(double)MOST), (double)MOST);
}

// Quantizes the rows of a warp (W lanes a row, E elements a lane) and stores integers and scale. f: the elements in fp32
// (with TURN, turned keys within 1.5 ulp of the larger product, else the elements themselves); exact(k): element k in
// fp64, read again from memory, for the few that need it. Every lane of the warp takes part; lanes with on = false hold
// zeros and store nothing.
//
// scale: of turned keys, |f| finds the candidates for the largest element (within 1e-6 of the largest, which covers f's
// error; nearly always one element of the row), their fp64 values decide; rounding to fp32 is monotonic, so the largest of
// the rounded quotients is the rounded largest quotient. (The fp32 division rounds the quotient of an fp32 element as the
// fp64 one followed by a rounding does: 53 bits are enough for that.)
// integers: y = f * (1 / scale) is within MOST * 2^-21 (6.1e-5 for 8 bits) of x / scale, which decides all but the values
// nearer than kNear to a border (1 in 5,000); those take the fp64 quotient, as do scales whose reciprocal leaves fp32's
// range. Adding 1.5 * 2^23 rounds y to an integer (ties to even) that stands in the sum's low byte.
template <int W, int BITS, bool TURN, int E, typename F>
__device__ __forceinline__ void quantize_store(const Row<E> &f, const F &exact, bool on, int l, uint8_t *row,
                                               float *scale_at) {
    constexpr int MOST = BITS == 8 ? 127 : 7;
    constexpr float kNear = MOST * 7.9e-7f;
    uint32_t mine = 0;  // |f| as bits: infinities and NaN come out largest
#pragma unroll
    for (int k = 0; k < E; k++) mine = max(mine, __float_as_uint(f.v[k]) & 0x7FFFFFFFu);
    uint32_t mb = mine;
#pragma unroll
    for (int o = W / 2; o; o >>= 1) mb = max(mb, __shfl_xor_sync(0xffffffffu, mb, o));
    const bool bad = mb >= 0x7F800000u;
    const float m = __uint_as_float(mb);
    float scale;
    if (TURN) {
        const float near = m - fmaxf(m * 1e-6f, 1e-44f);
        scale = 0.0f;
        if (__uint_as_float(mine) >= near && on && !bad) {
            uint32_t candidates = 0;
#pragma unroll
            for (int k = 0; k < E; k++) candidates |= (uint32_t)(fabsf(f.v[k]) >= near) << k;
            double best = 0.0;
            do {
                best = fmax(best, fabs(exact(__ffs(candidates) - 1)));
                candidates &= candidates - 1;
            } while (candidates);
            scale = best > 0.0 ? __double2float_rn(__ddiv_rn(best, (double)MOST)) : 0.0f;
        }
#pragma unroll
        for (int o = W / 2; o; o >>= 1) scale = fmaxf(scale, __shfl_xor_sync(0xffffffffu, scale, o));
    } else {
        scale = __fdiv_rn(m, (float)MOST);
    }
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(scale));  // 1 ulp
    uint32_t n[E];
    float far = scale >= 1e-36f ? 0.0f : 1.0f;  // the largest distance from an integer
#pragma unroll
    for (int k = 0; k < E; k++) {
        const float y = __fmul_rn(f.v[k], inv), t = __fadd_rn(y, 12582912.0f);
        far = fmaxf(far, fabsf(__fsub_rn(y, __fsub_rn(t, 12582912.0f))));
        n[k] = __float_as_uint(t);
    }
    if (far > 0.5f - kNear && !bad && on) {
#pragma unroll
        for (int k = 0; k < E; k++) {
            const float y = __fmul_rn(f.v[k], inv), d = __fsub_rn(y, __fsub_rn(__fadd_rn(y, 12582912.0f), 12582912.0f));
            if (!(scale >= 1e-36f) || fabsf(d) > 0.5f - kNear)
                n[k] = __float_as_uint(__fadd_rn(quotient<MOST>(exact(k), scale), 12582912.0f));
        }
    }
    if (!on) return;
    if (BITS == 8) {
        uint32_t w[E / 4];
#pragma unroll
        for (int k = 0; k < E; k += 4)
            w[k / 4] = __byte_perm(__byte_perm(n[k], n[k + 1], 0x0040), __byte_perm(n[k + 2], n[k + 3], 0x0040), 0x5410);
        if (bad) w[0] = w[E / 4 - 1] = 0;
        if constexpr (E == 8) *reinterpret_cast<uint2 *>(row + 8 * l) = make_uint2(w[0], w[1]);
        else *reinterpret_cast<uint32_t *>(row + 4 * l) = w[0];
    } else {
        uint32_t w = 0;
#pragma unroll
        for (int k = 0; k < E; k++) w |= (n[k] & 15) << (4 * k);
        if (bad) w = 0;
        if constexpr (E == 8) *reinterpret_cast<uint32_t *>(row + 4 * l) = w;
        else *reinterpret_cast<uint16_t *>(row + 2 * l) = (uint16_t)w;
    }
    if (l == 0) *scale_at = bad ? __int_as_float(0x7FC00000) : scale;
}

// One warp: 32 / W heads' keys and values of one token into the cache, or some heads of its queries rotated. Four blocks an
// SM hide more of the rows' loads and of the exchanges of the maxima than the few spills of 64 registers cost (8 prompts of
// 2,000 tokens, 32 + 8 heads of 128, bf16: 88 us against 94 with 80 registers and three blocks).
template <typename T, int W, int BITS, int E>
__global__ void __launch_bounds__(256, 4) kv_append_kernel(const KvParams p) {
    constexpr int R = 32 / W;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = lane & (W - 1), sub = lane / W;
    // a block's warps do alike work on neighbouring tokens (a block of both kinds keeps its queries' warps waiting idle for
    // those that quantize: 14,000 rows of 32 + 8 heads took 179 us so)
    const int chunk = blockIdx.y;
    const long long tok = (long long)blockIdx.x * 8 + warp;
    if (tok >= p.rows) return;
    const int end = p.bt.cu[p.bt.batch];
    if (tok == p.rows - 1 && end > p.rows && lane == 0) note(&g_kv_error, kBadLength);  // rows that the arrays lack
    if (tok >= end || tok < p.bt.cu[0]) return;  // rows of no sequence stay as they are
    const bool on = E * l < p.head, in_rot = E * l < p.rot;
    const bool is_q = chunk >= p.kv_chunks;
    int b = 0;
    long long at = 0;
    if (!is_q || !p.pos) {
        b = sequence_of(p.bt.cu, p.bt.batch, (int)tok);
        if (b >= p.bt.batch) return;
        const int first = p.bt.cu[b];
        if (first < 0 || first > tok) {  // cu that falls, or begins below 0
            if (lane == 0) note(&g_kv_error, kBadLength);
            return;
        }
        at = (long long)p.bt.lens[b] + tok - first;
    }
    Turn<E> t;
#pragma unroll
    for (int k = 0; k < E; k++) t.c[k] = 1.0f, t.s[k] = 0.0f;
    const float *trow = nullptr;
    if (p.rope) {
        const long long pos = p.pos ? p.pos[tok] : at;
        if (pos < 0 || pos >= p.table_rows) {
            if (lane == 0) note(&g_kv_error, kBadPosition);
            return;
        }
        trow = p.rope + pos * p.rot;
        t = load_turn<E>(trow, l, p.rot, p.pairs);
    }
    if (is_q) {
        const int h0 = (chunk - p.kv_chunks) * p.q_per;
        turn_heads<W, E>(static_cast<const T *>(p.q) + tok * p.q_stride + E * l,
                         static_cast<T *>(p.q_out) + tok * p.q_out_stride + E * l, h0, min(h0 + p.q_per, p.heads), p.head,
                         t, l, sub, p.rot, p.pairs);
        return;
    }
    const int h = chunk * R + sub;
    const bool live = on && h < p.kv_heads;
    const size_t src = (size_t)min(h, p.kv_heads - 1) * p.head;
    const T *kr = static_cast<const T *>(p.k) + tok * p.k_stride + src, *vr = static_cast<const T *>(p.v) + tok * p.v_stride + src;
    const Row<E> k = load_row<E>(kr + E * l, live), v = load_row<E>(vr + E * l, live);
    const long long slot = at > INT_MAX ? -1 : slot_of(p.bt, b, (int)at, &g_kv_error);
    if (slot < 0) return;
    const size_t page = (size_t)(slot >> p.bt.page_log2);
    const size_t row = ((page * p.kv_heads + min(h, p.kv_heads - 1)) << p.bt.page_log2) +
                       (size_t)(slot & ((1 << p.bt.page_log2) - 1));
    const int row_bytes = p.head * BITS / 8;
    quantize_store<W, BITS, false>(v, [&](int i) { return (double)to_f32(vr[E * l + i]); }, live, l, p.vq + row * row_bytes,
                                   p.vs + row);
    if (p.rope) {
        const Row<E> y = partners<W>(k, l, p.rot, p.pairs);
        // both products of an fp32 element and an fp32 cosine are exact in fp64: one rounding
        auto exact = [&](int i) {
            const int e = E * l + i;
            const double x = to_f32(kr[e]);
            if (e >= p.rot) return x;
            const bool first = p.pairs ? !(e & 1) : 2 * e < p.rot;
            const int angle = p.pairs ? e / 2 : first ? e : e - p.rot / 2;
            const double other = to_f32(kr[p.pairs ? e ^ 1 : first ? e + p.rot / 2 : e - p.rot / 2]);
            const double s = trow[p.rot / 2 + angle];
            return __fma_rn(x, (double)trow[angle], __dmul_rn(other, first ? -s : s));
        };
        quantize_store<W, BITS, true>(turned(k, y, t, in_rot), exact, live, l, p.kq + row * row_bytes, p.ks + row);
    } else {
        quantize_store<W, BITS, false>(k, [&](int i) { return (double)to_f32(kr[E * l + i]); }, live, l,
                                       p.kq + row * row_bytes, p.ks + row);
    }
}

// Eight elements of a cached row (integer * scale, rounded once to fp32, once more to a 16-bit output).
template <typename T, int BITS>
__device__ __forceinline__ void write8(uint2 u, float scale, T *dst) {
    int n[8];
    if (BITS == 8) {
#pragma unroll
        for (int k = 0; k < 4; k++) {
            n[k] = (int8_t)(u.x >> (8 * k));
            n[4 + k] = (int8_t)(u.y >> (8 * k));
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; k++) n[k] = (int)(u.x << (28 - 4 * k)) >> 28;
    }
    float f[8];
#pragma unroll
    for (int k = 0; k < 8; k++) f[k] = __fmul_rn(__int2float_rn(n[k]), scale);
    if constexpr (sizeof(T) == 4) {
        store4(dst, make_float4(f[0], f[1], f[2], f[3]));
        store4(dst + 4, make_float4(f[4], f[5], f[6], f[7]));
    } else {
        *reinterpret_cast<uint4 *>(dst) =
            make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
    }
}

// One block: the cached rows of some tokens, every head. The tokens' slots are looked up once, a thread each; then W
// lanes (eight elements a lane) copy a (token, head) row of keys and of values, kDeep rows in flight.
constexpr int kReadTokens = 32;  // tokens a block at most
constexpr int kDeep = 4;

template <typename T, int W, int BITS>
__global__ void __launch_bounds__(256) kv_read_kernel(const KvParams p) {
    __shared__ long long slots[kReadTokens];
    const int t0 = blockIdx.x * p.tokens_per_block, tid = threadIdx.x;
    const int nt = min(p.tokens_per_block, p.rows - t0);
    if (tid < nt) {
        const int tok = t0 + tid;
        long long slot = -1;
        const int end = p.bt.cu[p.bt.batch];
        if (tok == p.rows - 1 && end > p.rows) note(&g_kv_error, kBadLength);  // rows that the arrays lack
        if (tok < end && tok >= p.bt.cu[0]) {
            int lo = 0, hi = p.bt.batch;  // the first sequence that ends behind the row
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (p.bt.cu[mid + 1] <= tok) lo = mid + 1;
                else hi = mid;
            }
            if (lo < p.bt.batch) {
                const int first = p.bt.cu[lo];
                const long long at = (long long)p.bt.lens[lo] + tok - first;
                if (first < 0 || first > tok) note(&g_kv_error, kBadLength);  // cu that falls, or begins below 0
                else slot = at > INT_MAX ? -1 : slot_of(p.bt, lo, (int)at, &g_kv_error);
            }
        }
        slots[tid] = slot;
    }
    __syncthreads();
    const int l = tid & (W - 1), units = nt * p.kv_heads, mask = (1 << p.bt.page_log2) - 1;
    const int row_bytes = p.head * BITS / 8;
    if (8 * l >= p.head) return;
    for (int u0 = tid / W; u0 < units; u0 += kDeep * (256 / W)) {
        uint2 kw[kDeep], vw[kDeep];
        float ks[kDeep], vs[kDeep];
        bool live[kDeep];
        int ti[kDeep], h[kDeep];
#pragma unroll
        for (int i = 0; i < kDeep; i++) {
            const int u = u0 + i * (256 / W);
            ti[i] = u / p.kv_heads;
            h[i] = u - ti[i] * p.kv_heads;
            const long long slot = u < units ? slots[ti[i]] : -1;
            live[i] = slot >= 0;
            if (!live[i]) continue;
            const size_t row =
                (((size_t)(slot >> p.bt.page_log2) * p.kv_heads + h[i]) << p.bt.page_log2) + (size_t)(slot & mask);
            const uint8_t *kp = p.kq + row * row_bytes + l * BITS, *vp = p.vq + row * row_bytes + l * BITS;
            if (BITS == 8) {
                kw[i] = *reinterpret_cast<const uint2 *>(kp);
                vw[i] = *reinterpret_cast<const uint2 *>(vp);
            } else {
                kw[i].x = *reinterpret_cast<const uint32_t *>(kp);
                vw[i].x = *reinterpret_cast<const uint32_t *>(vp);
            }
            ks[i] = p.ks[row];
            vs[i] = p.vs[row];
        }
#pragma unroll
        for (int i = 0; i < kDeep; i++) {
            if (!live[i]) continue;
            const size_t o = (size_t)h[i] * p.head + 8 * l;
            write8<T, BITS>(kw[i], ks[i], static_cast<T *>(p.k_out) + (t0 + ti[i]) * p.k_out_stride + o);
            write8<T, BITS>(vw[i], vs[i], static_cast<T *>(p.v_out) + (t0 + ti[i]) * p.v_out_stride + o);
        }
    }
}

template <typename T, int BITS, int E>
static void launch_lanes(const KvParams &p, dim3 grid, cudaStream_t s) {
    const int lanes = (p.head + E - 1) / E;  // the fewest lanes that hold a row
    if (lanes <= 8) kv_append_kernel<T, 8, BITS, E><<<grid, 256, 0, s>>>(p);
    else if (lanes <= 16) kv_append_kernel<T, 16, BITS, E><<<grid, 256, 0, s>>>(p);
    else kv_append_kernel<T, 32, BITS, E><<<grid, 256, 0, s>>>(p);
}

template <typename T, int BITS>
static void launch_append(const KvParams &p, dim3 grid, bool wide, cudaStream_t s) {
    if constexpr (sizeof(T) == 2) {
        if (wide) return launch_lanes<T, BITS, 8>(p, grid, s);
    }
    launch_lanes<T, BITS, 4>(p, grid, s);
}

template <typename T, int BITS>
static void launch_read(const KvParams &p, unsigned grid, cudaStream_t s) {
    if (p.head <= 64) kv_read_kernel<T, 8, BITS><<<grid, 256, 0, s>>>(p);
    else kv_read_kernel<T, 16, BITS><<<grid, 256, 0, s>>>(p);
}

int *kv_error_word() {
    void *p = nullptr;
    return cudaGetSymbolAddress(&p, g_kv_error) == cudaSuccess ? static_cast<int *>(p) : nullptr;
}

// The cache's and the batch's arguments, checked; fills p. 0, or -1 after set_error().
int kv_check(const char *who, KvParams &p, void *kq, float *ks, void *vq, float *vs, int pages, int page, int kv_heads,
             int head, int bits, const int *table, int table_cols, const int *cu, const int *lens, int batch, int rows) {
    if (bits != 4 && bits != 8) {
        set_error("%s: unsupported bits=%d (need 4 or 8)", who, bits);
        return -1;
    }
    if (pages <= 0 || page < 16 || page > 1024 || (page & (page - 1)) || kv_heads <= 0 || head < 16 || head > 128 ||
        head % 16 || table_cols <= 0 || batch <= 0 || rows < 0) {
        set_error("%s: unsupported pages=%d page=%d kv_heads=%d head=%d table columns=%d batch=%d rows=%d (need page a "
                  "power of two in 16 .. 1024, head a multiple of 16 in 16 .. 128)",
                  who, pages, page, kv_heads, head, table_cols, batch, rows);
        return -1;
    }
    if (!kq || !ks || !vq || !vs || !table || !cu || !lens || ((uintptr_t)kq & 15) || ((uintptr_t)vq & 15) ||
        ((uintptr_t)ks & 15) || ((uintptr_t)vs & 15) || ((uintptr_t)table & 3) || ((uintptr_t)cu & 3) ||
        ((uintptr_t)lens & 3)) {
        set_error("%s: null or misaligned pointer (cache 16 bytes, table, cu and lens 4)", who);
        return -1;
    }
    p.kq = static_cast<uint8_t *>(kq);
    p.ks = ks;
    p.vq = static_cast<uint8_t *>(vq);
    p.vs = vs;
    p.bt.cu = cu;
    p.bt.lens = lens;
    p.bt.table = table;
    p.bt.batch = batch;
    p.bt.table_cols = table_cols;
    p.bt.pages = pages;
    p.bt.page_log2 = 31 - __builtin_clz((unsigned)page);
    p.rows = rows;
    p.kv_heads = kv_heads;
    p.head = head;
    return 0;
}

}  // namespace rows
}  // namespace mvb

using namespace mvb;
using namespace mvb::rows;

extern "C" int mvb_kv_append(void *kq, float *ks, void *vq, float *vs, int pages, int page, int kv_heads, int head,
                             int bits, const int *table, int table_cols, const int *cu, const int *lens, int batch,
                             int rows, const void *k, long long k_stride, const void *v, long long v_stride, int dtype,
                             const float *rope, const int *pos, int rot, int table_rows, int layout, const void *q,
                             long long q_stride, void *q_out, long long q_out_stride, int heads, void *stream) {
    const char *who = "mvb_kv_append";
    KvParams p = {};
    if (kv_check(who, p, kq, ks, vq, vs, pages, page, kv_heads, head, bits, table, table_cols, cu, lens, batch, rows))
        return -1;
    if (!known_type(dtype) || (layout != 0 && layout != 1)) {
        set_error("%s: unknown type %d or layout %d", who, dtype, layout);
        return -1;
    }
    if (rope ? rot <= 0 || rot % 8 || rot > head || table_rows < 0 : q != nullptr) {
        set_error("%s: unsupported rot=%d (a multiple of 8, at most head), or queries without a rope table", who, rot);
        return -1;
    }
    if (!rows) return 0;
    const uintptr_t need = 4 * type_bytes(dtype) - 1;
    if (!k || !v || ((uintptr_t)k & need) || ((uintptr_t)v & need) || ((uintptr_t)rope & 15) || ((uintptr_t)pos & 3) ||
        k_stride % 4 || v_stride % 4) {
        set_error("%s: null or misaligned pointer or stride (k and v four elements, rope 16 bytes)", who);
        return -1;
    }
    if (q && (!q_out || heads <= 0 || ((uintptr_t)q & need) || ((uintptr_t)q_out & need) || q_stride % 4 ||
              q_out_stride % 4)) {
        set_error("%s: queries need q_out and heads=%d > 0, both aligned to four elements", who, heads);
        return -1;
    }
    p.k = k;
    p.v = v;
    p.q = q;
    p.q_out = q_out;
    p.k_stride = k_stride;
    p.v_stride = v_stride;
    p.q_stride = q_stride;
    p.q_out_stride = q_out_stride;
    p.pos = pos;
    p.rope = rope;
    p.rot = rope ? rot : 0;
    p.table_rows = table_rows;
    p.pairs = layout;
    p.heads = q ? heads : 0;
    // 16 bytes a lane where everything is a multiple of that
    bool wide = dtype != kF32 && (!rope || rot % 16 == 0) && k_stride % 8 == 0 && v_stride % 8 == 0 &&
                !(((uintptr_t)k | (uintptr_t)v) & 15);
    if (q) wide = wide && q_stride % 8 == 0 && q_out_stride % 8 == 0 && !(((uintptr_t)q | (uintptr_t)q_out) & 15);
    const int lane_elems = wide ? 8 : 4, r = 32 / (head <= 8 * lane_elems ? 8 : head <= 16 * lane_elems ? 16 : 32);
    // one pass of a warp a chunk; where the machine is full anyway, 8 passes of a token's queries (its position and angles
    // are then looked up once for them)
    const bool full = rows >= 148 * 16;
    p.q_per = full ? 8 * r : r;
    p.kv_chunks = (kv_heads + r - 1) / r;
    p.chunks = p.kv_chunks + (p.heads + p.q_per - 1) / p.q_per;
    if (p.chunks > 65535) {
        set_error("%s: kv_heads=%d heads=%d are too many for one call", who, kv_heads, p.heads);
        return -1;
    }
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const dim3 grid((unsigned)(((long long)rows + 7) / 8), p.chunks);
    if (bits == 8) {
        if (dtype == kF32) launch_append<float, 8>(p, grid, wide, s);
        else if (dtype == kBF16) launch_append<__nv_bfloat16, 8>(p, grid, wide, s);
        else launch_append<__half, 8>(p, grid, wide, s);
    } else {
        if (dtype == kF32) launch_append<float, 4>(p, grid, wide, s);
        else if (dtype == kBF16) launch_append<__nv_bfloat16, 4>(p, grid, wide, s);
        else launch_append<__half, 4>(p, grid, wide, s);
    }
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) {
        set_error("%s: launch failed: %s", who, cudaGetErrorString(e));
        return -1;
    }
    return 0;
}

extern "C" int mvb_kv_read(const void *kq, const float *ks, const void *vq, const float *vs, int pages, int page,
                           int kv_heads, int head, int bits, const int *table, int table_cols, const int *cu,
                           const int *lens, int batch, int rows, void *k_out, long long k_stride, void *v_out,
                           long long v_stride, int dtype, void *stream) {
    const char *who = "mvb_kv_read";
    KvParams p = {};
    if (kv_check(who, p, const_cast<void *>(kq), const_cast<float *>(ks), const_cast<void *>(vq),
                 const_cast<float *>(vs), pages, page, kv_heads, head, bits, table, table_cols, cu, lens, batch, rows))
        return -1;
    if (!known_type(dtype)) {
        set_error("%s: unknown type %d", who, dtype);
        return -1;
    }
    if (!rows) return 0;
    const int esz = type_bytes(dtype);
    if (!k_out || !v_out || ((uintptr_t)k_out & 15) || ((uintptr_t)v_out & 15) || k_stride * esz % 16 ||
        v_stride * esz % 16) {
        set_error("%s: null or misaligned output or stride (16 bytes)", who);
        return -1;
    }
    p.k_out = k_out;
    p.v_out = v_out;
    p.k_out_stride = k_stride;
    p.v_out_stride = v_stride;
    // as many tokens a block as leave four blocks an SM, 32 at most
    int per = rows / (148 * 4);
    p.tokens_per_block = per < 1 ? 1 : per > kReadTokens ? kReadTokens : per;
    const unsigned grid = (unsigned)(((long long)rows + p.tokens_per_block - 1) / p.tokens_per_block);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (bits == 8) {
        if (dtype == kF32) launch_read<float, 8>(p, grid, s);
        else if (dtype == kBF16) launch_read<__nv_bfloat16, 8>(p, grid, s);
        else launch_read<__half, 8>(p, grid, s);
    } else {
        if (dtype == kF32) launch_read<float, 4>(p, grid, s);
        else if (dtype == kBF16) launch_read<__nv_bfloat16, 4>(p, grid, s);
        else launch_read<__half, 4>(p, grid, s);
    }
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) {
        set_error("%s: launch failed: %s", who, cudaGetErrorString(e));
        return -1;
    }
    return 0;
}
