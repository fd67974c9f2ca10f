// A paged key/value cache held in 8 or 4 bits: quantized as it is written (mvb_kv_append), read back (mvb_kv_read).
//
// Format: the integers of a (page, kv head) are page x head contiguous bytes (head / 2 for 4 bits, two's complement
// nibbles with element 2i low, the .qwb order), the scales page fp32 values. One scale covers one token's head: it then
// factors out of q.k and folds into the softmax weight of v, so that an attention can multiply the integers themselves,
// which 16-bit tensor-core operands hold exactly (per group of 32, as the weights have it, the keys' products would
// have to be scaled group by group).
//     scale = fl32(max |x| / Q), Q = 127 or 7;   integer = rint(x / scale), ties to even;   value = integer * scale
// x is the rotated key in fp64 (the products of an fp32 element with an fp32 cosine are exact there, so each element is
// rounded once), or the value itself: an integer next to a border comes out the same for every order of evaluation. A row
// with an infinity or a NaN gets the scale NaN and reads back as NaN. All-zero rows have scale 0.
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
    int kv_per, kv_chunks, q_per, chunks;
    // read
    void *k_out, *v_out;
    long long k_out_stride, v_out_stride;
    int tokens_per_block;
};

// rint(x / scale), |.| <= MOST. y = x * (1 / scale) in fp32 is within 127 * 3 * 2^-24 < 2.3e-5 of the quotient, which
// decides all but the values within 1e-4 of a border; those (1 in 5,000) take the fp64 quotient, as do scales whose
// reciprocal leaves fp32's range.
template <int MOST>
__device__ __forceinline__ int quantized(double x, float xf, float scale, float inv) {
    const float y = __fmul_rn(xf, inv);
    float n = rintf(y);
    if (scale < 1e-36f || fabsf(fabsf(__fsub_rn(y, n)) - 0.5f) < 1e-4f) {
        if (!(scale > 0.0f)) return 0;
        n = (float)rint(__ddiv_rn(x, (double)scale));
    }
    return max(-MOST, min(MOST, (int)n));
}

// Quantizes the rows of a warp (W lanes a row, four elements a lane) and stores integers and scale. x in fp64; every lane
// of the warp takes part; lanes with on = false hold zeros and store nothing.
template <int W, int BITS>
__device__ __forceinline__ void quantize_store(const double (&x)[4], bool on, int l, uint8_t *row, float *scale_at) {
    constexpr int MOST = BITS == 8 ? 127 : 7;
    double m = fmax(fmax(fabs(x[0]), fabs(x[1])), fmax(fabs(x[2]), fabs(x[3])));
    // x - x is 0 for finite x, NaN else
    bool bad = !((x[0] - x[0]) + (x[1] - x[1]) + (x[2] - x[2]) + (x[3] - x[3]) == 0.0);
#pragma unroll
    for (int o = W / 2; o; o >>= 1) {
        m = fmax(m, __shfl_xor_sync(0xffffffffu, m, o));
        bad |= (bool)__shfl_xor_sync(0xffffffffu, (int)bad, o);
    }
    float scale = __double2float_rn(__ddiv_rn(m, (double)MOST));
    const float inv = __frcp_rn(scale);
    int n[4];
#pragma unroll
    for (int k = 0; k < 4; k++) n[k] = bad ? 0 : quantized<MOST>(x[k], __double2float_rn(x[k]), scale, inv);
    if (!on) return;
    if (BITS == 8)
        *reinterpret_cast<uint32_t *>(row + 4 * l) =
            (n[0] & 255) | (n[1] & 255) << 8 | (n[2] & 255) << 16 | (uint32_t)n[3] << 24;
    else
        *reinterpret_cast<uint16_t *>(row + 2 * l) =
            (uint16_t)((n[0] & 15) | (n[1] & 15) << 4 | (n[2] & 15) << 8 | (n[3] & 15) << 12);
    if (l == 0) *scale_at = bad ? __int_as_float(0x7FC00000) : scale;
}

// One warp: some heads' keys and values of one token into the cache, or some heads of its queries rotated.
template <typename T, int W, int BITS>
__global__ void __launch_bounds__(256) kv_append_kernel(const KvParams p) {
    constexpr int R = 32 / W;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = lane & (W - 1), sub = lane / W;
    const long long item = (long long)blockIdx.x * 8 + warp;
    const int tok = (int)(item / p.chunks), chunk = (int)(item - (long long)tok * p.chunks);
    if (tok >= p.rows || tok >= p.bt.cu[p.bt.batch]) return;  // rows behind the last sequence stay as they are
    const bool on = 4 * l < p.head;
    const bool is_q = chunk >= p.kv_chunks;
    int b = 0;
    long long at = 0;
    if (!is_q || !p.pos) {
        b = sequence_of(p.bt.cu, p.bt.batch, tok);
        if (b >= p.bt.batch) return;
        at = (long long)p.bt.lens[b] + tok - p.bt.cu[b];
    }
    Turn t;
    t.c = make_float4(1.0f, 1.0f, 1.0f, 1.0f);
    t.s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (p.rope) {
        const long long pos = p.pos ? p.pos[tok] : at;
        if (pos < 0 || pos >= p.table_rows) {
            if (lane == 0) note(&g_kv_error, kBadPosition);
            return;
        }
        if (on) t = load_turn(p.rope + pos * p.rot, l, p.rot, p.pairs);
    }
    if (is_q) {
        const int h0 = (chunk - p.kv_chunks) * p.q_per, h1 = min(h0 + p.q_per, p.heads);
        const T *x = static_cast<const T *>(p.q) + tok * p.q_stride + 4 * l;
        T *out = static_cast<T *>(p.q_out) + tok * p.q_out_stride + 4 * l;
        constexpr int U = 4;
        for (int h = h0; h < h1; h += U * R) {
            float4 v[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int hh = h + u * R + sub;
                v[u] = on && hh < h1 ? load4(x + (size_t)hh * p.head) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int hh = h + u * R + sub;
                const float4 y = partners<W>(v[u], l, p.rot, p.pairs);
                if (on && hh < h1) store4(out + (size_t)hh * p.head, turned(v[u], y, t, l, p.rot, p.pairs));
            }
        }
        return;
    }
    const long long slot = at > INT_MAX ? -1 : slot_of(p.bt, b, (int)at, &g_kv_error);
    if (slot < 0) return;
    const int mask = (1 << p.bt.page_log2) - 1;
    const size_t page = (size_t)(slot >> p.bt.page_log2);
    const int row_bytes = p.head * BITS / 8;
    const int h0 = chunk * p.kv_per, h1 = min(h0 + p.kv_per, p.kv_heads);
    for (int h = h0; h < h1; h += R) {
        const int hh = h + sub;
        const bool live = on && hh < h1;
        const float4 z = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        const float4 kf =
            live ? load4(static_cast<const T *>(p.k) + tok * p.k_stride + (size_t)hh * p.head + 4 * l) : z;
        const float4 vf =
            live ? load4(static_cast<const T *>(p.v) + tok * p.v_stride + (size_t)hh * p.head + 4 * l) : z;
        const size_t row = ((page * p.kv_heads + min(hh, p.kv_heads - 1)) << p.bt.page_log2) + (slot & mask);
        double x[4] = {kf.x, kf.y, kf.z, kf.w};
        if (p.rope) {
            const float4 y = partners<W>(kf, l, p.rot, p.pairs);
            if (4 * l < p.rot) {
                const float yv[4] = {y.x, y.y, y.z, y.w}, c[4] = {t.c.x, t.c.y, t.c.z, t.c.w},
                            s[4] = {t.s.x, t.s.y, t.s.z, t.s.w};
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const double bs = __dmul_rn((double)yv[k], (double)s[k]);  // exact: 24 + 24 bits
                    x[k] = __fma_rn(x[k], (double)c[k], is_first(k, l, p.rot, p.pairs) ? -bs : bs);
                }
            }
        }
        quantize_store<W, BITS>(x, live, l, p.kq + row * row_bytes, p.ks + row);
        const double xv[4] = {vf.x, vf.y, vf.z, vf.w};
        quantize_store<W, BITS>(xv, live, l, p.vq + row * row_bytes, p.vs + row);
    }
}

// Eight elements of a cached row (integer * scale, rounded once to fp32, once more to a 16-bit output).
template <typename T, int BITS>
__device__ __forceinline__ void read8(const uint8_t *src, float scale, T *dst) {
    int n[8];
    if (BITS == 8) {
        const uint2 u = *reinterpret_cast<const uint2 *>(src);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            n[k] = (int8_t)(u.x >> (8 * k));
            n[4 + k] = (int8_t)(u.y >> (8 * k));
        }
    } else {
        const uint32_t u = *reinterpret_cast<const uint32_t *>(src);
#pragma unroll
        for (int k = 0; k < 8; k++) n[k] = (int)(u << (28 - 4 * k)) >> 28;
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
// lanes (eight elements a lane) copy a (token, head) row of keys and of values.
constexpr int kReadTokens = 32;  // tokens a block at most

template <typename T, int W, int BITS>
__global__ void __launch_bounds__(256) kv_read_kernel(const KvParams p) {
    __shared__ long long slots[kReadTokens];
    const int t0 = blockIdx.x * p.tokens_per_block, tid = threadIdx.x;
    const int nt = min(p.tokens_per_block, p.rows - t0);
    if (tid < nt) {
        const int tok = t0 + tid;
        long long slot = -1;
        if (tok < p.bt.cu[p.bt.batch]) {
            int lo = 0, hi = p.bt.batch;  // the first sequence that ends behind the row
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (p.bt.cu[mid + 1] <= tok) lo = mid + 1;
                else hi = mid;
            }
            if (lo < p.bt.batch) {
                const long long at = (long long)p.bt.lens[lo] + tok - p.bt.cu[lo];
                slot = at > INT_MAX ? -1 : slot_of(p.bt, lo, (int)at, &g_kv_error);
            }
        }
        slots[tid] = slot;
    }
    __syncthreads();
    const int l = tid & (W - 1), units = nt * p.kv_heads, mask = (1 << p.bt.page_log2) - 1;
    const int row_bytes = p.head * BITS / 8;
    if (8 * l >= p.head) return;
#pragma unroll 4
    for (int u = tid / W; u < units; u += 256 / W) {
        const int ti = u / p.kv_heads, h = u - ti * p.kv_heads;
        const long long slot = slots[ti];
        if (slot < 0) continue;
        const size_t row =
            (((size_t)(slot >> p.bt.page_log2) * p.kv_heads + h) << p.bt.page_log2) + (size_t)(slot & mask);
        const size_t o = (size_t)h * p.head + 8 * l;
        read8<T, BITS>(p.kq + row * row_bytes + l * BITS, p.ks[row],
                       static_cast<T *>(p.k_out) + (t0 + ti) * p.k_out_stride + o);
        read8<T, BITS>(p.vq + row * row_bytes + l * BITS, p.vs[row],
                       static_cast<T *>(p.v_out) + (t0 + ti) * p.v_out_stride + o);
    }
}

template <typename T, int BITS>
static void launch_append(const KvParams &p, unsigned grid, cudaStream_t s) {
    if (p.head <= 64) kv_append_kernel<T, 16, BITS><<<grid, 256, 0, s>>>(p);
    else kv_append_kernel<T, 32, BITS><<<grid, 256, 0, s>>>(p);
}

template <typename T, int BITS>
static void launch_read(const KvParams &p, unsigned grid, cudaStream_t s) {
    if (p.head <= 64) kv_read_kernel<T, 8, BITS><<<grid, 256, 0, s>>>(p);
    else kv_read_kernel<T, 16, BITS><<<grid, 256, 0, s>>>(p);
}

int kv_take_error(cudaStream_t s) {
    int v = 0;
    if (cudaMemcpyFromSymbolAsync(&v, g_kv_error, sizeof v, 0, cudaMemcpyDeviceToHost, s) != cudaSuccess ||
        cudaStreamSynchronize(s) != cudaSuccess)
        return -1;
    const int z = 0;
    if (v && (cudaMemcpyToSymbolAsync(g_kv_error, &z, sizeof z, 0, cudaMemcpyHostToDevice, s) != cudaSuccess ||
              cudaStreamSynchronize(s) != cudaSuccess))
        return -1;
    return v;
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
    // one pass of a warp a chunk for small calls (latency), more heads a warp where the machine is full anyway (the
    // sequence, page and table look-ups are then made once for them)
    const int r = head <= 64 ? 2 : 1;
    const bool full = (long long)rows * (kv_heads + p.heads) >= 148ll * 64 * 4 * r;
    p.kv_per = full ? 4 * r : r;
    p.q_per = full ? 8 * r : r;
    p.kv_chunks = (kv_heads + p.kv_per - 1) / p.kv_per;
    p.chunks = p.kv_chunks + (p.heads + p.q_per - 1) / p.q_per;
    const long long blocks = ((long long)rows * p.chunks + 7) / 8;
    if (blocks > INT_MAX) {
        set_error("%s: rows=%d are too many for one call", who, rows);
        return -1;
    }
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const unsigned grid = (unsigned)blocks;
    if (bits == 8) {
        if (dtype == kF32) launch_append<float, 8>(p, grid, s);
        else if (dtype == kBF16) launch_append<__nv_bfloat16, 8>(p, grid, s);
        else launch_append<__half, 8>(p, grid, s);
    } else {
        if (dtype == kF32) launch_append<float, 4>(p, grid, s);
        else if (dtype == kBF16) launch_append<__nv_bfloat16, 4>(p, grid, s);
        else launch_append<__half, 4>(p, grid, s);
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
