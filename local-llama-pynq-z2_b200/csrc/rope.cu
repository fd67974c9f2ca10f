// Rotary positions: a table of cosines and sines (mvb_rope_table) and the rotation of (tokens, heads, head) rows by it
// (mvb_rope). The decode step has its rotation inside its attention kernel; this is the operator for callers that keep
// their own queries and keys.
//
// Bound: each element is read and written once; the table row of a token is read once for all its heads (8192 tokens x 40
// heads of 128, bf16, 64 turned: 5.4 TB/s).
#include <limits.h>

#include "../../include/matvec_b200.h"
#include "mvb_runtime.h"
#include "rope_rows.cuh"

namespace mvb {
namespace rows {

static __device__ int g_rope_error;

// table[p][i] = factor * cos((start + p) * freq[i]), table[p][half + i] = factor * sin(...): the angle, its cosine
// and sine in fp64 (an fp32 angle at position 100,000 is off by 0.004), rounded once.
__global__ void rope_table_kernel(const double *freq, float *table, int half, long long n, int start, double factor) {
    for (long long k = (long long)blockIdx.x * blockDim.x + threadIdx.x; k < n; k += (long long)gridDim.x * blockDim.x) {
        const long long p = k / half;
        const int i = (int)(k - p * half);
        double s, c;
        sincos(__dmul_rn((double)(start + p), freq[i]), &s, &c);
        table[p * 2 * half + i] = (float)__dmul_rn(factor, c);
        table[p * 2 * half + half + i] = (float)__dmul_rn(factor, s);
    }
}

struct RopeParams {
    const void *x;
    void *out;
    const int *pos;
    const float *table;
    long long x_stride, out_stride;  // elements from one token to the next
    int tokens, heads, head, rot, table_rows, pairs;
    int heads_per_warp, chunks;  // a warp turns heads_per_warp heads of one token; chunks = warps a token
};

// W lanes hold a row, E elements each; a warp turns heads_per_warp heads of one token.
template <typename T, int W, int E>
__global__ void __launch_bounds__(256) rope_kernel(const RopeParams p) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = lane & (W - 1), sub = lane / W;
    const long long tok = (long long)blockIdx.x * 8 + warp;
    if (tok >= p.tokens) return;
    const int h0 = blockIdx.y * p.heads_per_warp, h1 = min(h0 + p.heads_per_warp, p.heads);
    const int pos = p.pos[tok];
    if ((unsigned)pos >= (unsigned)p.table_rows) {
        if (lane == 0) note(&g_rope_error, kBadPosition);
        return;
    }
    const Turn<E> t = load_turn<E>(p.table + (size_t)pos * p.rot, l, p.rot, p.pairs);
    turn_heads<W, E>(static_cast<const T *>(p.x) + tok * p.x_stride + E * l,
                     static_cast<T *>(p.out) + tok * p.out_stride + E * l, h0, h1, p.head, t, l, sub, p.rot, p.pairs);
}

template <typename T, int E>
static void launch_lanes(const RopeParams &p, dim3 grid, cudaStream_t s) {
    // the fewest lanes that hold a row
    const int lanes = (p.head + E - 1) / E;
    if (lanes <= 8) rope_kernel<T, 8, E><<<grid, 256, 0, s>>>(p);
    else if (lanes <= 16) rope_kernel<T, 16, E><<<grid, 256, 0, s>>>(p);
    else rope_kernel<T, 32, E><<<grid, 256, 0, s>>>(p);
}

template <typename T>
static void launch_rope(const RopeParams &p, dim3 grid, bool wide, cudaStream_t s) {
    if constexpr (sizeof(T) == 2) {
        if (wide) return launch_lanes<T, 8>(p, grid, s);
    }
    launch_lanes<T, 4>(p, grid, s);
}

int *rope_error_word() {
    void *p = nullptr;
    return cudaGetSymbolAddress(&p, g_rope_error) == cudaSuccess ? static_cast<int *>(p) : nullptr;
}

}  // namespace rows
}  // namespace mvb

using namespace mvb;
using namespace mvb::rows;

extern "C" int mvb_rope_table(const double *freq, float *table, int half, int positions, int start, double factor,
                              void *stream) {
    if (!freq || !table || ((uintptr_t)freq & 7) || ((uintptr_t)table & 3)) {
        set_error("mvb_rope_table: null or misaligned pointer");
        return -1;
    }
    if (half <= 0 || positions < 0 || start < 0 || start > INT_MAX - positions) {
        set_error("mvb_rope_table: unsupported half=%d positions=%d start=%d", half, positions, start);
        return -1;
    }
    if (!positions) return 0;
    const long long n = (long long)positions * half;
    const unsigned grid = (unsigned)(n + 255 < 256ll * 148 * 8 ? (n + 255) / 256 : 148 * 8);
    rope_table_kernel<<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(freq, table, half, n, start, factor);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) {
        set_error("mvb_rope_table: launch failed: %s", cudaGetErrorString(e));
        return -1;
    }
    return 0;
}

extern "C" int mvb_rope(const void *x, const int *pos, const float *table, void *out, int dtype, int tokens, int heads,
                        int head, int rot, int table_rows, int layout, long long x_stride, long long out_stride,
                        void *stream) {
    if (!known_type(dtype) || (layout != 0 && layout != 1)) {
        set_error("mvb_rope: unknown type %d or layout %d", dtype, layout);
        return -1;
    }
    if (tokens < 0 || heads <= 0 || head <= 0 || head % 8 || head > 128 || rot <= 0 || rot % 8 || rot > head ||
        table_rows < 0 || x_stride % 4 || out_stride % 4) {
        set_error("mvb_rope: unsupported tokens=%d heads=%d head=%d rot=%d (need head and rot multiples of 8, rot <= "
                  "head <= 128, strides multiples of 4)", tokens, heads, head, rot);
        return -1;
    }
    if (!tokens) return 0;
    const uintptr_t need = 4 * type_bytes(dtype) - 1;
    if (!x || !out || !pos || !table || ((uintptr_t)x & need) || ((uintptr_t)out & need) || ((uintptr_t)pos & 3) ||
        ((uintptr_t)table & 15)) {
        set_error("mvb_rope: null or misaligned pointer (x and out four elements, table 16 bytes)");
        return -1;
    }
    RopeParams p;
    p.x = x;
    p.out = out;
    p.pos = pos;
    p.table = table;
    p.x_stride = x_stride;
    p.out_stride = out_stride;
    p.tokens = tokens;
    p.heads = heads;
    p.head = head;
    p.rot = rot;
    p.table_rows = table_rows;
    p.pairs = layout;
    // 16 bytes a lane where everything is a multiple of that (8192 tokens x 40 heads of 128, bf16: 43 us with 8 bytes a
    // lane and 4 heads a warp, 32 us so)
    const bool wide = dtype != kF32 && rot % 16 == 0 && x_stride % 8 == 0 && out_stride % 8 == 0 &&
                      !(((uintptr_t)x | (uintptr_t)out) & 15);
    const int lane_elems = wide ? 8 : 4, r = 32 / (head <= 8 * lane_elems ? 8 : head <= 16 * lane_elems ? 16 : 32);
    // a whole token a warp when there are tokens enough to fill the machine, else fewer heads a warp (latency)
    p.heads_per_warp = tokens >= 148 * 24 ? heads : (long long)tokens * heads >= 148ll * 64 * 4 * r ? 4 * r : r;
    p.chunks = (heads + p.heads_per_warp - 1) / p.heads_per_warp;
    if (p.chunks > 65535) {
        set_error("mvb_rope: heads=%d are too many for one call", heads);
        return -1;
    }
    const dim3 grid((unsigned)(((long long)tokens + 7) / 8), p.chunks);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == kF32) launch_rope<float>(p, grid, wide, s);
    else if (dtype == kBF16) launch_rope<__nv_bfloat16>(p, grid, wide, s);
    else launch_rope<__half>(p, grid, wide, s);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) {
        set_error("mvb_rope: launch failed: %s", cudaGetErrorString(e));
        return -1;
    }
    return 0;
}
