// The rotation of one row's elements, shared by rope.cu and by the cache append of kvcache.cu.
//
// A row of `head` elements lies over head / E lanes, E consecutive elements a lane: 16 bytes where pointers, strides and
// rot allow it (E = 4 fp32 or 8 16-bit elements), else four elements. Its first `rot` elements are turned by the angles
// of the row's position: pair i (elements i and i + rot / 2 in the half layout, 2i and 2i + 1 in the pairs layout)
// becomes (a cos - b sin, b cos + a sin). rot is a multiple of 2 E, so in the half layout both halves are whole lanes and a
// lane's partners are the elements of the lane rot / (2 E) away: one shuffle each.
#pragma once
#include "rows.cuh"

namespace mvb {
namespace rows {

// E elements of a row as fp32, as they come from memory, and back.
template <int E> struct Row { float v[E]; };

template <int E, typename T>
__device__ __forceinline__ Row<E> load_row(const T *p, bool on) {
    Row<E> r;
    if constexpr (E == 4) {
        const float4 f = on ? load4(p) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        r.v[0] = f.x; r.v[1] = f.y; r.v[2] = f.z; r.v[3] = f.w;
    } else {
        const uint4 u = on ? *reinterpret_cast<const uint4 *>(p) : make_uint4(0, 0, 0, 0);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (Type<T>::kId == kBF16) {
                r.v[2 * i] = __uint_as_float(w[i] << 16);
                r.v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
            } else {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
                r.v[2 * i] = f.x;
                r.v[2 * i + 1] = f.y;
            }
        }
    }
    return r;
}

template <int E, typename T>
__device__ __forceinline__ void store_row(T *p, const Row<E> &r) {
    if constexpr (E == 4)
        store4(p, make_float4(r.v[0], r.v[1], r.v[2], r.v[3]));
    else
        *reinterpret_cast<uint4 *>(p) = make_uint4(pack2<T>(r.v[0], r.v[1]), pack2<T>(r.v[2], r.v[3]),
                                                   pack2<T>(r.v[4], r.v[5]), pack2<T>(r.v[6], r.v[7]));
}

// A lane's cosines and sines: one an element (half layout), or one a pair, in both elements' places (pairs layout). The
// sine of a pair's first element has its sign turned, so that every element is x cos + partner sin.
template <int E> struct Turn { float c[E], s[E]; };

// l: the lane's place in its row (elements E l ..); trow: the position's table row, rot / 2 cosines then sines.
template <int E>
__device__ __forceinline__ Turn<E> load_turn(const float *trow, int l, int rot, bool pairs) {
    Turn<E> t;
#pragma unroll
    for (int k = 0; k < E; k++) t.c[k] = 1.0f, t.s[k] = 0.0f;
    if (E * l >= rot) return t;
    if (pairs) {
#pragma unroll
        for (int k = 0; k < E; k += 4) {
            const float2 c = *reinterpret_cast<const float2 *>(trow + (E * l + k) / 2);
            const float2 s = *reinterpret_cast<const float2 *>(trow + rot / 2 + (E * l + k) / 2);
            t.c[k] = t.c[k + 1] = c.x;
            t.c[k + 2] = t.c[k + 3] = c.y;
            t.s[k] = -s.x;
            t.s[k + 1] = s.x;
            t.s[k + 2] = -s.y;
            t.s[k + 3] = s.y;
        }
    } else {
        const bool first = 2 * E * l < rot;
        const int i = first ? E * l : E * l - rot / 2;
#pragma unroll
        for (int k = 0; k < E; k += 4) {
            const float4 c = *reinterpret_cast<const float4 *>(trow + i + k);
            const float4 s = *reinterpret_cast<const float4 *>(trow + rot / 2 + i + k);
            t.c[k] = c.x; t.c[k + 1] = c.y; t.c[k + 2] = c.z; t.c[k + 3] = c.w;
            t.s[k] = first ? -s.x : s.x; t.s[k + 1] = first ? -s.y : s.y;
            t.s[k + 2] = first ? -s.z : s.z; t.s[k + 3] = first ? -s.w : s.w;
        }
    }
    return t;
}

// The partner of each of a lane's elements. Every lane of the warp takes part; W lanes a row.
template <int W, int E>
__device__ __forceinline__ Row<E> partners(const Row<E> &x, int l, int rot, bool pairs) {
    Row<E> y;
    if (pairs) {
#pragma unroll
        for (int k = 0; k < E; k++) y.v[k] = x.v[k ^ 1];
    } else {
        const int half = rot / (2 * E), src = l < half ? l + half : l - half;  // outside rot the value is not used
#pragma unroll
        for (int k = 0; k < E; k++) y.v[k] = __shfl_sync(0xffffffffu, x.v[k], src, W);
    }
    return y;
}

// x turned, in fp32: one rounded product and one fused multiply-add an element.
template <int E>
__device__ __forceinline__ Row<E> turned(const Row<E> &x, const Row<E> &y, const Turn<E> &t, bool in_rot) {
    if (!in_rot) return x;
    Row<E> r;
#pragma unroll
    for (int k = 0; k < E; k++) r.v[k] = __fmaf_rn(x.v[k], t.c[k], __fmul_rn(y.v[k], t.s[k]));
    return r;
}

// Some heads (h0 .. h1 - 1) of one token's row turned from x to out (both at the token's first head, this lane's
// elements): a warp takes 32 / W heads at a time, four such steps in flight.
template <int W, int E, typename T>
__device__ __forceinline__ void turn_heads(const T *x, T *out, int h0, int h1, int head, const Turn<E> &t, int l, int sub,
                                           int rot, bool pairs) {
    constexpr int R = 32 / W, U = 4;
    const bool on = E * l < head, in_rot = E * l < rot;
    for (int h = h0; h < h1; h += U * R) {
        Row<E> v[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int hh = h + u * R + sub;
            v[u] = load_row<E>(x + (size_t)hh * head, on && hh < h1);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int hh = h + u * R + sub;
            const Row<E> y = partners<W>(v[u], l, rot, pairs);
            if (on && hh < h1) store_row(out + (size_t)hh * head, turned(v[u], y, t, in_rot));
        }
    }
}

}  // namespace rows
}  // namespace mvb
