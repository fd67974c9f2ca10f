// The rotation of one row's elements, shared by rope.cu and by the cache append of kvcache.cu.
//
// A row of `head` elements lies over head / 4 lanes, four consecutive elements a lane. Its first `rot` elements are
// turned by the angles of the row's position: pair i (elements i and i + rot / 2 in the half layout, 2i and 2i + 1
// in the pairs layout) becomes (a cos - b sin, b cos + a sin). rot is a multiple of 8, so in the half layout both
// halves are whole lanes and a lane's partners are the four elements of the lane rot / 8 away: one shuffle each.
#pragma once
#include "rows.cuh"

namespace mvb {
namespace rows {

// A lane's cosines and sines: of its four elements (half layout), or of its two pairs (x, y) (pairs layout).
struct Turn {
    float4 c, s;
};

// l: the lane's place in its row (elements 4l .. 4l + 3); trow: the position's table row, rot / 2 cosines then sines.
__device__ __forceinline__ Turn load_turn(const float *trow, int l, int rot, bool pairs) {
    Turn t;
    t.c = make_float4(1.0f, 1.0f, 1.0f, 1.0f);
    t.s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (4 * l >= rot) return t;
    if (pairs) {
        const float2 c = *reinterpret_cast<const float2 *>(trow + 2 * l);
        const float2 s = *reinterpret_cast<const float2 *>(trow + rot / 2 + 2 * l);
        t.c = make_float4(c.x, c.x, c.y, c.y);
        t.s = make_float4(s.x, s.x, s.y, s.y);
    } else {
        const int i = 4 * l < rot / 2 ? 4 * l : 4 * l - rot / 2;
        t.c = *reinterpret_cast<const float4 *>(trow + i);
        t.s = *reinterpret_cast<const float4 *>(trow + rot / 2 + i);
    }
    return t;
}

// The partner of each of a lane's elements (b for a, a for b). Every lane of the warp takes part; W lanes a row.
template <int W>
__device__ __forceinline__ float4 partners(float4 x, int l, int rot, bool pairs) {
    if (pairs) return make_float4(x.y, x.x, x.w, x.z);
    const int src = 8 * l < rot ? l + rot / 8 : l - rot / 8;  // outside the rotated lanes the value is not used
    return make_float4(__shfl_sync(0xffffffffu, x.x, src, W), __shfl_sync(0xffffffffu, x.y, src, W),
                       __shfl_sync(0xffffffffu, x.z, src, W), __shfl_sync(0xffffffffu, x.w, src, W));
}

// Whether element k (0 .. 3) of lane l is the first of its pair.
__device__ __forceinline__ bool is_first(int k, int l, int rot, bool pairs) { return pairs ? !(k & 1) : 8 * l < rot; }

// x turned, in fp32: x cos -+ partner sin, the second product inside the fused multiply-add (one rounding each).
__device__ __forceinline__ float4 turned(float4 x, float4 y, const Turn &t, int l, int rot, bool pairs) {
    if (4 * l >= rot) return x;
    auto one = [&](float a, float b, float c, float s, int k) {
        const float bs = __fmul_rn(b, s);
        return __fmaf_rn(a, c, is_first(k, l, rot, pairs) ? -bs : bs);
    };
    return make_float4(one(x.x, y.x, t.c.x, t.s.x, 0), one(x.y, y.y, t.c.y, t.s.y, 1), one(x.z, y.z, t.c.z, t.s.z, 2),
                       one(x.w, y.w, t.c.w, t.s.w, 3));
}

}  // namespace rows
}  // namespace mvb
