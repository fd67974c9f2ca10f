// What the serving operators (rope.cu, kvcache.cu, tree_attention.cu, logprobs.cu) share: element types, rows of a
// batch, pages of the quantized cache, and the error word that a kernel sets instead of touching memory that an index
// out of range names.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace mvb {
namespace rows {

// element types of the C ABI (MVB_F32, MVB_BF16, MVB_F16)
enum : int { kF32 = 0, kBF16 = 1, kF16 = 2 };

// what a kernel found in its index arrays (mvb_serve_status)
enum : int { kOk = 0, kBadPage = 1, kBadLength = 2, kBadPosition = 3, kBadToken = 4, kWaitRanOut = 5 };

template <typename T> struct Type;
template <> struct Type<float> { static constexpr int kId = kF32; };
template <> struct Type<__nv_bfloat16> { static constexpr int kId = kBF16; };
template <> struct Type<__half> { static constexpr int kId = kF16; };

inline bool known_type(int dtype) { return dtype >= kF32 && dtype <= kF16; }
inline int type_bytes(int dtype) { return dtype == kF32 ? 4 : 2; }

__device__ __forceinline__ void note(int *error, int code) { atomicCAS(error, kOk, code); }

// Four consecutive elements in fp32. The address is aligned to four elements.
__device__ __forceinline__ float4 load4(const float *p) { return *reinterpret_cast<const float4 *>(p); }
__device__ __forceinline__ float4 load4(const __nv_bfloat16 *p) {
    const uint2 u = *reinterpret_cast<const uint2 *>(p);
    return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xFFFF0000u), __uint_as_float(u.y << 16),
                       __uint_as_float(u.y & 0xFFFF0000u));
}
__device__ __forceinline__ float4 load4(const __half *p) {
    const uint2 u = *reinterpret_cast<const uint2 *>(p);
    const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&u.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&u.y));
    return make_float4(a.x, a.y, b.x, b.y);
}

// Two fp32 values rounded to a packed pair of 16-bit ones (the first in the low half).
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// Four fp32 values, each rounded once to the output's type.
__device__ __forceinline__ void store4(float *p, float4 f) { *reinterpret_cast<float4 *>(p) = f; }
template <typename T>
__device__ __forceinline__ void store4(T *p, float4 f) {
    *reinterpret_cast<uint2 *>(p) = make_uint2(pack2<T>(f.x, f.y), pack2<T>(f.z, f.w));
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }

// A batch of sequences: rows cu[b] .. cu[b + 1] - 1 belong to sequence b and stand at its positions lens[b] and on;
// position p of sequence b is slot p % page of page table[b * table_cols + p / page].
struct Batch {
    const int *cu, *lens, *table;
    int batch, table_cols, pages, page_log2;
};

// The sequence of a row: the number of sequences that end at or before it (batch for a row behind the last). A
// 32-way search by the whole warp, one load a level: one level up to 32 sequences, two up to 1,024.
__device__ __forceinline__ int sequence_of(const int *cu, int batch, int row) {
    const int lane = threadIdx.x & 31;
    int lo = 0, n = batch;
    while (n > 0) {
        const int step = (n + 31) / 32;
        const int i = lo + (lane + 1) * step;  // cu[i] <= row: sequences lo .. i - 1 end before the row
        const bool before = i <= lo + n && cu[i] <= row;
        const int k = __popc(__ballot_sync(0xffffffffu, before));
        const int left = lo + n;
        lo += k * step;
        // the steps after the k-th hold a boundary inside the next step (or the ragged end)
        n = min(step - 1, left - lo);
    }
    return lo;
}

// The slot index page * page_size + slot of position `pos` of sequence b, or -1 with the error noted.
__device__ __forceinline__ long long slot_of(const Batch &bt, int b, int pos, int *error) {
    const int col = pos >> bt.page_log2;
    if (pos < 0 || col >= bt.table_cols) {
        note(error, kBadLength);
        return -1;
    }
    const int pg = bt.table[(size_t)b * bt.table_cols + col];
    if ((unsigned)pg >= (unsigned)bt.pages) {
        note(error, kBadPage);
        return -1;
    }
    return ((long long)pg << bt.page_log2) + (pos & ((1 << bt.page_log2) - 1));
}

}  // namespace rows
}  // namespace mvb
