// Attention of a batch's new tokens (one, a chain, or a tree of drafted ones) over the paged 8- or 4-bit cache
// (mvb_tree_attention). The new tokens' keys and values are in the cache already (mvb_kv_append): token i of sequence b
// stands at position ctx + i and sees positions below ctx, and of the new ones those its mask bits allow.
//
//     S = scale * ks[t] * (q . k[t]),  P = exp(S - max),  O = sum_t P[t] vs[t] v[t] / sum_t P[t]
//
// with k and v the cached integers, which fp16 holds exactly: the products take them as they are, the keys' scales
// multiply S and the values' scales multiply P. q is put in fp16 after a power of two of its row's largest element was
// taken out (2 ^ e; a bf16 or fp16 q keeps every bit that is above 2^-33 of the row's largest); an fp32 q goes in two
// parts, high and low (22 bits). P vs goes to fp16 in a unit of its row's own (`moved`), rounded once for bf16 callers (2^-11, an
// eighth of the output's own half step); for fp16 and fp32 callers in two parts (22 bits), since one rounding would be as
// large as an fp16 output's own. What is far below the row's largest is held to a fixed step: 2^-27 of that at most.
// max, sum and O are fp32.
//
// This kernel: 8 * NT query rows (new tokens x the query heads of one kv head) at a time; a handful of rows does little
// arithmetic per cached byte, so the work is to stream the cache with few instructions a byte. One warp owns slices of 16
// keys (HDP = 128) or 32 (HDP = 64): cp.async into its own ring of three stages, no barrier with the other warps. The
// products are mma.m16n8k16 with the cache as the 16-row operand (S^T = K Q^T, O^T = V^T P^T): eight query rows cost
// eight columns, and a slice's fragments, converted from bytes in registers, serve all NT column tiles. S^T leaves a lane
// with (key, two rows); movmatrix turns that into the operand of the second product. The order of the head's elements
// inside a product is free as long as q and k agree, and so is the order of the keys in P v: both are chosen so that a
// lane reads whole 4- to 16-byte pieces. Keys of a sequence are split over the warps of a CTA and over the CTAs of a
// cluster (up to 16), whose partial (max, sum, O) are joined in distributed shared memory in a fixed order: one launch, no
// workspace, the same bits on every run. Few long sequences: over several clusters each, so that every SM has a part; the
// clusters' results go to the caller's workspace and join_kernel adds them.
// Measured (32 heads of 128 over 8 kv heads, int8, bf16): 64 sequences of 8,000 keys, one token each: 114 us in a burst
// (5.3 TB/s), 126 for a second on end, where the power limit takes a tenth of the clock. One of 131,001 keys: 62, 77, 95 us for 4, 16, 24 rows; there a warp's chain over
// a slice (1.6 us, int4 alike) is the bound.
#include <cooperative_groups.h>
#include <limits.h>
#include <math.h>

#include <mutex>

#include "../../include/matvec_b200.h"
#include "mvb_runtime.h"
#include "tree_attention.cuh"

namespace mvb {
namespace attn {

using namespace rows;
namespace cg = cooperative_groups;

static __device__ int g_attn_error;

constexpr int kStages = 3;

template <int HDP, int BITS>
struct Slice {
    static constexpr int kKeys = HDP == 128 ? 16 : 32;
    static constexpr int kSub = kKeys / 16;            // 16-key pieces, each inside one page
    static constexpr int kRow = HDP * BITS / 8;        // bytes of a row in shared memory
    static constexpr int kScales = 2 * kKeys * kRow;   // offset of the scales in a stage
    static constexpr int kStage = 2 * kKeys * kRow + 2 * kKeys * 4;
    static constexpr int kWarp = kStages * kStage;  // a warp's ring
    static constexpr int kPieces = BITS == 8 ? kRow / 32 : kRow / 16;  // cp.async a lane and 16-key piece, at most
};

// Where byte `off` of row `row` lies: 16-byte chunks of each 128-byte line permuted so that the lanes of a fragment load
// (rows r with four neighbouring chunks for the keys, rows 2c with all chunks for the values) fall on different banks.
template <int RS>
__device__ __forceinline__ int place(int row, int off) {
    if (RS == 128) return row * 128 + (((off >> 4) ^ ((((row >> 1) & 3) << 1) ^ ((row & 1) << 2))) << 4) + (off & 15);
    if (RS == 64) return (row >> 1) * 128 + (((((row & 1) << 2) | (off >> 4)) ^ (((row >> 1) & 3) << 1)) << 4) + (off & 15);
    return (row >> 2) * 128 + (((((row & 3) << 1) | (off >> 4)) ^ (((row >> 2) & 1) << 1)) << 4) + (off & 15);
}

__device__ __forceinline__ void mma16816(float (&d)[4], const uint4 &a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

template <int BYTES>
__device__ __forceinline__ void cp_async(uint32_t dst, const void *src) {
    if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}

__device__ __forceinline__ uint32_t transposed(uint32_t x) {  // of an 8 x 8 tile of 16-bit elements
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// The head element that element e (0 .. 3: k = 2c, 2c + 1, 2c + 8, 2c + 9) of lane column c holds in k-step ks: a lane
// reads 16 elements (64 * (ks / 4) + 16 c ..) at once and spreads them over four k-steps as the conversions leave them:
// bytes (0, 2) and (1, 3) of a word, nibbles (o, o + 4) and (o + 1, o + 5).
template <int BITS>
__device__ __forceinline__ int element_of(int ks, int c, int e) {
    const int base = 64 * (ks >> 2) + 16 * c, w = ks & 3;
    if (BITS == 8) return base + 4 * w + (e >> 1) + 2 * (e & 1);
    return base + 8 * (w >> 1) + 2 * (w & 1) + (e >> 1) + 4 * (e & 1);
}

// Parts of q and of P for each caller's type.
template <typename T> struct Parts { static constexpr int kQ = 1, kP = 1; };
template <> struct Parts<__half> { static constexpr int kQ = 1, kP = 2; };
template <> struct Parts<float> { static constexpr int kQ = 2, kP = 2; };

template <typename T, int BITS, int HDP, int NT, int kWarps>
__global__ void __launch_bounds__(kWarps * 32, kWarps == 8 && NT <= 2 ? 2 : 1) tree_attention_kernel(const AttnParams p) {
    using S = Slice<HDP, BITS>;
    constexpr int KS = HDP / 16;                 // k-steps of q.k, and 16-element tiles of O
    constexpr int RUN = HDP / 8;                 // a lane's elements of a value row: RUN * r ..
    constexpr int QP = Parts<T>::kQ, PP = Parts<T>::kP;
    constexpr int ROWS = 8 * NT;
    constexpr bool QREG = NT * QP * KS <= (NT == 1 && !(QP == 2 && kWarps == 16) ? 16 : 8);  // q's fragments in registers, else
    // read again for every slice (16 warps, fp32: 32 registers of them spill others; one sequence of 131,001 keys, 4 rows,
    // 82 us so, 73 with q read again)
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float row_factor[ROWS], warp_m[kWarps][ROWS], warp_l[kWarps][ROWS], cta_m[ROWS], cta_l[ROWS];
    __shared__ float all_m[16][ROWS], all_l[16][ROWS];
    uint2 *qfrag = reinterpret_cast<uint2 *>(smem);  // [QP][NT][KS][32 lanes]
    uint8_t *pipe = smem + QP * NT * KS * 256;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    const int b = blockIdx.z, kvh = blockIdx.y / p.qtiles, qt = blockIdx.y - kvh * p.qtiles;
    const int split = blockIdx.x % p.splits, super = blockIdx.x / p.splits;
    const Sequence s = sequence_at(p, b, &g_attn_error);
    const int nrows = s.n * p.group, R0 = qt * ROWS;
    if (R0 >= nrows) return;  // the whole cluster returns together

    // this warp's slices
    const int ns = (s.len + S::kKeys - 1) / S::kKeys;
    const int s0 = (int)((long long)ns * blockIdx.x / gridDim.x), s1 = (int)((long long)ns * (blockIdx.x + 1) / gridDim.x);
    const int row_bytes = p.head * BITS / 8, piece = row_bytes % 16 ? 8 : 16;
    uint8_t *mine = pipe + warp * S::kWarp;
    const uint32_t mine_u = (uint32_t)__cvta_generic_to_shared(mine);
    int doff[S::kPieces];  // shared-memory place of this lane's i-th piece of a 16-key run, or -1
#pragma unroll
    for (int i = 0; i < S::kPieces; i++) {
        const int o = (lane + 32 * i) * piece;
        doff[i] = o < 16 * row_bytes ? place<S::kRow>(o / row_bytes, o % row_bytes) : -1;
    }
    auto issue = [&](int sl, int stage) {
#pragma unroll
        for (int sub = 0; sub < S::kSub; sub++) {
            const int key = sl * S::kKeys + 16 * sub;
            if (key >= s.len) break;
            const int pg = page_of(p, b, key, &g_attn_error);
            const size_t row = (((size_t)pg * p.kv_heads + kvh) << p.bt.page_log2) + (key & ((1 << p.bt.page_log2) - 1));
            const uint8_t *kp = p.kq + row * row_bytes + lane * piece, *vp = p.vq + row * row_bytes + lane * piece;
            const uint32_t d = mine_u + stage * S::kStage + sub * 16 * S::kRow;
            if (piece == 16) {
#pragma unroll
                for (int i = 0; i < S::kPieces; i++)
                    if (doff[i] >= 0) {
                        cp_async<16>(d + doff[i], kp + 512 * i);
                        cp_async<16>(d + S::kKeys * S::kRow + doff[i], vp + 512 * i);
                    }
            } else {
#pragma unroll
                for (int i = 0; i < S::kPieces; i++)
                    if (doff[i] >= 0) {
                        cp_async<8>(d + doff[i], kp + 256 * i);
                        cp_async<8>(d + S::kKeys * S::kRow + doff[i], vp + 256 * i);
                    }
            }
            // the scales: lanes 0 .. 3 the keys', 4 .. 7 the values'
            if (lane < 8)
                cp_async<16>(mine_u + stage * S::kStage + S::kScales + sub * 64 + (lane >> 2) * S::kKeys * 4 + 16 * c,
                             (lane < 4 ? p.ks : p.vs) + row + 4 * c);
        }
    };
    int sl_next = s0 + warp;
    for (int st = 0; st < kStages - 1; st++) {
        if (sl_next < s1) issue(sl_next, st);
        sl_next += kWarps;
        asm volatile("cp.async.commit_group;" ::: "memory");
    }

    // q: a warp scales its rows by powers of two into fp32, then every warp builds fragments. The rows are staged in the
    // rings' last stages, which the first slices above leave free: with room of their own (8 KB) two CTAs of 16 rows a kv
    // head of 128 in 8 bits miss an SM's shared memory by 1.3 KB each.
    static_assert((kStages - 1) * S::kStage + ((ROWS - 1) / kWarps + 1) * HDP * 4 <= S::kWarp, "q rows in the last stage");
    auto qrow = [&](int i) {
        return reinterpret_cast<float *>(pipe + i % kWarps * S::kWarp + (kStages - 1) * S::kStage) + i / kWarps * HDP;
    };
    for (int i = warp; i < ROWS; i += kWarps) {
        const int R = R0 + i;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (R < nrows && 4 * lane < p.head)
            v = load4(static_cast<const T *>(p.q) + (size_t)(s.row0 + R / p.group) * p.q_stride +
                      (size_t)(kvh * p.group + R % p.group) * p.head + 4 * lane);
        int e = max(max(exponent_of(v.x), exponent_of(v.y)), max(exponent_of(v.z), exponent_of(v.w)));
#pragma unroll
        for (int o = 16; o; o >>= 1) e = max(e, __shfl_xor_sync(0xffffffffu, e, o));
        // largest element in [2^8, 2^9); a row of zeros or subnormals keeps the factor of the smallest exponent
        const int k = max(-100, min(e - 127 - 8, 119));
        if (4 * lane < HDP) {
            const float f = pow2(-k);
            reinterpret_cast<float4 *>(qrow(i))[lane] = make_float4(v.x * f, v.y * f, v.z * f, v.w * f);
        }
        if (lane == 0) row_factor[i] = pow2(k);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < NT * KS * 32; i += kWarps * 32) {
        const int ln = i & 31, ks = (i >> 5) % KS, nt = (i >> 5) / KS;
        const float *a = qrow(nt * 8 + (ln >> 2));
        float f[4];
#pragma unroll
        for (int e = 0; e < 4; e++) f[e] = a[element_of<BITS>(ks, ln & 3, e)];
        qfrag[i] = make_uint2(pack2<__half>(f[0], f[1]), pack2<__half>(f[2], f[3]));
        if (QP == 2) {
#pragma unroll
            for (int e = 0; e < 4; e++) f[e] = f[e] - __half2float(__float2half_rn(f[e]));
            qfrag[NT * KS * 32 + i] = make_uint2(pack2<__half>(f[0], f[1]), pack2<__half>(f[2], f[3]));
        }
    }
    __syncthreads();
    uint2 qreg[QREG ? QP * NT * KS : 1];
    if (QREG) {
#pragma unroll
        for (int i = 0; i < QP * NT * KS; i++) qreg[i] = qfrag[i * 32 + lane];
    }

    // this lane's rows of column tile nt: 8 nt + 2c, + 1
    float O[NT][KS][4], unit[NT][2], l[NT][2], rf[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
        for (int j = 0; j < KS; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) O[nt][j][e] = 0.0f;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            unit[nt][h] = INFINITY;
            l[nt][h] = 0.0f;
            rf[nt][h] = row_factor[nt * 8 + 2 * c + h];
        }
    }

    // where this lane's fragments lie in a stage (+ 16 * kRow * sub; the rows 8 further lie 8 * kRow further)
    const int k_at = place<S::kRow>(r, BITS == 8 ? 16 * c : 8 * c);
    const int k_at1 = HDP == 128 ? place<S::kRow>(r, BITS == 8 ? 64 + 16 * c : 32 + 8 * c) : 0;
    constexpr int WORDS = RUN * BITS / 32;  // 32-bit words of a key's elements: 4, 2 (8 bits), 2, 1 (4 bits)
    const int v_at = S::kKeys * S::kRow + place<S::kRow>(2 * c, r * WORDS * 4);
    const int v_at1 = S::kKeys * S::kRow + place<S::kRow>(2 * c + 1, r * WORDS * 4);

    int stage = 0;
    for (int sl = s0 + warp; sl < s1; sl += kWarps) {
        {
            const int st = stage >= 1 ? stage - 1 : kStages - 1;  // the stage read last time round
            if (sl_next < s1) issue(sl_next, st);
            sl_next += kWarps;
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
        __syncwarp();
        const uint8_t *kt = mine + stage * S::kStage;
        const float *ksc = reinterpret_cast<const float *>(kt + S::kScales), *vsc = ksc + S::kKeys;
        const int key0 = sl * S::kKeys;

        float sc[NT][S::kSub][4];  // (key r, row 2c), (key r, row 2c + 1), (key r + 8, ..), ..
#pragma unroll
        for (int sub = 0; sub < S::kSub; sub++) {
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int e = 0; e < 4; e++) sc[nt][sub][e] = 0.0f;
#pragma unroll
            for (int ch = 0; ch < HDP / 64; ch++) {
                uint32_t kb[2][4][2];  // [key r, r + 8][k-step of this chunk][low, high k]
#pragma unroll
                for (int n = 0; n < 2; n++) {
                    const uint8_t *src = kt + (ch ? k_at1 : k_at) + (sub * 16 + n * 8) * S::kRow;
                    if (BITS == 8) {
                        const uint4 u = *reinterpret_cast<const uint4 *>(src);
                        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            kb[n][k][0] = bytes_to_half2(w[k]);
                            kb[n][k][1] = bytes_to_half2(w[k] >> 8);
                        }
                    } else {
                        const uint2 u = *reinterpret_cast<const uint2 *>(src);
                        const uint32_t w[2] = {u.x, u.y};
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            kb[n][k][0] = nibbles_to_half2(w[k >> 1], 2 * (k & 1));
                            kb[n][k][1] = nibbles_to_half2(w[k >> 1], 2 * (k & 1) + 1);
                        }
                    }
                }
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const uint4 a = make_uint4(kb[0][k][0], kb[1][k][0], kb[0][k][1], kb[1][k][1]);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int part = 0; part < QP; part++) {
                            const int i = (part * NT + nt) * KS + 4 * ch + k;
                            const uint2 q = QREG ? qreg[QREG ? i : 0] : qfrag[i * 32 + lane];
                            mma16816(sc[nt][sub], a, q.x, q.y);
                        }
                }
            }
        }
        // the scales of this lane's keys; S in units of the row's factor; the mask where some key is new or none
        float vv[S::kSub][2];
        const bool tail = key0 + S::kKeys > s.ctx;
        uint32_t move = 0;  // one bit for each of this lane's rows
#pragma unroll
        for (int sub = 0; sub < S::kSub; sub++)
#pragma unroll
            for (int n = 0; n < 2; n++) {
                const float kk = ksc[sub * 16 + n * 8 + r] * p.scale_log2;
                vv[sub][n] = vsc[sub * 16 + n * 8 + r];
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    sc[nt][sub][2 * n] *= kk;
                    sc[nt][sub][2 * n + 1] *= kk;
                }
            }
        if (tail) {
#pragma unroll
            for (int sub = 0; sub < S::kSub; sub++)
#pragma unroll
                for (int n = 0; n < 2; n++) {
                    const int key = key0 + sub * 16 + n * 8 + r;
                    if (key >= s.len) vv[sub][n] = 0.0f;
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int h = 0; h < 2; h++)
                            if (!allowed(p, s, (R0 + nt * 8 + 2 * c + h) / p.group, key)) sc[nt][sub][2 * n + h] = -INFINITY;
                }
        }
        // The rows' units move only when a row needs it: every lane looks at its own scores and scales, one vote a slice; the
        // maxima are exchanged only then.
        float mx[NT][2], mv = 0.0f;
#pragma unroll
        for (int sub = 0; sub < S::kSub; sub++)
#pragma unroll
            for (int n = 0; n < 2; n++)  // (an infinite scale makes the rows that see it infinite, and no unit)
                if (fabsf(vv[sub][n]) < INFINITY) mv = fmaxf(mv, fabsf(vv[sub][n]));
        const float limit = unit_limit(mv);
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                float x = fmaxf(sc[nt][0][h], sc[nt][0][2 + h]);
#pragma unroll
                for (int sub = 1; sub < S::kSub; sub++) x = fmaxf(x, fmaxf(sc[nt][sub][h], sc[nt][sub][2 + h]));
                mx[nt][h] = x * rf[nt][h];
                move |= (uint32_t)(mx[nt][h] + unit[nt][h] > limit) << (2 * nt + h);
            }
        if (__any_sync(0xffffffffu, move)) {
            move = __reduce_or_sync(0xffffffffu, move);
            float lv[S::kSub][2];
#pragma unroll
            for (int sub = 0; sub < S::kSub; sub++)
#pragma unroll
                for (int n = 0; n < 2; n++) lv[sub][n] = log_scale(vv[sub][n]);
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    if (!((move >> (2 * nt + h)) & 1)) continue;
                    float t = mx[nt][h], top = -INFINITY;
#pragma unroll
                    for (int sub = 0; sub < S::kSub; sub++)
#pragma unroll
                        for (int n = 0; n < 2; n++)
                            top = fmaxf(top, __fmaf_rn(sc[nt][sub][2 * n + h], rf[nt][h], lv[sub][n]));
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) {
                        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, o));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                    }
                    // only the rows that are behind move, so that a row's result does not depend on its neighbours
                    const float to = moved<PP>(unit[nt][h], t, top), f = unit_factor(unit[nt][h], to);
                    unit[nt][h] = to;
                    l[nt][h] *= f;
#pragma unroll
                    for (int j = 0; j < KS; j++) {
                        O[nt][j][h] *= f;
                        O[nt][j][2 + h] *= f;
                    }
                }
        }
#pragma unroll
        for (int sub = 0; sub < S::kSub; sub++) {
            uint32_t P[PP][NT][2];  // [part][column tile][keys 0 .. 7, 8 .. 15]: the operand of the second product
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                float pv[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float x = exp2_fast(__fmaf_rn(sc[nt][sub][e], rf[nt][e & 1], or_zero(unit[nt][e & 1])));
                    l[nt][e & 1] += x;
                    pv[e] = x * vv[sub][e >> 1];
                }
                if (tail) {  // a masked key's value scale may be anything: its weight is zero, not zero times that
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (sc[nt][sub][e] == -INFINITY) pv[e] = 0.0f;
                }
                P[0][nt][0] = transposed(pack2<__half>(pv[0], pv[1]));
                P[0][nt][1] = transposed(pack2<__half>(pv[2], pv[3]));
                if (PP == 2) {
#pragma unroll
                    for (int e = 0; e < 4; e++) pv[e] -= __half2float(__float2half_rn(pv[e]));
                    P[PP - 1][nt][0] = transposed(pack2<__half>(pv[0], pv[1]));
                    P[PP - 1][nt][1] = transposed(pack2<__half>(pv[2], pv[3]));
                }
            }
            // values: lane (r, c) takes elements RUN * r .. of keys 2c, 2c + 1, 2c + 8, 2c + 9 of this piece
            uint32_t w[4][WORDS];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const uint8_t *src = kt + (k & 1 ? v_at1 : v_at) + (sub * 16 + 8 * (k >> 1)) * S::kRow;
                if constexpr (WORDS == 4) {
                    const uint4 u = *reinterpret_cast<const uint4 *>(src);
                    w[k][0] = u.x; w[k][1] = u.y; w[k][2] = u.z; w[k][3] = u.w;
                } else if constexpr (WORDS == 2) {
                    const uint2 u = *reinterpret_cast<const uint2 *>(src);
                    w[k][0] = u.x; w[k][1] = u.y;
                } else {
                    w[k][0] = *reinterpret_cast<const uint32_t *>(src);
                }
            }
#pragma unroll
            for (int i = 0; i < WORDS; i++) {
                constexpr int PER = 32 / BITS;  // elements a word
                uint32_t vb[PER][2];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const uint32_t lo = __byte_perm(w[2 * h][i], w[2 * h + 1][i], 0x5410);
                    const uint32_t hi = __byte_perm(w[2 * h][i], w[2 * h + 1][i], 0x7632);
                    if (BITS == 8) {
                        vb[0][h] = bytes_to_half2(lo);
                        vb[1][h] = bytes_to_half2(lo >> 8);
                        vb[2][h] = bytes_to_half2(hi);
                        vb[3][h] = bytes_to_half2(hi >> 8);
                    } else {
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            vb[k][h] = nibbles_to_half2(lo, k);
                            vb[(4 + k) % PER][h] = nibbles_to_half2(hi, k);
                        }
                    }
                }
#pragma unroll
                for (int k = 0; k < PER; k += 2) {  // element tile j: elements RUN * r + 2j (rows r), + 2j + 1 (rows r + 8)
                    const uint4 a = make_uint4(vb[k][0], vb[k + 1][0], vb[k][1], vb[k + 1][1]);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        // The products' own sums are cut towards zero, at 2^-23 for every 16 keys and part: some 1e-4 over 16,000 keys
                        // of a warp whose values have one sign, a quarter of an fp16 output's half step. An fp32 caller's
                        // slices are therefore added here, rounded to nearest (an fp16 caller's so: 4 to 10 % longer).
                        constexpr bool APART = sizeof(T) == 4;
                        float (&o)[4] = O[nt][(PER * i + k) / 2];
                        float t[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int part = 0; part < PP; part++) mma16816(APART ? t : o, a, P[part][nt][0], P[part][nt][1]);
                        if (APART) {
#pragma unroll
                            for (int e = 0; e < 4; e++) o[e] += t[e];
                        }
                    }
                }
            }
        }
        __syncwarp();  // every lane has read the stage before the next turn refills it
        stage = stage + 1 == kStages ? 0 : stage + 1;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();

    // join the warps: O in the unit of the sums to shared memory, then (max, sum) of each row
    float *po = reinterpret_cast<float *>(pipe);  // [kWarps][ROWS][HDP]
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            float sum = l[nt][h];
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            const int row = nt * 8 + 2 * c + h;
            const float2 ml = normal_sum(unit[nt][h], sum);
            const float back = sum == 0.0f ? 0.0f : pow2_of((float)(127 - exponent_of(sum)));
            if (r == 0) {
                warp_m[warp][row] = ml.x;
                warp_l[warp][row] = ml.y;
            }
            float *d = po + ((size_t)warp * ROWS + row) * HDP + RUN * r;
#pragma unroll
            for (int j = 0; j < KS; j += 2)
                *reinterpret_cast<float4 *>(d + 2 * j) = make_float4(O[nt][j][h] * back, O[nt][j][2 + h] * back,
                                                                     O[nt][j + 1][h] * back, O[nt][j + 1][2 + h] * back);
        }
    __syncthreads();
    const int rows_here = min(ROWS, nrows - R0);
    auto finish = [&](int row, int d4, float4 o, float sum, float mm) {
        const int R = R0 + row, tok = s.row0 + R / p.group, head = kvh * p.group + R % p.group;
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;  // no key: o is zero too
        if (p.supers > 1) {
            const size_t at = ((size_t)super * p.rows + tok) * p.heads + head;
            if (4 * d4 < p.head)
                *reinterpret_cast<float4 *>(p.work + at * p.head + 4 * d4) =
                    make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
            if (d4 == 0) work_ml(p)[at] = make_float2(mm, sum);
            return;
        }
        if (4 * d4 < p.head)
            store4(static_cast<T *>(p.out) + (size_t)tok * p.out_stride + (size_t)head * p.head + 4 * d4,
                   make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
        if (d4 == 0 && p.lse)
            p.lse[(size_t)tok * p.heads + head] =
                sum == 0.0f ? -INFINITY : (mm + log2f(sum)) * 0.693147180559945309f;
    };
    for (int i = threadIdx.x; i < rows_here * (HDP / 4); i += kWarps * 32) {
        const int row = i / (HDP / 4), d4 = i % (HDP / 4);
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; w++) mm = fmaxf(mm, warp_m[w][row]);
        float sum = 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < kWarps; w++) {
            const float4 x = *reinterpret_cast<const float4 *>(po + ((size_t)w * ROWS + row) * HDP + 4 * d4);
            if (warp_l[w][row] != 0.0f) {  // this warp saw a key (a NaN sum among them)
                const float f = exp2_fast(warp_m[w][row] - mm);
                sum += f * warp_l[w][row];
                o.x += f * x.x;
                o.y += f * x.y;
                o.z += f * x.z;
                o.w += f * x.w;
            }
        }
        if (p.splits == 1) {
            finish(row, d4, o, sum, mm);
        } else {
            *reinterpret_cast<float4 *>(po + (size_t)row * HDP + 4 * d4) = o;  // this thread's own place of warp 0
            if (d4 == 0) {
                cta_m[row] = mm;
                cta_l[row] = sum;
            }
        }
    }
    if (p.splits == 1) return;
    // join the cluster: CTA `split` takes every splits-th piece, reading its sisters' shared memory in rank order
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    for (int i = threadIdx.x; i < p.splits * rows_here; i += kWarps * 32) {
        const int w = i / rows_here, row = i - w * rows_here;
        all_m[w][row] = *cluster.map_shared_rank(&cta_m[row], w);
        all_l[w][row] = *cluster.map_shared_rank(&cta_l[row], w);
    }
    __syncthreads();
    for (int i = threadIdx.x * p.splits + split; i < rows_here * (HDP / 4); i += kWarps * 32 * p.splits) {
        const int row = i / (HDP / 4), d4 = i % (HDP / 4);
        float mm = -INFINITY;
        for (int w = 0; w < p.splits; w++) mm = fmaxf(mm, all_m[w][row]);
        float sum = 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
        for (int w = 0; w < p.splits; w++) {
            const float4 x = *reinterpret_cast<const float4 *>(cluster.map_shared_rank(po + (size_t)row * HDP + 4 * d4, w));
            const float lw = all_l[w][row];
            if (lw == 0.0f) continue;
            const float f = exp2_fast(all_m[w][row] - mm);
            sum += f * lw;
            o.x += f * x.x;
            o.y += f * x.y;
            o.z += f * x.z;
            o.w += f * x.w;
        }
        finish(row, d4, o, sum, mm);
    }
    cluster.sync();  // no CTA leaves while a sister reads its shared memory
}

// How many clusters a sequence may be split over: as many as the caller's workspace holds parts of.
int most_supers(const AttnParams &p) {
    const size_t one = work_need(p, 1);
    const size_t n = p.work && one ? p.work_bytes / one : 1;
    return n < 2 ? 1 : n > kMaxSupers ? kMaxSupers : (int)n;
}

template <typename T, int BITS, int HDP, int NT, int kWarps>
static cudaError_t launch_warps(AttnParams p, int max_len, cudaStream_t stream) {
    using S = Slice<HDP, BITS>;
    constexpr int ROWS = 8 * NT;
    constexpr size_t frag = (size_t)Parts<T>::kQ * NT * (HDP / 16) * 256;
    constexpr size_t ring = (size_t)kWarps * S::kWarp, join = (size_t)kWarps * ROWS * HDP * 4;
    constexpr size_t smem = frag + (ring > join ? ring : join);
    static_assert(smem <= 227 * 1024 - 8192, "shared memory of a CTA");
    auto kernel = tree_attention_kernel<T, BITS, HDP, NT, kWarps>;
    if (!tiles_fit(p, ROWS)) return kTooManyRows;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    // a unit: one slice a warp, 0.7 us (2 where two CTAs of an SM stream); a CTA starts and joins in about 6 us, a second
    // kernel in 2; a cluster's join grows with its CTAs (one sequence of 2,000 keys, 8 kv heads, int8, 4 | 16 rows: clusters
    // of 4, 8, 16 take 11.6, 9.7, 10.0 | 15.4, 13.7, 14.8 us)
    const Split cut = choose_splits((long long)p.qtiles * p.kv_heads * p.bt.batch, p.bt.batch,
                                    (double)max_len / (kWarps * S::kKeys), 3.0, 8.0, NT == 1 ? 0.14 : 0.26, 2.0,
                                    1.0, most_supers(p),
                                    [&](int n) { return cluster_slots((const void *)kernel, n, kWarps * 32, smem); });
    p.splits = cut.splits;
    p.supers = cut.supers;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.splits * p.supers, p.kv_heads * p.qtiles, p.bt.batch);
    cfg.blockDim = dim3(kWarps * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = p.splits;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, kernel, p);
    return e == cudaSuccess && p.supers > 1 ? launch_join(p, rows::Type<T>::kId, stream) : e;
}

template <typename T, int BITS, int HDP, int NT>
static cudaError_t launch(const AttnParams &p, int max_len, cudaStream_t stream) {
    using S = Slice<HDP, BITS>;
    // Two CTAs of 8 warps an SM; or, where the jobs are so few that clusters of 16 leave one CTA an SM, and the sequences
    // long enough for it, one of 16 warps (16 jobs of 131,001 int8 keys: 102 us so, 90 with 8 warps).
    // Three column tiles need more registers: one CTA of 12 warps.
    const long long base = ((long long)p.max_new * p.group + 8 * NT - 1) / (8 * NT) * p.kv_heads * p.bt.batch;
    if constexpr (NT <= 2) {
        if (base <= 9 && max_len >= 2 * 16 * 16 * S::kKeys) return launch_warps<T, BITS, HDP, NT, 16>(p, max_len, stream);
        return launch_warps<T, BITS, HDP, NT, 8>(p, max_len, stream);
    } else {
        return launch_warps<T, BITS, HDP, NT, 12>(p, max_len, stream);
    }
}

template <typename T, int BITS, int HDP>
static cudaError_t launch_rows(const AttnParams &p, int max_len, cudaStream_t stream) {
    const long long rows = (long long)p.max_new * p.group;
    if (rows <= 8) return launch<T, BITS, HDP, 1>(p, max_len, stream);
    if (rows <= 16) return launch<T, BITS, HDP, 2>(p, max_len, stream);
    return launch<T, BITS, HDP, 3>(p, max_len, stream);
}

template <typename T, int BITS>
static cudaError_t launch_size(const AttnParams &p, int max_len, cudaStream_t stream) {
    // Above 24 rows the tensor-core kernel; above 16 too for heads behind 64 unless P goes in two parts for fp16 callers or a
    // few sequences leave SMs without a second CTA anyway. 24 rows, 8 kv heads, int8, here | there, 64 sequences of 2,000
    // keys and 16 of 4,000: heads of 128, bf16 92 | 86 and 50 | 43 us, fp32 110 | 100 and 66 | 49, fp16 (int4) 92 | 101 and
    // 54 | 50; heads of 64, bf16 66 | 82 and 34 | 41. One sequence of 131,001, bf16: 95 | 98.
    const long long rows = (long long)p.max_new * p.group;
    const bool many = (long long)p.bt.batch * p.kv_heads > 18 && p.head > 64 && rows::Type<T>::kId != rows::kF16;
    if (rows > (many ? 16 : 24)) return launch_tc(p, rows::Type<T>::kId, BITS, max_len, stream);
    return p.head <= 64 ? launch_rows<T, BITS, 64>(p, max_len, stream) : launch_rows<T, BITS, 128>(p, max_len, stream);
}

// A thread takes four elements of a (new token, head): the parts of the clusters, weighted by sum * 2^(max - largest). Few
// rows spread over many blocks, and a thread loads all its parts before it uses one: this is latency only.
template <typename T>
__global__ void __launch_bounds__(128) join_kernel(const AttnParams p) {
    cudaGridDependencySynchronize();  // the blocks are in place when the parts are
    const Sequence s = sequence_at(p, blockIdx.y, &g_attn_error);
    if ((int)blockIdx.x >= s.n) return;
    const int tok = s.row0 + blockIdx.x, quads = p.head / 4, i = blockIdx.z * 128 + threadIdx.x;
    if (i >= p.heads * quads) return;
    const int head = i / quads, d4 = i - head * quads;
    const float2 *ml = work_ml(p) + (size_t)tok * p.heads + head;
    const float *part = p.work + ((size_t)tok * p.heads + head) * p.head + 4 * d4;
    const size_t next = (size_t)p.rows * p.heads;  // rows of one part
    float2 x[kMaxSupers];
    float4 v[kMaxSupers];
#pragma unroll
    for (int w = 0; w < kMaxSupers; w++)
        if (w < p.supers) {
            x[w] = ml[w * next];
            v[w] = *reinterpret_cast<const float4 *>(part + w * next * p.head);
        }
    float m = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kMaxSupers; w++)
        if (w < p.supers) m = fmaxf(m, x[w].x);
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < kMaxSupers; w++) {
        if (w >= p.supers || x[w].y == 0.0f) continue;
        const float f = x[w].y * exp2_fast(x[w].x - m);
        sum += f;
        o.x = __fmaf_rn(f, v[w].x, o.x);
        o.y = __fmaf_rn(f, v[w].y, o.y);
        o.z = __fmaf_rn(f, v[w].z, o.z);
        o.w = __fmaf_rn(f, v[w].w, o.w);
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    store4(static_cast<T *>(p.out) + (size_t)tok * p.out_stride + (size_t)head * p.head + 4 * d4,
           make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
    if (d4 == 0 && p.lse)
        p.lse[(size_t)tok * p.heads + head] = sum == 0.0f ? -INFINITY : (m + log2f(sum)) * 0.693147180559945309f;
}

cudaError_t launch_join(const AttnParams &p, int dtype, cudaStream_t s) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.max_new, p.bt.batch, (p.heads * (p.head / 4) + 127) / 128);
    cfg.blockDim = dim3(128);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (dtype == kF32) return cudaLaunchKernelEx(&cfg, join_kernel<float>, p);
    if (dtype == kBF16) return cudaLaunchKernelEx(&cfg, join_kernel<__nv_bfloat16>, p);
    return cudaLaunchKernelEx(&cfg, join_kernel<__half>, p);
}

int cluster_slots(const void *kernel, int n, int threads, size_t smem) {
    struct Entry {
        const void *kernel;
        int device, n, threads, slots;
        size_t smem;
    };
    static std::mutex mutex;
    static Entry known[1024];
    static int count = 0;
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess) return n == 1 ? 148 : 0;
    std::lock_guard<std::mutex> lock(mutex);
    for (int i = 0; i < count; i++)
        if (known[i].kernel == kernel && known[i].device == device && known[i].n == n && known[i].threads == threads &&
            known[i].smem == smem)
            return known[i].slots;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(n);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = n;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int clusters = 0;
    if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) != cudaSuccess) {
        cudaGetLastError();
        return 0;  // not kept: the next call asks again
    }
    if (count < (int)(sizeof known / sizeof known[0])) known[count++] = Entry{kernel, device, n, threads, clusters * n, smem};
    return clusters * n;
}

int *attn_error_word() {
    void *p = nullptr;
    return cudaGetSymbolAddress(&p, g_attn_error) == cudaSuccess ? static_cast<int *>(p) : nullptr;
}

}  // namespace attn
}  // namespace mvb

using namespace mvb;
using namespace mvb::attn;

// Bytes of workspace that let a call of these sizes split its sequences over more SMs than clusters reach: for few jobs
// (sequences x kv heads x tiles of query rows) with long contexts; 0 where a workspace would not be used.
extern "C" size_t mvb_tree_attention_work(int rows, int heads, int kv_heads, int head, int batch, int max_new, int max_len) {
    if (rows <= 0 || heads <= 0 || kv_heads <= 0 || head <= 0 || batch <= 0 || max_new <= 0) return 0;
    const long long jobs = (long long)batch * kv_heads * (((long long)max_new * (heads / kv_heads) + 255) / 256);
    if (jobs > 18 || max_len < 16384) return 0;
    AttnParams p = {};
    p.rows = rows;
    p.heads = heads;
    p.head = head;
    return work_need(p, kMaxSupers);
}

extern "C" int mvb_tree_attention(const void *q, long long q_stride, const void *kq, const float *ks, const void *vq,
                                  const float *vs, int pages, int page, int kv_heads, int head, int bits,
                                  const int *table, int table_cols, const int *cu, const int *lens, int batch, int rows,
                                  int heads, int dtype, const void *tree, int words, float scale, int max_new,
                                  int max_len, void *out, long long out_stride, float *lse, void *work,
                                  size_t work_bytes, void *stream) {
    const char *who = "mvb_tree_attention";
    if (bits != 4 && bits != 8) {
        set_error("%s: unsupported bits=%d (need 4 or 8)", who, bits);
        return -1;
    }
    if (!rows::known_type(dtype)) {
        set_error("%s: unknown type %d", who, dtype);
        return -1;
    }
    if (pages <= 0 || page < 16 || page > 1024 || (page & (page - 1)) || kv_heads <= 0 || head < 16 || head > 128 ||
        head % 16 || table_cols <= 0 || batch <= 0 || batch > 65535 || rows < 0 || heads <= 0 || heads % kv_heads) {
        set_error("%s: unsupported pages=%d page=%d heads=%d kv_heads=%d head=%d table columns=%d batch=%d rows=%d (need "
                  "page a power of two in 16 .. 1024, head a multiple of 16 in 16 .. 128, heads a multiple of kv_heads, "
                  "batch <= 65535)", who, pages, page, heads, kv_heads, head, table_cols, batch, rows);
        return -1;
    }
    if (max_new < 0 || max_len < 0 || (tree && words < 1) || !(fabsf(scale) <= 3e38f)) {
        set_error("%s: unsupported max_new=%d max_len=%d words=%d scale=%g", who, max_new, max_len, words, (double)scale);
        return -1;
    }
    if (!rows || !max_new) return 0;
    const uintptr_t need = 4 * rows::type_bytes(dtype) - 1;
    if (!q || !out || !kq || !ks || !vq || !vs || !table || !cu || !lens || ((uintptr_t)q & need) ||
        ((uintptr_t)out & need) || ((uintptr_t)kq & 15) || ((uintptr_t)vq & 15) || ((uintptr_t)ks & 15) ||
        ((uintptr_t)vs & 15) || ((uintptr_t)table & 3) || ((uintptr_t)cu & 3) || ((uintptr_t)lens & 3) ||
        ((uintptr_t)tree & 7) || ((uintptr_t)lse & 3) || ((uintptr_t)work & 15) || q_stride % 4 || out_stride % 4) {
        set_error("%s: null or misaligned pointer or stride (cache 16 bytes, q and out four elements, tree 8)", who);
        return -1;
    }
    AttnParams p = {};
    p.q = q;
    p.out = out;
    p.lse = lse;
    p.kq = static_cast<const uint8_t *>(kq);
    p.vq = static_cast<const uint8_t *>(vq);
    p.ks = ks;
    p.vs = vs;
    p.bt.cu = cu;
    p.bt.lens = lens;
    p.bt.table = table;
    p.bt.batch = batch;
    p.bt.table_cols = table_cols;
    p.bt.pages = pages;
    p.bt.page_log2 = 31 - __builtin_clz((unsigned)page);
    p.tree = static_cast<const unsigned long long *>(tree);
    p.words = words;
    p.q_stride = q_stride;
    p.out_stride = out_stride;
    p.scale_log2 = scale * 1.44269504088896341f;
    p.rows = rows;
    p.heads = heads;
    p.kv_heads = kv_heads;
    p.group = heads / kv_heads;
    p.head = head;
    p.max_new = max_new;
    p.work = static_cast<float *>(work);
    p.work_bytes = work ? work_bytes : 0;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (bits == 8)
        e = dtype == rows::kF32 ? launch_size<float, 8>(p, max_len, st)
            : dtype == rows::kBF16 ? launch_size<__nv_bfloat16, 8>(p, max_len, st) : launch_size<__half, 8>(p, max_len, st);
    else
        e = dtype == rows::kF32 ? launch_size<float, 4>(p, max_len, st)
            : dtype == rows::kBF16 ? launch_size<__nv_bfloat16, 4>(p, max_len, st) : launch_size<__half, 4>(p, max_len, st);
    if (e == kTooManyRows) {
        set_error("%s: max_new=%d x heads=%d are too many rows for one call (need ceil(max_new * heads / kv_heads / 128) * "
                  "kv_heads <= 65535)", who, max_new, heads);
        return -1;
    }
    if (e != cudaSuccess) {
        set_error("%s: launch failed: %s", who, cudaGetErrorString(e));
        return -1;
    }
    return 0;
}
