// Attention of a batch's new tokens (one, a chain, or a tree of drafted ones) over the paged 8- or 4-bit cache
// (mvb_tree_attention). The new tokens' keys and values are in the cache already (mvb_kv_append): token i of sequence b
// stands at position ctx + i and sees positions below ctx, and of the new ones those its mask bits allow.
//
//     S = scale * ks[t] * (q . k[t]),  P = exp(S - max),  O = sum_t P[t] vs[t] v[t] / sum_t P[t]
//
// with k and v the cached integers, which fp16 holds exactly: the products take them as they are, the keys' scales
// multiply S and the values' scales multiply P. q is put in fp16 after a power of two of its row's largest element was
// taken out (2 ^ e; a bf16 or fp16 q keeps every bit that is above 2^-33 of the row's largest); an fp32 q goes in two
// parts, high and low (22 bits), and its P too, so that fp32 callers get fp32 results: two products each instead of one.
// Else P is rounded to fp16 once (2^-12), less than the output's own rounding. max, sum and O are fp32.
//
// This kernel: up to 16 * MT query rows (new tokens x the query heads of one kv head) at a time; a handful of rows does
// little arithmetic per cached byte, so the work is to stream the cache. One warp owns 16-key slices (HDP = 128; 32
// keys for HDP = 64): cp.async into its own ring of three stages, no barrier with the other warps; keys go from bytes
// to fp16 fragments of mma.m16n8k16 in registers. The order of the head's elements inside a product is free as long as
// q and k agree, and so is the order of the keys in P v: both are chosen so that a lane reads whole 4- to 16-byte
// pieces. Keys of a sequence are split over the warps of a CTA and over the CTAs of a cluster (up to 16), whose partial
// (max, sum, O) are joined in distributed shared memory in a fixed order: one launch, no workspace, the same bits on
// every run.
#include <cooperative_groups.h>
#include <limits.h>
#include <math.h>

#include "../../include/matvec_b200.h"
#include "mvb_runtime.h"
#include "tree_attention.cuh"

namespace mvb {
namespace attn {

using namespace rows;
namespace cg = cooperative_groups;

static __device__ int g_attn_error;

constexpr int kWarps = 8;
constexpr int kStages = 3;
constexpr float kPScale = 256.0f;   // P' = P * vs * kPScale / W stays below 64 * 256 in fp16
constexpr float kLazy = 6.0f;       // the running maximum moves only when it is 2^6 behind

template <int HDP, int BITS>
struct Slice {
    static constexpr int kKeys = HDP == 128 ? 16 : 32;
    static constexpr int kSub = kKeys / 16;            // 16-key pieces, each inside one page
    static constexpr int kRow = HDP * BITS / 8;        // bytes of a row in shared memory
    static constexpr int kScales = 2 * kKeys * kRow;   // offset of the scales in a stage
    static constexpr int kStage = 2 * kKeys * kRow + 2 * kKeys * 4;
    static constexpr int kWarp = kStages * kStage;
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

__device__ __forceinline__ void cp_async(uint32_t dst, const void *src, int bytes) {
    if (bytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}

// The head element that element e (0 .. 3: k = 2c, 2c + 1, 2c + 8, 2c + 9) of lane column c holds in k-step ks: a lane
// reads 16 elements (64 * (ks / 4) + 16 c ..) at once and spreads them over four k-steps, in byte order for 8 bits, as
// (o, o + 4), (o + 1, o + 5) of each 8 for 4 bits.
template <int BITS>
__device__ __forceinline__ int element_of(int ks, int c, int e) {
    const int base = 64 * (ks >> 2) + 16 * c, w = ks & 3;
    if (BITS == 8) return base + 4 * w + e;
    return base + 8 * (w >> 1) + 2 * (w & 1) + (e >> 1) + 4 * (e & 1);
}

template <typename T, int BITS, int HDP, int MT>
__global__ void __launch_bounds__(kWarps * 32, MT == 1 ? 2 : 1) tree_attention_kernel(const AttnParams p) {
    using S = Slice<HDP, BITS>;
    constexpr int KS = HDP / 16, NT = HDP / 8;   // k-steps of q.k; 8-column tiles of O (tile j: elements NT * n + j)
    constexpr int NP = sizeof(T) == 4 ? 2 : 1;   // parts of q and of P
    constexpr int ROWS = 16 * MT;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float row_factor[ROWS], warp_m[kWarps][ROWS], warp_l[kWarps][ROWS], cta_m[ROWS], cta_l[ROWS];
    uint4 *qfrag = reinterpret_cast<uint4 *>(smem);  // [NP][MT][KS][32 lanes]
    uint8_t *pipe = smem + NP * MT * KS * 512;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    const int b = blockIdx.z, kvh = blockIdx.y / p.qtiles, qt = blockIdx.y - kvh * p.qtiles, split = blockIdx.x;
    const Sequence s = sequence_at(p, b, &g_attn_error);
    const int nrows = s.n * p.group, R0 = qt * ROWS;
    if (R0 >= nrows) return;  // the whole cluster returns together

    // this warp's slices
    const int ns = (s.len + S::kKeys - 1) / S::kKeys;
    const int s0 = (int)((long long)ns * split / p.splits), s1 = (int)((long long)ns * (split + 1) / p.splits);
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
#pragma unroll
            for (int i = 0; i < S::kPieces; i++)
                if (doff[i] >= 0) {
                    cp_async(d + doff[i], kp + 32 * i * piece, piece);
                    cp_async(d + S::kKeys * S::kRow + doff[i], vp + 32 * i * piece, piece);
                }
            const uint32_t ds = mine_u + stage * S::kStage + S::kScales + sub * 64;
            if (lane < 4) cp_async(ds + 16 * lane, p.ks + row + 4 * lane, 16);
            else if (lane < 8) cp_async(ds + S::kKeys * 4 + 16 * (lane - 4), p.vs + row + 4 * (lane - 4), 16);
        }
    };
    int sl_next = s0 + warp;
    for (int st = 0; st < kStages - 1; st++) {
        if (sl_next < s1) issue(sl_next, st);
        sl_next += kWarps;
        asm volatile("cp.async.commit_group;" ::: "memory");
    }

    // q: a warp scales a row by a power of two into fp32 (staged behind the pipeline), then every warp builds fragments
    float *qrow = reinterpret_cast<float *>(pipe + kWarps * S::kWarp);  // [ROWS][HDP]
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
            reinterpret_cast<float4 *>(qrow + i * HDP)[lane] = make_float4(v.x * f, v.y * f, v.z * f, v.w * f);
        }
        if (lane == 0) row_factor[i] = pow2(k);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < MT * KS * 32; i += kWarps * 32) {
        const int ln = i & 31, ks = (i >> 5) % KS, mt = (i >> 5) / KS;
        const float *a = qrow + (mt * 16 + (ln >> 2)) * HDP, *bq = a + 8 * HDP;
        float f[8];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int d = element_of<BITS>(ks, ln & 3, e);
            f[e] = a[d];
            f[4 + e] = bq[d];
        }
        const uint4 hi = make_uint4(pack2<__half>(f[0], f[1]), pack2<__half>(f[4], f[5]), pack2<__half>(f[2], f[3]),
                                    pack2<__half>(f[6], f[7]));
        qfrag[i] = hi;
        if (NP == 2) {
#pragma unroll
            for (int e = 0; e < 8; e++) f[e] = f[e] - __half2float(__float2half_rn(f[e]));
            qfrag[MT * KS * 32 + i] = make_uint4(pack2<__half>(f[0], f[1]), pack2<__half>(f[4], f[5]),
                                                 pack2<__half>(f[2], f[3]), pack2<__half>(f[6], f[7]));
        }
    }
    __syncthreads();

    float O[MT][NT][4], m[MT][2], l[MT][2], rf[MT][2];
    int draft[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) O[mt][j][e] = 0.0f;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            m[mt][h] = -INFINITY;
            l[mt][h] = 0.0f;
            rf[mt][h] = row_factor[mt * 16 + r + 8 * h];
            draft[mt][h] = (R0 + mt * 16 + r + 8 * h) / p.group;
        }
    }
    float W = pow2(-100);  // at or above every |vs| so far, a power of two

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
        const uint8_t *kt = mine + stage * S::kStage, *vt = kt + S::kKeys * S::kRow;
        const float *ksc = reinterpret_cast<const float *>(kt + S::kScales), *vsc = ksc + S::kKeys;
        const int key0 = sl * S::kKeys;

        float sc[MT][S::kSub][2][4];
#pragma unroll
        for (int sub = 0; sub < S::kSub; sub++) {
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int n = 0; n < 2; n++)
#pragma unroll
                    for (int e = 0; e < 4; e++) sc[mt][sub][n][e] = 0.0f;
#pragma unroll
            for (int ch = 0; ch < HDP / 64; ch++) {
                uint32_t kb[2][4][2];  // [8-key tile][k-step of this chunk][b0, b1]
#pragma unroll
                for (int n = 0; n < 2; n++) {
                    const int row = sub * 16 + n * 8 + r;
                    if (BITS == 8) {
                        const uint4 u = *reinterpret_cast<const uint4 *>(kt + place<S::kRow>(row, 64 * ch + 16 * c));
                        const uint32_t w[4] = {u.x ^ 0x80808080u, u.y ^ 0x80808080u, u.z ^ 0x80808080u, u.w ^ 0x80808080u};
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            kb[n][k][0] = bytes_to_half2(w[k], 0x4140u);
                            kb[n][k][1] = bytes_to_half2(w[k], 0x4342u);
                        }
                    } else {
                        const uint2 u = *reinterpret_cast<const uint2 *>(kt + place<S::kRow>(row, 32 * ch + 8 * c));
                        const uint32_t w[2] = {u.x ^ 0x88888888u, u.y ^ 0x88888888u};
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            kb[n][k][0] = nibbles_to_half2(w[k >> 1], 2 * (k & 1));
                            kb[n][k][1] = nibbles_to_half2(w[k >> 1], 2 * (k & 1) + 1);
                        }
                    }
                }
#pragma unroll
                for (int k = 0; k < 4; k++)
#pragma unroll
                    for (int mt = 0; mt < MT; mt++)
#pragma unroll
                        for (int part = 0; part < NP; part++) {
                            const uint4 a = qfrag[((part * MT + mt) * KS + 4 * ch + k) * 32 + lane];
#pragma unroll
                            for (int n = 0; n < 2; n++) mma16816(sc[mt][sub][n], a, kb[n][k][0], kb[n][k][1]);
                        }
            }
        }
        // scales of this lane's keys, the mask, and the values' scales
        const bool tail = key0 + S::kKeys > s.ctx;  // some key is a new token's, or none
        float vv[S::kSub][2][2], mv = 0.0f;
#pragma unroll
        for (int sub = 0; sub < S::kSub; sub++)
#pragma unroll
            for (int n = 0; n < 2; n++) {
                const int i = sub * 16 + n * 8 + 2 * c;
                const float2 k2 = *reinterpret_cast<const float2 *>(ksc + i);
                const float2 v2 = *reinterpret_cast<const float2 *>(vsc + i);
                const float kk[2] = {k2.x * p.scale_log2, k2.y * p.scale_log2};
                vv[sub][n][0] = key0 + i < s.len ? v2.x : 0.0f;
                vv[sub][n][1] = key0 + i + 1 < s.len ? v2.y : 0.0f;
                // (an infinite scale makes the rows that see it infinite; it must not set W for the others)
#pragma unroll
                for (int e = 0; e < 2; e++)
                    if (fabsf(vv[sub][n][e]) < INFINITY) mv = fmaxf(mv, fabsf(vv[sub][n][e]));
#pragma unroll
                for (int mt = 0; mt < MT; mt++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        float u = sc[mt][sub][n][e] * kk[e & 1];
                        if (tail && !allowed(p, s, draft[mt][e >> 1], key0 + i + (e & 1))) u = -INFINITY;
                        sc[mt][sub][n][e] = u;
                    }
            }
        mv = fmaxf(mv, __shfl_xor_sync(0xffffffffu, mv, 1));
        mv = fmaxf(mv, __shfl_xor_sync(0xffffffffu, mv, 2));
        // running maxima (log2 units); they move only when some row is kLazy behind
        float mx[MT][2];
        bool move = mv > W;
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                float x = -INFINITY;
#pragma unroll
                for (int sub = 0; sub < S::kSub; sub++)
#pragma unroll
                    for (int n = 0; n < 2; n++) x = fmaxf(x, fmaxf(sc[mt][sub][n][2 * h], sc[mt][sub][n][2 * h + 1]));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
                mx[mt][h] = fmaxf(m[mt][h], x * rf[mt][h]);
                move |= mx[mt][h] > m[mt][h] + kLazy || (m[mt][h] == -INFINITY && mx[mt][h] != -INFINITY);
            }
        if (__any_sync(0xffffffffu, move)) {
            float wf = 1.0f;
            if (mv > W) {
                const float w2 = pow2(min(exponent_of(mv) - 127 + 1, 127));
                wf = W / w2;
                W = w2;
            }
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const float a = m[mt][h] == -INFINITY ? 0.0f : exp2_fast(m[mt][h] - mx[mt][h]);
                    m[mt][h] = mx[mt][h];
                    l[mt][h] *= a;
                    const float f = a * wf;
#pragma unroll
                    for (int j = 0; j < NT; j++) {
                        O[mt][j][2 * h] *= f;
                        O[mt][j][2 * h + 1] *= f;
                    }
                }
        }
        const float vf = kPScale / W;
#pragma unroll
        for (int sub = 0; sub < S::kSub; sub++) {
            uint4 P[MT][NP];
#pragma unroll
            for (int mt = 0; mt < MT; mt++) {
                float pv[2][4];
#pragma unroll
                for (int n = 0; n < 2; n++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int h = e >> 1;
                        const float base = m[mt][h] == -INFINITY ? 0.0f : m[mt][h];
                        const float x = exp2_fast(__fmaf_rn(sc[mt][sub][n][e], rf[mt][h], -base));
                        l[mt][h] += x;
                        // a masked key's value scale may be anything: its weight is zero, not zero times that
                        pv[n][e] = sc[mt][sub][n][e] == -INFINITY ? 0.0f : x * (vv[sub][n][e & 1] * vf);
                    }
                P[mt][0] = make_uint4(pack2<__half>(pv[0][0], pv[0][1]), pack2<__half>(pv[0][2], pv[0][3]),
                                      pack2<__half>(pv[1][0], pv[1][1]), pack2<__half>(pv[1][2], pv[1][3]));
                if (NP == 2) {
#pragma unroll
                    for (int n = 0; n < 2; n++)
#pragma unroll
                        for (int e = 0; e < 4; e++) pv[n][e] -= __half2float(__float2half_rn(pv[n][e]));
                    P[mt][NP - 1] = make_uint4(pack2<__half>(pv[0][0], pv[0][1]), pack2<__half>(pv[0][2], pv[0][3]),
                                               pack2<__half>(pv[1][0], pv[1][1]), pack2<__half>(pv[1][2], pv[1][3]));
                }
            }
            // values: lane (r, c) takes elements NT * r .. of keys 2c, 2c + 1, 2c + 8, 2c + 9 of this piece
            constexpr int WORDS = NT * BITS / 32;  // 32-bit words of a key's elements: 4, 2 (8 bits), 2, 1 (4 bits)
            uint32_t w[4][WORDS];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const uint8_t *src = vt + place<S::kRow>(sub * 16 + 2 * c + (k & 1) + 8 * (k >> 1), r * WORDS * 4);
                if constexpr (WORDS == 4) {
                    const uint4 u = *reinterpret_cast<const uint4 *>(src);
                    w[k][0] = u.x; w[k][1] = u.y; w[k][2] = u.z; w[k][3] = u.w;
                } else if constexpr (WORDS == 2) {
                    const uint2 u = *reinterpret_cast<const uint2 *>(src);
                    w[k][0] = u.x; w[k][1] = u.y;
                } else {
                    w[k][0] = *reinterpret_cast<const uint32_t *>(src);
                }
#pragma unroll
                for (int i = 0; i < WORDS; i++) w[k][i] ^= BITS == 8 ? 0x80808080u : 0x88888888u;
            }
#pragma unroll
            for (int i = 0; i < WORDS; i++) {
                constexpr int PER = 32 / BITS;  // elements a word
                uint32_t vb[PER][2];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    if (BITS == 8) {
                        const uint32_t lo = __byte_perm(w[2 * h][i], w[2 * h + 1][i], 0x5140);
                        const uint32_t hi = __byte_perm(w[2 * h][i], w[2 * h + 1][i], 0x7362);
                        vb[0][h] = bytes_to_half2(lo, 0x4140u);
                        vb[1][h] = bytes_to_half2(lo, 0x4342u);
                        vb[2][h] = bytes_to_half2(hi, 0x4140u);
                        vb[3][h] = bytes_to_half2(hi, 0x4342u);
                    } else {
                        const uint32_t lo = __byte_perm(w[2 * h][i], w[2 * h + 1][i], 0x5410);
                        const uint32_t hi = __byte_perm(w[2 * h][i], w[2 * h + 1][i], 0x7632);
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            vb[k][h] = nibbles_to_half2(lo, k);
                            vb[(4 + k) % PER][h] = nibbles_to_half2(hi, k);
                        }
                    }
                }
#pragma unroll
                for (int k = 0; k < PER; k++)
#pragma unroll
                    for (int mt = 0; mt < MT; mt++)
#pragma unroll
                        for (int part = 0; part < NP; part++)
                            mma16816(O[mt][PER * i + k], P[mt][part], vb[k][0], vb[k][1]);
            }
        }
        __syncwarp();  // every lane has read the stage before the next turn refills it
        stage = stage + 1 == kStages ? 0 : stage + 1;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();

    // join the warps: O in its own units to shared memory, then (max, sum) of each row
    float *po = reinterpret_cast<float *>(pipe);  // [kWarps][ROWS][HDP]
    const float back = W / kPScale;
#pragma unroll
    for (int mt = 0; mt < MT; mt++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            float sum = l[mt][h];
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            const int row = mt * 16 + r + 8 * h;
            if (c == 0) {
                warp_m[warp][row] = m[mt][h];
                warp_l[warp][row] = sum;
            }
            float *d = po + ((size_t)warp * ROWS + row) * HDP + NT * 2 * c;
#pragma unroll
            for (int e = 0; e < 2; e++)
#pragma unroll
                for (int j = 0; j < NT; j += 4)
                    *reinterpret_cast<float4 *>(d + NT * e + j) =
                        make_float4(O[mt][j][2 * h + e] * back, O[mt][j + 1][2 * h + e] * back,
                                    O[mt][j + 2][2 * h + e] * back, O[mt][j + 3][2 * h + e] * back);
        }
    __syncthreads();
    const int rows_here = min(ROWS, nrows - R0);
    auto finish = [&](int row, int d4, float4 o, float sum, float mm) {
        const int R = R0 + row, tok = s.row0 + R / p.group, head = kvh * p.group + R % p.group;
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;  // no key: o is zero too
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
    for (int i = threadIdx.x * p.splits + split; i < rows_here * (HDP / 4); i += kWarps * 32 * p.splits) {
        const int row = i / (HDP / 4), d4 = i % (HDP / 4);
        float mm = -INFINITY;
        for (int w = 0; w < p.splits; w++) mm = fmaxf(mm, *cluster.map_shared_rank(&cta_m[row], w));
        float sum = 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int w = 0; w < p.splits; w++) {
            const float lw = *cluster.map_shared_rank(&cta_l[row], w);
            if (lw == 0.0f) continue;
            const float f = exp2_fast(*cluster.map_shared_rank(&cta_m[row], w) - mm);
            const float4 x = *reinterpret_cast<const float4 *>(cluster.map_shared_rank(po + (size_t)row * HDP + 4 * d4, w));
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

template <typename T, int BITS, int HDP, int MT>
static cudaError_t launch(AttnParams p, int max_len, cudaStream_t stream) {
    using S = Slice<HDP, BITS>;
    constexpr int ROWS = 16 * MT, NP = sizeof(T) == 4 ? 2 : 1;
    constexpr size_t frag = (size_t)NP * MT * (HDP / 16) * 512;
    constexpr size_t ring = (size_t)kWarps * S::kWarp + (size_t)ROWS * HDP * 4, join = (size_t)kWarps * ROWS * HDP * 4;
    constexpr size_t smem = frag + (ring > join ? ring : join);
    static_assert(smem <= 227 * 1024 - 4096, "shared memory of a CTA");
    auto kernel = tree_attention_kernel<T, BITS, HDP, MT>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    p.qtiles = (int)(((long long)p.max_new * p.group + ROWS - 1) / ROWS);
    if ((long long)p.qtiles * p.kv_heads > 65535) return cudaErrorInvalidConfiguration;
    const long long base = (long long)p.qtiles * p.kv_heads * p.bt.batch;
    // split a sequence over more CTAs while the grid leaves SMs idle and every warp still has a slice
    int splits = 1;
    while (splits < 16 && base * splits * 2 <= 2 * 148 && (long long)splits * 2 * kWarps * S::kKeys <= max_len) splits *= 2;
    p.splits = splits;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(splits, p.kv_heads * p.qtiles, p.bt.batch);
    cfg.blockDim = dim3(kWarps * 32);
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

template <typename T, int BITS>
static cudaError_t launch_size(const AttnParams &p, int max_len, cudaStream_t stream) {
    const bool wide = (long long)p.max_new * p.group > 16;
    if (p.head <= 64) return wide ? launch<T, BITS, 64, 2>(p, max_len, stream) : launch<T, BITS, 64, 1>(p, max_len, stream);
    return wide ? launch<T, BITS, 128, 2>(p, max_len, stream) : launch<T, BITS, 128, 1>(p, max_len, stream);
}

int attn_take_error(cudaStream_t s) {
    int v = 0;
    if (cudaMemcpyFromSymbolAsync(&v, g_attn_error, sizeof v, 0, cudaMemcpyDeviceToHost, s) != cudaSuccess ||
        cudaStreamSynchronize(s) != cudaSuccess)
        return -1;
    const int z = 0;
    if (v && (cudaMemcpyToSymbolAsync(g_attn_error, &z, sizeof z, 0, cudaMemcpyHostToDevice, s) != cudaSuccess ||
              cudaStreamSynchronize(s) != cudaSuccess))
        return -1;
    return v;
}

}  // namespace attn
}  // namespace mvb

using namespace mvb;
using namespace mvb::attn;

extern "C" int mvb_tree_attention(const void *q, long long q_stride, const void *kq, const float *ks, const void *vq,
                                  const float *vs, int pages, int page, int kv_heads, int head, int bits,
                                  const int *table, int table_cols, const int *cu, const int *lens, int batch, int rows,
                                  int heads, int dtype, const void *tree, int words, float scale, int max_new,
                                  int max_len, void *out, long long out_stride, float *lse, void *stream) {
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
        ((uintptr_t)tree & 7) || ((uintptr_t)lse & 3) || q_stride % 4 || out_stride % 4) {
        set_error("%s: null or misaligned pointer or stride (cache 16 bytes, q and out four elements, tree 8)", who);
        return -1;
    }
    if (((long long)max_new * (heads / kv_heads) + 15) / 16 * kv_heads > 65535) {
        set_error("%s: max_new=%d x heads=%d are too many rows for one call", who, max_new, heads);
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
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (bits == 8)
        e = dtype == rows::kF32 ? launch_size<float, 8>(p, max_len, st)
            : dtype == rows::kBF16 ? launch_size<__nv_bfloat16, 8>(p, max_len, st) : launch_size<__half, 8>(p, max_len, st);
    else
        e = dtype == rows::kF32 ? launch_size<float, 4>(p, max_len, st)
            : dtype == rows::kBF16 ? launch_size<__nv_bfloat16, 4>(p, max_len, st) : launch_size<__half, 4>(p, max_len, st);
    if (e != cudaSuccess) {
        set_error("%s: launch failed: %s", who, cudaGetErrorString(e));
        return -1;
    }
    return 0;
}
