// mvb_tree_attention for many query rows (new tokens x the query heads of one kv head): trees of dozens of tokens, prompt
// chunks. Same arithmetic as tree_attention.cu (exact integers in fp16, one scale a row, fp32 statistics), on the
// 5th-generation tensor cores, since each cached byte now meets 17 to 256 rows.
//
// One CTA: up to MT = 2 tiles of 128 query rows against 64 keys a step. The cache is converted once for all rows: raw
// pages -> (bulk copies) -> raw bytes -> (converter warps) -> fp16 tiles in the 128-byte swizzled layout, two of each. Keys
// are the K-major B operand of S = Q K^T; values, stored by key, are the MN-major B operand of O += P V. P is the A
// operand in tensor memory, written over the S it came from. Tensor memory: two 64-column slots of S for each row tile
// (so that the next step's scores stand ready when a softmax ends), then O0 | O1, 128 columns each.
//
// Warp roles (768 threads):
//   warp 0          one thread issues the MMAs: PV0 QK0'' PV1 QK1'' a step. (The oldest warp, which the scheduler prefers:
//                   as warp 12 it waited for issue slots behind the softmax.)
//   warp 1          with two row tiles, bulk copies of the raw pages, as many stages ahead as fit (3 to 6); with one the
//                   converters' own, which then have the time for it.
//   warps 2, 4, 6 and 3, 5, 7  converters of K, of V, a step's tile a warp: bytes -> fp16; the scales.
//   warps 8-15, 16-23  softmax of row tile 0, 1: two threads a row, 32 of the step's keys each, so that every scheduler has
//                   four such warps to hide one another's latencies (with one thread a row, 64 keys each, a step took 2,350
//                   clocks). S from tensor memory, keys' scales, maximum, exponentials, values' scales, P in fp16 back to
//                   tensor memory. A row's unit moves only when it has to (then O is scaled in tensor memory, after the product
//                   before has ended): a row's two threads vote on that with the barrier that also keeps either's P off
//                   the other's unread S, and exchange their maxima only then. The vote asks the step's largest score and
//                   its largest value scale; only where both together might pass is the product looked at key by key. The
//                   unit is folded into the exponent, so it multiplies P and the row's sum alike.
// What bounds it: for two row tiles of head 128 and 64 keys the exponentials take 1,024 clocks (16 a clock), the MMAs
// 1,280 (QK at N = 64 waits for shared memory: 48 clocks a product against 32), and shared memory carries 224 KB, 1,800
// clocks (QK's operands 96, PV's 32, the conversion 64, the softmax's scales 32); the step takes about 2,300. 16 trees of 64
// tokens, 16,000 keys, 32 heads of 128 over 8 kv heads, int8, bf16: 170 us in a burst (631 TFLOP/s), 184 for a second on end,
// where the power limit takes a tenth of the clock; their longest sequence's CTAs, 125 steps, take most of it. With one row
// tile the chain of a step is the bound (64 sequences of 2,000 keys, 32 | 128 rows: 88 | 106 us, 1,500 | 1,800 clocks a step).
// Up to 128 query rows (MT = 1): both softmax groups take the same rows, for every other step each, with an O and
// (max, sum) of their own; the two parts are joined like those of the cluster.
// The keys of a sequence are split over the CTAs of a cluster, joined in distributed shared memory in a fixed order.
// Every mbarrier wait is bounded (1 s): a wait that runs out notes the error and the roles stop.
// Every barrier is waited on before its next phase can end (each role's next arrival needs what the waiter does after),
// and by a warp that has seen the phase before.
#include <cooperative_groups.h>
#include <math.h>

#include <type_traits>

#include "../../include/matvec_b200.h"
#include "barriers.cuh"
#include "mvb_runtime.h"
#include "tree_attention.cuh"

namespace mvb {
namespace attn {

using namespace rows;
namespace cg = cooperative_groups;

static __device__ int g_tc_error;
__device__ __forceinline__ bool bar_wait(uint64_t *bar, uint32_t parity) { return rows::bar_wait(bar, parity, &g_tc_error); }
constexpr int kTcThreads = 768;
constexpr int kMmaWarp = 0, kLoadWarp = 1;  // first, since the scheduler prefers the oldest warp
constexpr int kBN = 64;              // keys a step
// A parity says which of two phases a barrier is in, so a waiter must have seen the phase before: the barriers that several
// warps of a kind wait on in turn are as many as make the same warp wait on each (multiples of 3).
constexpr int kTurns = 6;            // barriers of raw stages filled and read, and of tiles set free
constexpr int kScales = 8;           // steps whose scales are kept

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar))
                 : "memory");
}
// One lane of a converged warp. The compiler knows that a branch on elect.sync has one lane, and keeps the products'
// descriptors in uniform registers across it; from a branch on the lane number, or with the products predicated, each
// takes ten instructions more to issue (with busy warps beside it 400 clocks against the 64 that it runs).
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}

// Shared-memory matrix descriptor of a 128-byte swizzled tile: rows of 128 bytes, 8-row groups 1024 bytes apart (stride
// offset); lead: from one block of 64 elements to the next along the major dimension (MN-major tiles only).
__device__ __forceinline__ uint64_t tile_desc(uint32_t addr, uint32_t lead) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)(lead >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// Instruction descriptor of kind::f16: D fp32 (bits 4-5 = 1), A and B fp16, B MN-major in bit 16, N >> 3 in bits 17-22,
// M >> 4 in bits 24-28.
__host__ __device__ constexpr uint32_t idesc_f16(int m, int n, bool b_mn) {
    return (1u << 4) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
        : "memory");
}

// 32 or 16 consecutive columns of this thread's lane, and 16 back.
__device__ __forceinline__ void tmem_load32(uint32_t addr, float *r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]),
          "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]), "=f"(r[16]),
          "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]),
          "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_load16(uint32_t addr, float *r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15}, [%16];"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]),
          "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_store16(uint32_t addr, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Pairs of fp32 in one instruction.
__device__ __forceinline__ uint64_t pair2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void split2(uint64_t p, float &a, float &b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p));
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

__device__ __forceinline__ float max3(float a, float b, float c) {  // the largest that is a number
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// Sixteen cached integers (16 bytes, or 8 of nibbles) as fp16 in their order: two 16-byte pieces.
template <int BITS>
__device__ __forceinline__ uint4 load_sixteen(const uint8_t *src) {
    if (BITS == 8) return *reinterpret_cast<const uint4 *>(src);
    const uint2 u = *reinterpret_cast<const uint2 *>(src);
    return make_uint4(u.x, u.y, 0, 0);
}
template <int BITS>
__device__ __forceinline__ void sixteen(uint4 u, uint4 &a, uint4 &b) {
    uint32_t h[8];
    if (BITS == 8) {
        const uint32_t w[4] = {u.x ^ 0x80808080u, u.y ^ 0x80808080u, u.z ^ 0x80808080u, u.w ^ 0x80808080u};
        const uint32_t bias = 0x64806480u;  // 1024 + 128
#pragma unroll
        for (int i = 0; i < 4; i++) {
            h[2 * i] = __byte_perm(w[i], 0x64646464u, 0x4140);
            h[2 * i + 1] = __byte_perm(w[i], 0x64646464u, 0x4342);
            asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(h[2 * i]) : "r"(bias));
            asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(h[2 * i + 1]) : "r"(bias));
        }
    } else {
        const uint32_t w[2] = {u.x, u.y};
#pragma unroll
        for (int i = 0; i < 2; i++) {
            uint32_t g[4];  // (k, k + 4)
#pragma unroll
            for (int k = 0; k < 4; k++) g[k] = nibbles_to_half2(w[i], k);
            h[4 * i] = __byte_perm(g[0], g[1], 0x5410);
            h[4 * i + 1] = __byte_perm(g[2], g[3], 0x5410);
            h[4 * i + 2] = __byte_perm(g[0], g[1], 0x7632);
            h[4 * i + 3] = __byte_perm(g[2], g[3], 0x7632);
        }
    }
    a = make_uint4(h[0], h[1], h[2], h[3]);
    b = make_uint4(h[4], h[5], h[6], h[7]);
}

// 32 mask bits of new tokens j .. j + 31 for new token i (negative j: cached positions, allowed).
__device__ __forceinline__ uint32_t mask32(const AttnParams &p, const Sequence &s, int i, int j) {
    if (i >= s.n) return j + 31 < 0 ? 0xFFFFFFFFu : j < 0 ? (1u << -j) - 1 : 0u;
    auto from = [&](int k) -> uint32_t {  // bits of k .. k + 31, k >= 0
        uint32_t w;
        if (!p.tree) {
            w = i < k ? 0u : i - k >= 31 ? 0xFFFFFFFFu : (2u << (i - k)) - 1;
        } else {
            const unsigned long long *t = p.tree + (size_t)(s.row0 + i) * p.words;
            const int at = k >> 6, sh = k & 63;
            unsigned long long x = at < p.words ? t[at] >> sh : 0ull;
            if (sh > 32 && at + 1 < p.words) x |= t[at + 1] << (64 - sh);
            w = (uint32_t)x;
        }
        return s.n - k >= 32 ? w : s.n <= k ? 0u : w & ((1u << (s.n - k)) - 1);
    };
    if (j >= 0) return from(j);
    if (j <= -32) return 0xFFFFFFFFu;
    return (from(0) << -j) | ((1u << -j) - 1);
}

template <int QP, int BITS, int HDP, int MT>
struct TcSmem {
    static constexpr int kBlocks = HDP / 64;                      // blocks of 64 elements (128 bytes)
    static constexpr int kQTile = kBlocks * 128 * 128;            // an fp16 tile of 128 rows
    static constexpr int kTile = kBlocks * kBN * 128;             // of kBN keys
    static constexpr int kQ = 0;                                  // [MT][QP] tiles
    static constexpr int kK = kQ + MT * QP * kQTile;              // [2]
    static constexpr int kV = kK + 2 * kTile;                     // [2]
    static constexpr int kRawRow = HDP * BITS / 8;
    static constexpr int kRawTile = kBN * kRawRow;
    static constexpr int kRawAt = kV + 2 * kTile;                 // [kRaw] K
    static constexpr int kRawV = kRawTile + 2 * kBN * 4;          // a stage of V | ks | vs
    static constexpr int kRawStage = kRawTile + kRawV;
    // raw stages of keys and of values, as many as fit, up to 6; rings of their own, since keys are converted up to four
    // steps before their values are
    static constexpr int kRest = 32 * 1024;  // what follows the stages, at most
    static constexpr int kFit = (227 * 1024 - kRest - kRawAt) / kRawStage;
    static constexpr int kRaw = kFit >= 6 ? 6 : MT == 1 && kFit == 5 ? 4 : kFit;
    // MT = 1: the barrier of step j + kRaw (% kTurns) was step j + kRaw - kTurns's: complete when step j's stage is refilled, since
    // j's tile was only free after step j - 2 (or it is the same warp's); not so for 5 stages
    static_assert(kRaw >= 3 && !(MT == 1 && kRaw == 5), "raw stages");
    // the partial O of both softmax groups, [256][HDP] fp32, lies over the tiles
    static constexpr int kJoin = 256 * HDP * 4;
    static constexpr int kRawVAt = kRawAt + kRaw * kRawTile;      // [kRaw] V | ks | vs
    static constexpr int kEnd = kRawAt + kRaw * kRawStage;
    static constexpr int kScale = kEnd > kJoin ? kEnd : kJoin;    // [kScales][kk | vv] fp32
    static constexpr int kRow = kScale + kScales * 2 * kBN * 4;   // row factors [MT][128]
    static constexpr int kXm = kRow + MT * 128 * 4;               // what a row's two threads exchange [2][2][128]
    static constexpr int kMl = kXm + 4 * 128 * 4;               // (max, sum) of both groups' rows [2][256]
    static constexpr int kAll = kMl + 2 * 256 * 4;                // every part's weights, and their sums [MT * 128]
    static constexpr int kAllEnd = kAll + (kMaxSplits * (3 - MT) + 1) * MT * 128 * 4;
    static constexpr int kPmBytes = kMaxSplits * (3 - MT) * MT * 128 * 4;  // every part's maxima, behind the partial O
    static constexpr bool kPmInside = kEnd - kJoin >= kPmBytes;
    static constexpr int kPm = kPmInside ? kJoin : kAllEnd;
    static constexpr int kBar = kAllEnd + (kPmInside ? 0 : kPmBytes);
    static constexpr size_t kBytes = kBar + 640 + 1024;           // + alignment
    static_assert(kBytes <= 227 * 1024, "shared memory of a CTA");
};

// Before the first product of a span: a thread's half of O, from column `at` on, goes into its sums, whose last element is the
// unit they are in. Heads up to 64 leave tensor memory free behind O, which holds the sums then; else they are in local
// memory. A call of its own, so that the steps keep their registers.
template <int HDP>
__device__ __noinline__ void keep(float *sums, uint32_t at, float unit, bool first, uint64_t *pv_done, uint32_t parity) {
    constexpr bool TM = HDP == 64;
    bar_wait(pv_done, parity);
    fence_after();
    float &in = sums[TM ? 0 : HDP / 2];
    const float f = first ? 0.0f : unit_factor(in, unit);
    in = unit;
#pragma unroll 1
    for (int c = 0; c < HDP / 2; c += 16) {
        float o[16];
        tmem_load16(at + c, o);
        if constexpr (TM) {
            float had[16];
            tmem_load16(at + HDP + c, had);
            wait_load();
#pragma unroll
            for (int e = 0; e < 16; e++) had[e] = first ? o[e] : __fmaf_rn(had[e], f, o[e]);
            tmem_store16(at + HDP + c, reinterpret_cast<const uint32_t *>(had));
        } else {
            wait_load();
#pragma unroll
            for (int e = 0; e < 16; e++) sums[c + e] = first ? o[e] : __fmaf_rn(sums[c + e], f, o[e]);
        }
    }
    if (TM) wait_store();
}

template <typename T, int QP, int PP, int BITS, int HDP, int MT>
__global__ void __launch_bounds__(kTcThreads, 1) tree_attention_tc_kernel(const AttnParams p) {
    using S = TcSmem<QP, BITS, HDP, MT>;
    constexpr int ROWS = MT * 128;
    constexpr bool ALT = MT == 1;            // the groups alternate over the steps
    constexpr int PARTS = ALT ? 2 : 1;       // partial results of a row in a CTA
    constexpr int kRaw = S::kRaw;
    // The products' sums are cut towards zero at 2^-23 for every 16 keys and part, which adds up: values of one sign lost
    // 1e-5 over 4,096 keys of an fp32 caller and 2e-3 over 500,000. So a group's product starts anew every kSpan steps, and its
    // threads add what there was to sums of their own, rounded to nearest. That takes about 3,000 clocks for heads of 128 (the
    // sums, 260 bytes a thread, come from L2). bf16 callers, whose output's half step is 4e-3 and whose products have one
    // part, go without.
    constexpr int kSpan = PP == 1 ? 1 << 30 : sizeof(T) == 4 ? 16 : 128;
    constexpr bool SPANS = PP > 1;
    extern __shared__ __align__(1024) uint8_t raw_smem[];
    uint8_t *smem = raw_smem + ((1024u - (smem_addr(raw_smem) & 1023u)) & 1023u);
    uint64_t *bar = reinterpret_cast<uint64_t *>(smem + S::kBar);
    // (slot = step & 1 where there are two, step % kScales of scales, % kTurns of raw stages and of tiles set free)
    uint64_t *raw_full = bar, *raw_empty = raw_full + 2 * kTurns /* K, V */, *k_ready = raw_empty + 2 * kTurns, *k_free = k_ready + 2,
             *v_ready = k_free + kTurns, *v_free = v_ready + 2, *s_full = v_free + kTurns /* [m][slot] */,
             *p_ready = s_full + 4 /* [m][slot] */, *pv_done = p_ready + 4 /* [m] */, *sc_ready = pv_done + 2,
             *q_ready = sc_ready + kScales, *o_done = q_ready + 1;
    uint32_t *tmem_at = reinterpret_cast<uint32_t *>(o_done + 1);
    float *limits = reinterpret_cast<float *>(bar + 62);  // [kScales] of the rows' units beside each step's value scales
    float *row_factor = reinterpret_cast<float *>(smem + S::kRow);
    float *cta_m = reinterpret_cast<float *>(smem + S::kMl), *cta_l = cta_m + 256;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int b = blockIdx.z, kvh = blockIdx.y / p.qtiles, qt = blockIdx.y - kvh * p.qtiles;
    const int split = blockIdx.x % p.splits, super = blockIdx.x / p.splits;
    const Sequence s = sequence_at(p, b, &g_tc_error);
    const int nrows = s.n * p.group, R0 = qt * ROWS;
    if (R0 >= nrows) return;  // the whole cluster returns together
    const int nt = (s.len + kBN - 1) / kBN;
    const int t0 = (int)((long long)nt * blockIdx.x / gridDim.x), t1 = (int)((long long)nt * (blockIdx.x + 1) / gridDim.x);
    const int mine = t1 - t0;

    if (tid == 0) {
        for (int i = 0; i < 2 * kTurns; i++) {
            bar_init(&raw_full[i], 1);
            bar_init(&raw_empty[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            bar_init(&k_ready[i], 1);
            bar_init(&v_ready[i], 1);
            bar_init(&pv_done[i], 1);
        }
        for (int i = 0; i < 4; i++) {
            bar_init(&s_full[i], 1);
            bar_init(&p_ready[i], 8);
        }
        for (int i = 0; i < kScales; i++) bar_init(&sc_ready[i], 1);
        for (int i = 0; i < kTurns; i++) {
            bar_init(&k_free[i], 1);
            bar_init(&v_free[i], 1);
        }
        bar_init(q_ready, 16);
        bar_init(o_done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_at)), "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_at;
    const int row_bytes = p.head * BITS / 8;

    if (warp < 8) {
        // raw pages
        const int run = min(1 << p.bt.page_log2, kBN), runs = kBN / run;  // keys a copy, copies a step
        const int *entries = p.bt.table + (size_t)b * p.bt.table_cols;
        auto entry = [&](int j) {  // this lane's entry of the page table in step j
            const int key = (t0 + j) * kBN + lane * run;
            return lane < runs && j < mine && key < s.len ? entries[key >> p.bt.page_log2] : 0;
        };
        auto stage = [&](int kv, int j) {
            return smem + (kv ? S::kRawVAt + j % kRaw * S::kRawV : S::kRawAt + j % kRaw * S::kRawTile);
        };
        auto load = [&](int kv, int j, int found) {  // a step's keys, or its values and both scales
            uint64_t *full = &raw_full[kv * kTurns + j % kTurns];
            uint8_t *raw = stage(kv, j);
            const int key = (t0 + j) * kBN + lane * run;
            const bool on = lane < runs && key < s.len;
            const uint32_t n = __popc(__ballot_sync(0xffffffffu, on));
            if (lane == 0) bar_expect(full, n * (uint32_t)run * (row_bytes + (kv ? 8 : 0)));
            __syncwarp();
            if (on) {
                const size_t row = (((size_t)checked_page(p, found, &g_tc_error) * p.kv_heads + kvh) << p.bt.page_log2) +
                                   (key & ((1 << p.bt.page_log2) - 1));
                const uint32_t bytes = run * row_bytes;
                bulk_load(raw + lane * bytes, (kv ? p.vq : p.kq) + row * row_bytes, bytes, full);
                if (kv) {
                    uint8_t *sc = raw + S::kRawTile + lane * run * 4;
                    bulk_load(sc, p.ks + row, run * 4, full);
                    bulk_load(sc + kBN * 4, p.vs + row, run * 4, full);
                }
            }
        };
        if (warp >= 2) {
            // ---------------- converters: a tile a warp, two keys a lane ----------------
            // warps 2, 4, 6 take the keys of every third step, 3, 5, 7 the values (two warps a tile, every tile: waits and
            // fences of each step took as long as its conversion, 2,300 clocks together)
            const int kv = warp & 1, pieces = p.head / 16;
            uint64_t *ready = kv ? v_ready : k_ready, *free_ = kv ? v_free : k_free;
            uint8_t *tiles = smem + (kv ? S::kV : S::kK);
            if (pieces < HDP / 16 && warp < 6)  // the columns behind the head are never converted: zeros add nothing
                for (int i = lane; i < S::kTile / 16; i += 32)
                    reinterpret_cast<uint4 *>(tiles + ((warp - 2) >> 1) * S::kTile)[i] = make_uint4(0, 0, 0, 0);
            asm volatile("bar.sync 1, 192;" ::: "memory");
            // ALT: a warp that has converted a step's tile refills its stage with the step kRaw ahead (a loader, which shares
            // its scheduler with the softmax, came too late: one sequence of 131,001 keys, 64 rows, 123 us against 105)
            int j = (warp - 2) >> 1;
            if (ALT) {
                const int found0 = entry(j), found1 = entry(j + 3);
                if (j < mine) load(kv, j, found0);
                if (j + 3 < min(mine, kRaw)) load(kv, j + 3, found1);
            }
            for (; j < mine; j += 3) {
                const int found = ALT ? entry(j + kRaw) : 0;
                const int slot = j & 1, turn = j % kTurns, ss = j % kScales;
                const uint8_t *raw = stage(kv, j);
                if (!bar_wait(&raw_full[kv * kTurns + turn], (j / kTurns) & 1)) break;
                if (kv) {
                    // the scales, before the tile is free: the softmax of kScales steps ago, their last reader, is done (this
                    // warp's step before last waited for the product of five steps ago)
                    float *sc = reinterpret_cast<float *>(smem + S::kScale) + ss * 2 * kBN;
                    const float *rsc = reinterpret_cast<const float *>(raw + S::kRawTile);
                    float mv = 0.0f;
#pragma unroll
                    for (int key = lane; key < kBN; key += 32) {
                        const bool live = (t0 + j) * kBN + key < s.len;
                        const float x = live ? rsc[kBN + key] : 0.0f;
                        sc[key] = live ? rsc[key] * p.scale_log2 : 0.0f;
                        sc[kBN + key] = x;
                        if (fabsf(x) < INFINITY) mv = fmaxf(mv, fabsf(x));  // an infinite scale limits no unit
                    }
#pragma unroll
                    for (int o = 16; o; o >>= 1) mv = fmaxf(mv, __shfl_xor_sync(0xffffffffu, mv, o));
                    if (lane == 0) limits[ss] = unit_limit(mv);
                    __syncwarp();
                    if (lane == 0) bar_arrive(&sc_ready[ss]);
                }
                // the tile's last product has ended
                if (j >= 2 && !bar_wait(&free_[(j - 2) % kTurns], ((j - 2) / kTurns) & 1)) break;
#pragma unroll 1
                for (int key = lane; key < kBN; key += 32) {
                    const uint8_t *src = raw + key * row_bytes;
                    uint8_t *dst = tiles + slot * S::kTile + key * 128;
                    // the lanes of a quarter warp start at different pieces: different banks
                    if (pieces == HDP / 16) {
                        constexpr int PIECES = HDP / 16;
                        const int first = key & (PIECES - 1);
                        uint4 raw16[PIECES];  // all loads first (16 integers each: 16 bytes, or 8 in the low half)
#pragma unroll
                        for (int i = 0; i < PIECES; i++) raw16[i] = load_sixteen<BITS>(src + (i ^ first) * 2 * BITS);
#pragma unroll
                        for (int i = 0; i < PIECES; i++) {
                            uint4 x, y;
                            sixteen<BITS>(raw16[i], x, y);
                            const int c = i ^ first, at = (c >> 2) * (kBN * 128) + ((((2 * c) & 7) ^ (key & 7)) << 4);
                            *reinterpret_cast<uint4 *>(dst + at) = x;
                            *reinterpret_cast<uint4 *>(dst + (at ^ 16)) = y;
                        }
                    } else {
                        int c = key % pieces;
                        for (int i = 0; i < pieces; i++) {
                            uint4 x, y;
                            sixteen<BITS>(load_sixteen<BITS>(src + c * 2 * BITS), x, y);
                            const int at = (c >> 2) * (kBN * 128) + ((((2 * c) & 7) ^ (key & 7)) << 4);
                            *reinterpret_cast<uint4 *>(dst + at) = x;
                            *reinterpret_cast<uint4 *>(dst + (at ^ 16)) = y;
                            c = c + 1 == pieces ? 0 : c + 1;
                        }
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) bar_arrive(&ready[slot]);
                if (!ALT && lane == 0) bar_arrive(&raw_empty[kv * kTurns + turn]);
                if (ALT && j + kRaw < mine) load(kv, j + kRaw, found);
            }
            // gave up: copies in flight land before the CTA can end
            for (int n = max(0, j - 2); ALT && j < mine && n < min(mine, j + kRaw); n++)
                bar_wait(&raw_full[kv * kTurns + n % kTurns], (n / kTurns) & 1);
        } else if (warp == kMmaWarp) {
            // ---------------- MMA issue ----------------
            if (mine > 0 && elect_one()) {
                constexpr uint32_t qk = idesc_f16(128, kBN, false), pv = idesc_f16(128, HDP, true);
                const uint32_t t = tmem;
                const uint64_t q0 = tile_desc(smem_addr(smem + S::kQ), 16), k0 = tile_desc(smem_addr(smem + S::kK), 16),
                               v0 = tile_desc(smem_addr(smem + S::kV), kBN * 128);  // start addresses count 16 bytes
                // the group's i-th step is step j of the CTA: the same for both groups, or every other one
                auto step_of = [&](int m, int i) { return ALT ? 2 * i + m : i; };
                bool ok = bar_wait(q_ready, 0);
                auto scores = [&](int m, int i) {  // S_m[i & 1] = Q K^T, every part of q; false: gave up
                    const int j = step_of(m, i), slot = j & 1;
                    if (j >= mine) return true;
                    if ((ALT || m == 0) && !bar_wait(&k_ready[slot], (j >> 1) & 1)) return false;
                    fence_after();
#pragma unroll
                    for (int part = 0; part < QP; part++)
#pragma unroll
                        for (int k = 0; k < HDP / 16; k++)
                            mma_ss(t + m * 128 + (i & 1) * 64,
                                   q0 + ((((ALT ? 0 : m) * QP + part) * S::kQTile + (k >> 2) * 16384 + (k & 3) * 32) >> 4),
                                   k0 + ((slot * S::kTile + (k >> 2) * (kBN * 128) + (k & 3) * 32) >> 4), qk,
                                   part > 0 || k > 0);
                    commit(&s_full[2 * m + (i & 1)]);
                    if (ALT || m == 1) commit(&k_free[j % kTurns]);
                    return true;
                };
#pragma unroll 1
                for (int i = 0; i < 2 && ok; i++) ok = scores(0, i) && scores(1, i);
#pragma unroll 1
                for (int i = 0; step_of(0, i) < mine && ok; i++) {
#pragma unroll
                    for (int m = 0; m < 2; m++) {
                        const int j = step_of(m, i), slot = j & 1;
                        if (!ok || j >= mine) break;
                        if ((ALT || m == 0) && !(ok = bar_wait(&v_ready[slot], (j >> 1) & 1))) break;
                        if (!(ok = bar_wait(&p_ready[2 * m + (i & 1)], (i >> 1) & 1))) break;
                        fence_after();
#pragma unroll
                        for (int part = 0; part < PP; part++)
#pragma unroll
                            for (int k = 0; k < kBN / 16; k++)
                                mma_ts(t + 256 + m * 128, t + m * 128 + (i & 1) * 64 + part * 32 + k * 8,
                                       v0 + ((slot * S::kTile + k * 2048) >> 4), pv,
                                       (SPANS ? i % kSpan : i) > 0 || part > 0 || k > 0);
                        commit(&pv_done[m]);
                        if (ALT || m == 1) commit(&v_free[j % kTurns]);
                        ok = scores(m, i + 2);
                    }
                }
                commit(o_done);
            }
        } else if (!ALT && warp == kLoadWarp) {
            // ---------------- raw pages: keys LEAD steps ahead of their values, as the scores are of the products ----------------
            // (a loader, since two row tiles leave the converters no time: 16 trees of 64 tokens 169 us, loaded by them 178)
            constexpr int LEAD = 2;
            auto refill = [&](int kv, int j, int found) {
                const int before = j - kRaw;  // the step that had the stage before
                if (before >= 0 && !bar_wait(&raw_empty[kv * kTurns + before % kTurns], (before / kTurns) & 1)) return false;
                load(kv, j, found);
                return true;
            };
            // this lane's entries of the page table, read two steps ahead of their use; found[k]: of the step k before j
            int next = entry(0), after = entry(1), found[LEAD + 1];
            for (int j = 0; j < mine + LEAD; j++) {
#pragma unroll
                for (int k = LEAD; k; k--) found[k] = found[k - 1];
                found[0] = next;
                next = after;
                after = entry(j + 2);
                if (j < mine && !refill(0, j, found[0])) break;
                if (j >= LEAD && !refill(1, j - LEAD, found[LEAD])) break;
            }
            // copies in flight land before the CTA can end
            for (int j = mine > kRaw ? mine - kRaw : 0; j < mine; j++)
                for (int kv = 0; kv < 2; kv++) bar_wait(&raw_full[kv * kTurns + j % kTurns], (j / kTurns) & 1);
        }
    } else {
        // ---------------- softmax: two threads a row ----------------
        // q: a warp takes a row, scales it by a power of two and stores its fp16 parts, swizzled
        constexpr int DEEP = 4;  // rows of a warp in flight
        for (int i0 = warp - 8; i0 < ROWS; i0 += 16 * DEEP) {
            float4 v[DEEP];
#pragma unroll
            for (int u = 0; u < DEEP; u++) {  // (no branch around the loads: all of them are in flight at once)
                const int R = min(R0 + i0 + 16 * u, nrows - 1), tok = R / p.group;
                v[u] = load4(static_cast<const T *>(p.q) + (size_t)(s.row0 + tok) * p.q_stride +
                             (size_t)(kvh * p.group + R - tok * p.group) * p.head + min(4 * lane, p.head - 4));
            }
#pragma unroll
            for (int u = 0; u < DEEP; u++)
                if (R0 + i0 + 16 * u >= nrows || 4 * lane >= p.head) v[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int u = 0; u < DEEP; u++) {
                const int i = i0 + 16 * u;
                int e = max(max(exponent_of(v[u].x), exponent_of(v[u].y)), max(exponent_of(v[u].z), exponent_of(v[u].w)));
#pragma unroll
                for (int o = 16; o; o >>= 1) e = max(e, __shfl_xor_sync(0xffffffffu, e, o));
                const int k = max(-100, min(e - 127 - 8, 119));
                if (lane == 0) row_factor[i] = pow2(k);
                const float f = pow2(-k);
                float x[4] = {v[u].x * f, v[u].y * f, v[u].z * f, v[u].w * f};
                if (4 * lane < HDP) {
                    const int r = i & 127;
                    uint8_t *d = smem + S::kQ + (i >> 7) * QP * S::kQTile + (lane >> 4) * 16384 + r * 128 +
                                 ((((lane & 15) >> 1) ^ (r & 7)) << 4) + (lane & 1) * 8;
                    *reinterpret_cast<uint2 *>(d) = make_uint2(pack2<__half>(x[0], x[1]), pack2<__half>(x[2], x[3]));
                    if (QP == 2) {
#pragma unroll
                        for (int j = 0; j < 4; j++) x[j] -= __half2float(__float2half_rn(x[j]));
                        *reinterpret_cast<uint2 *>(d + S::kQTile) =
                            make_uint2(pack2<__half>(x[0], x[1]), pack2<__half>(x[2], x[3]));
                    }
                }
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) bar_arrive(q_ready);
        asm volatile("bar.sync 10, 512;" ::: "memory");  // the row factors, among the softmax warps
        const int m = (warp - 8) >> 3, half = ((warp - 8) >> 2) & 1, row = tid & 127;
        const int pair = 2 + m * 4 + (warp & 3);  // the named barrier of a row's two warps
        float *mine_x = reinterpret_cast<float *>(smem + S::kXm) + (m * 2 + half) * 128 + row;
        const float *other_x = reinterpret_cast<const float *>(smem + S::kXm) + (m * 2 + 1 - half) * 128 + row;
        const uint32_t lane_at = tmem + ((uint32_t)(row & 96) << 16), o_at = lane_at + 256 + m * 128;
        const int R = R0 + (ALT ? 0 : m * 128) + row, draft = R / p.group;
        const float rf = row_factor[ALT ? row : m * 128 + row];
        float unit = INFINITY, l = 0.0f;
        // This thread's half of O in 16 columns: held from here on where that leaves the steps fewer spills (64 sequences of
        // 2,000 keys, 32 rows: bf16 88 us held, 91 not; fp16 102 and 99), else made anew.
        constexpr bool HELD = ALT && (QP == 2 || PP == 1);
        const int held = HELD ? half * (HDP / 32) : 0;
        float sums[SPANS && HDP == 128 ? HDP / 2 + 1 : 1];  // what spans before summed (or tensor memory), and its unit
        // One step; TAIL: some of its keys are new tokens, or none (a variant of its own: the mask's branches cost the
        // others more than their arithmetic).
        auto step = [&](int i, auto is_tail) -> bool {
            constexpr bool TAIL = decltype(is_tail)::value;
            const int j = ALT ? 2 * i + m : i, slot = i & 1, par = (i >> 1) & 1, ss = j % kScales, key0 = (t0 + j) * kBN;
            const uint32_t s_at = lane_at + m * 128 + slot * 64;
            const bool fine = bar_wait(&s_full[2 * m + slot], par) && bar_wait(&sc_ready[ss], (j / kScales) & 1);
            fence_after();
            const float *kk = reinterpret_cast<const float *>(smem + S::kScale) + ss * 2 * kBN + 32 * half, *vv = kk + kBN;
            float u[32];
            tmem_load32(s_at + 32 * half, u);
            const float limit = limits[ss];
            const uint32_t bits = TAIL ? mask32(p, s, draft, key0 + 32 * half - s.ctx) : ~0u;
            wait_load();
            float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
                const float4 k4 = *reinterpret_cast<const float4 *>(kk + i);
                split2(mul2(pair2(u[i], u[i + 1]), pair2(k4.x, k4.y)), u[i], u[i + 1]);
                split2(mul2(pair2(u[i + 2], u[i + 3]), pair2(k4.z, k4.w)), u[i + 2], u[i + 3]);
                if (TAIL) {
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (!((bits >> (i + e)) & 1)) u[i + e] = -INFINITY;
                }
                top[0] = max3(top[0], u[i], u[i + 1]);
                top[1] = max3(top[1], u[i + 2], u[i + 3]);
            }
            float now = fmaxf(top[0], top[1]) * rf;
            uint32_t vote;  // of both warps; after it both have read their S
            asm volatile(
                "{\n\t.reg .pred a, b;\n\tsetp.ne.u32 a, %1, 0;\n\t"
                "barrier.cta.red.or.pred b, %2, 64, a;\n\tselp.u32 %0, 1, 0, b;\n\t}"
                : "=r"(vote)
                : "r"((uint32_t)(now + unit > limit || !fine)), "r"(pair)
                : "memory");
            if (vote) {
                auto larger = [&](float x) {  // of both threads of the row
                    *mine_x = x;
                    asm volatile("bar.sync %0, 64;" ::"r"(pair) : "memory");
                    const float theirs = *other_x;
                    asm volatile("bar.sync %0, 64;" ::"r"(pair) : "memory");
                    return x != x || theirs != theirs ? __int_as_float(0x7FC00000) : fmaxf(x, theirs);
                };
                // a wait that ran out on either side ends both (NaN stands for it; scores that are all NaN count as none)
                now = larger(!fine ? __int_as_float(0x7FC00000) : now == now ? now : -INFINITY);
                if (__any_sync(0xffffffffu, now != now)) return false;
                float w = 0.0f;  // (by exponentials: with a logarithm of each scale 128 rows of fp16 took 5 % longer)
#pragma unroll
                for (int i = 0; i < 32; i++) w = fmaxf(w, product_of(u[i], rf, now, vv[i]));
                // Only the rows that are behind move, so that a row's result does not depend on its neighbours.
                const float to = moved<PP>(unit, now, now + __log2f(larger(w))), f = unit_factor(unit, to);
                unit = to;
                l *= f;
                if (i > 0 && __any_sync(0xffffffffu, f != 1.0f)) {
                    // (the product of two steps ago has ended: this step's scores were issued after it; where this wait
                    // runs out, the results are void and the error is noted)
                    bar_wait(&pv_done[m], (i - 1) & 1);
                    fence_after();
#pragma unroll 1
                    for (int c = HELD ? held : half * (HDP / 32), end = c + HDP / 32; c < end; c++) {
                        float o[16];
                        tmem_load16(o_at + 16 * c, o);
                        wait_load();
#pragma unroll
                        for (int e = 0; e < 16; e++) o[e] *= f;
                        tmem_store16(o_at + 16 * c, reinterpret_cast<const uint32_t *>(o));
                    }
                }
            }
            const uint64_t rf2 = pair2(rf, rf), base2 = pair2(or_zero(unit), or_zero(unit));
            uint64_t sum[2] = {0, 0};
            uint32_t hi[16], low[PP == 2 ? 16 : 1];
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
                const float4 w4 = *reinterpret_cast<const float4 *>(vv + i);
                const uint64_t w2[2] = {pair2(w4.x, w4.y), pair2(w4.z, w4.w)};
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int at = i + 2 * h;
                    float a, d;
                    split2(fma2(pair2(u[at], u[at + 1]), rf2, base2), a, d);
                    const uint64_t e2 = pair2(exp2_fast(a), exp2_fast(d));
                    sum[h] = add2(sum[h], e2);
                    float x, y;
                    split2(mul2(e2, w2[h]), x, y);
                    if (TAIL) {  // a masked key's scale may be anything: its weight is zero, not zero times that
                        if (u[at] == -INFINITY) x = 0.0f;
                        if (u[at + 1] == -INFINITY) y = 0.0f;
                    }
                    const uint32_t q = pack2<__half>(x, y);
                    hi[at / 2] = q;
                    if (PP == 2) {
                        const float2 r = __half22float2(*reinterpret_cast<const __half2 *>(&q));
                        low[PP == 2 ? at / 2 : 0] = pack2<__half>(x - r.x, y - r.y);
                    }
                }
            }
            tmem_store16(s_at + 16 * half, hi);
            if (PP == 2) tmem_store16(s_at + 32 + 16 * half, low);
            float a, d, a2, d2;
            split2(sum[0], a, d);
            split2(sum[1], a2, d2);
            l += (a + d) + (a2 + d2);
            wait_store();
            if constexpr (SPANS) {
                if (i > 0 && i % kSpan == 0)
                    keep<HDP>(sums, o_at + (HELD ? 16 * held : half * (HDP / 2)), unit, i == kSpan, &pv_done[m], (i - 1) & 1);
            }
            fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(&p_ready[2 * m + slot]);
            return true;
        };
        // this group's steps, those wholly below the context first
        auto share = [&](int n) { return ALT ? max(0, n - m + 1) / 2 : max(0, n); };
        const int steps = share(mine), plain = share(min(mine, s.ctx / kBN - t0));
        bool ok = true;
        // A warp whose 32 rows all lie behind the last only keeps the barriers' count: what the product makes of its rows
        // is not read.
        const bool idle = R - lane >= nrows;
#pragma unroll 1
        for (int i = 0; idle && i < steps && ok; i++) {
            ok = bar_wait(&s_full[2 * m + (i & 1)], (i >> 1) & 1);
            if (ok && lane == 0) bar_arrive(&p_ready[2 * m + (i & 1)]);
        }
        ok = ok && !idle;
#pragma unroll 1
        for (int i = 0; i < plain && ok; i++) ok = step(i, std::false_type{});
#pragma unroll 1
        for (int i = plain; i < steps && ok; i++) ok = step(i, std::true_type{});
        if (mine > 0) bar_wait(o_done, 0);
        fence_after();
        // the row's sum of both threads
        *mine_x = l;
        asm volatile("bar.sync %0, 64;" ::"r"(pair) : "memory");
        l = half ? *other_x + l : l + *other_x;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // both in the row's unit
        const int c0 = half * (HDP / 32);
        auto load_o = [&](int c, float *o) {  // 16 columns of O, with what was summed before
            tmem_load16(o_at + 16 * c, o);
            wait_load();
            if constexpr (SPANS) {
                if (steps <= kSpan) return;
                const float f = unit_factor(sums[HDP == 128 ? HDP / 2 : 0], unit);
                float had[16];
                if constexpr (HDP == 64) {
                    tmem_load16(o_at + HDP + 16 * c, had);
                    wait_load();
                }
#pragma unroll
                for (int e = 0; e < 16; e++)
                    o[e] = __fmaf_rn(HDP == 64 ? had[e] : sums[HDP == 64 ? 0 : 16 * (c - c0) + e], f, o[e]);
            }
        };
        if (!ALT && p.splits * p.supers == 1) {
            const int tok = s.row0 + R / p.group, head = kvh * p.group + R % p.group;
            if (R < nrows && p.lse && half == 0)
                p.lse[(size_t)tok * p.heads + head] =
                    l == 0.0f ? -INFINITY : (log2f(l) - unit) * 0.693147180559945309f;
#pragma unroll 1
            for (int c = c0; c < c0 + HDP / 32; c++) {
                float o[16];
                if (mine > 0) load_o(c, o);
                if (R >= nrows) continue;
                T *d = static_cast<T *>(p.out) + (size_t)tok * p.out_stride + (size_t)head * p.head + 16 * c;
#pragma unroll
                for (int i = 0; i < 16; i += 4)
                    if (16 * c + i < p.head)
                        store4(d + i, l == 0.0f ? make_float4(0.0f, 0.0f, 0.0f, 0.0f)
                                                : make_float4(o[i] * inv, o[i + 1] * inv, o[i + 2] * inv, o[i + 3] * inv));
            }
        } else {
            // this group's part: O divided by its own sum, the row's (max, sum) beside it
            if (half == 0) {
                const float2 ml = normal_sum(unit, l);
                cta_m[m * 128 + row] = ml.x;
                cta_l[m * 128 + row] = ml.y;
            }
            float *po = reinterpret_cast<float *>(smem) + (size_t)(m * 128 + row) * HDP;
#pragma unroll 1
            for (int c = c0; c < c0 + HDP / 32; c++) {
                float o[16];
                if (steps > 0) load_o(c, o);
                // the 16-byte pieces of a row start at different places: different banks
#pragma unroll
                for (int i = 0; i < 16; i += 4)
                    *reinterpret_cast<float4 *>(po + ((16 * c + i) ^ ((row & 7) << 2))) =
                        steps <= 0 || l == 0.0f ? make_float4(0.0f, 0.0f, 0.0f, 0.0f)
                                                : make_float4(o[i] * inv, o[i + 1] * inv, o[i + 2] * inv, o[i + 3] * inv);
            }
        }
    }
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    if (!ALT && p.splits * p.supers == 1) return;

    // join the cluster: weights of every CTA's rows first, then each CTA takes its share of the elements
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    float *weight = reinterpret_cast<float *>(smem + S::kAll), *total = weight + kMaxSplits * PARTS * ROWS;
    float *part_m = reinterpret_cast<float *>(smem + S::kPm);
    const int rows_here = min(ROWS, nrows - R0), parts = p.splits * PARTS;  // part n: CTA n / PARTS, group n % PARTS
#pragma unroll 4
    for (int i = tid; i < parts * ROWS; i += kTcThreads) {
        const int n = i / ROWS, at = (n % PARTS) * 128 + i % ROWS;
        part_m[i] = *cluster.map_shared_rank(&cta_m[at], n / PARTS);
        weight[i] = *cluster.map_shared_rank(&cta_l[at], n / PARTS);
    }
    __syncthreads();
    for (int i = tid; i < rows_here; i += kTcThreads) {
        float m = -INFINITY, sum = 0.0f;
        for (int n = 0; n < parts; n++) m = fmaxf(m, part_m[n * ROWS + i]);
        for (int n = 0; n < parts; n++) {
            const float l = weight[n * ROWS + i], w = l == 0.0f ? 0.0f : l * exp2_fast(part_m[n * ROWS + i] - m);
            weight[n * ROWS + i] = w;
            sum += w;
        }
        total[i] = sum;
        if (split == 0) {
            const int R = R0 + i;
            const size_t at = (size_t)(s.row0 + R / p.group) * p.heads + kvh * p.group + R % p.group;
            if (p.supers > 1) work_ml(p)[(size_t)super * p.rows * p.heads + at] = make_float2(m, sum);
            else if (p.lse) p.lse[at] = sum == 0.0f ? -INFINITY : (m + log2f(sum)) * 0.693147180559945309f;
        }
    }
    __syncthreads();
    const int total4 = rows_here * (HDP / 4);
    for (int i = tid + split * kTcThreads; i < total4; i += kTcThreads * p.splits) {
        const int row = i / (HDP / 4), d4 = i % (HDP / 4);
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
        for (int n = 0; n < parts; n++) {
            const float4 x = *reinterpret_cast<const float4 *>(cluster.map_shared_rank(
                reinterpret_cast<const float *>(smem) + (size_t)((n % PARTS) * 128 + row) * HDP + ((4 * d4) ^ ((row & 7) << 2)),
                n / PARTS));
            const float f = weight[n * ROWS + row];
            o.x = __fmaf_rn(f, x.x, o.x);
            o.y = __fmaf_rn(f, x.y, o.y);
            o.z = __fmaf_rn(f, x.z, o.z);
            o.w = __fmaf_rn(f, x.w, o.w);
        }
        if (4 * d4 >= p.head) continue;
        const float sum = total[row], inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        const int R = R0 + row, tok = s.row0 + R / p.group, head = kvh * p.group + R % p.group;
        o = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
        if (p.supers > 1)
            *reinterpret_cast<float4 *>(p.work + (((size_t)super * p.rows + tok) * p.heads + head) * p.head + 4 * d4) = o;
        else
            store4(static_cast<T *>(p.out) + (size_t)tok * p.out_stride + (size_t)head * p.head + 4 * d4, o);
    }
    cluster.sync();  // no CTA leaves while a sister reads its shared memory
}

static int slots(const void *kernel, int n, size_t smem) { return cluster_slots(kernel, n, kTcThreads, smem); }

template <typename T, int QP, int PP, int BITS, int HDP, int MT>
static cudaError_t launch(AttnParams p, int max_len, cudaStream_t stream) {
    using S = TcSmem<QP, BITS, HDP, MT>;
    // more than half of an SM's shared memory, so that no second CTA waits for tensor memory
    constexpr size_t smem = S::kBytes > 116 * 1024 ? S::kBytes : 116 * 1024;
    auto kernel = tree_attention_tc_kernel<T, QP, PP, BITS, HDP, MT>;
    if (!tiles_fit(p, MT * 128)) return kTooManyRows;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    const long long base = (long long)p.qtiles * p.kv_heads * p.bt.batch;
    // a unit: a step, 1.2 us with two row tiles; a CTA starts, fills and joins in about 8 us, a second kernel takes 4
    const Split cut = choose_splits(base, p.bt.batch, (double)max_len / kBN, 6.0, 8.0, 0.0, 3.0, 4.0, most_supers(p),
                                    [&](int n) { return slots((const void *)kernel, n, smem); });
    p.splits = cut.splits;
    p.supers = cut.supers;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.splits * p.supers, p.kv_heads * p.qtiles, p.bt.batch);
    cfg.blockDim = dim3(kTcThreads);
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

template <typename T, int QP, int PP, int BITS, int HDP>
static cudaError_t launch_tiles(const AttnParams &p, int max_len, cudaStream_t s) {
    // two parts of q for two row tiles of 128-element heads do not fit in shared memory
    if constexpr (QP == 1 || HDP == 64) {
        if ((long long)p.max_new * p.group > 128) return launch<T, QP, PP, BITS, HDP, 2>(p, max_len, s);
    }
    return launch<T, QP, PP, BITS, HDP, 1>(p, max_len, s);
}

template <int BITS, int HDP>
static cudaError_t launch_type(const AttnParams &p, int dtype, int max_len, cudaStream_t s) {
    if (dtype == kF32) return launch_tiles<float, 2, 2, BITS, HDP>(p, max_len, s);
    if (dtype == kBF16) return launch_tiles<__nv_bfloat16, 1, 1, BITS, HDP>(p, max_len, s);
    return launch_tiles<__half, 1, 2, BITS, HDP>(p, max_len, s);
}

cudaError_t launch_tc(const AttnParams &p, int dtype, int bits, int max_len, cudaStream_t s) {
    if (bits == 8) return p.head <= 64 ? launch_type<8, 64>(p, dtype, max_len, s) : launch_type<8, 128>(p, dtype, max_len, s);
    return p.head <= 64 ? launch_type<4, 64>(p, dtype, max_len, s) : launch_type<4, 128>(p, dtype, max_len, s);
}

int *tc_error_word() {
    void *p = nullptr;
    return cudaGetSymbolAddress(&p, g_tc_error) == cudaSuccess ? static_cast<int *>(p) : nullptr;
}

}  // namespace attn
}  // namespace mvb
