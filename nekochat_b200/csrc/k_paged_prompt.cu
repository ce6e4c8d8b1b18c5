// Attention of many query rows over a paged cache (neko_op_paged_attention): prompts and long continuations, on
// tcgen05.
//
// A prompt of 8,192 bf16 tokens, 16 heads on 8: 320 to 337 us, 816 to 860 TFLOP/s of the causal half's products (50 % of the measured
// rate); 350 us and more in a second of such calls, under the power cap.
// Per pair of row tiles and 128 keys about 4,080 cycles against 2,048 of the UMMAs: each row tile's chain is S, softmax (2,010
// cycles: TMEM reads 330, maximum and meeting 500, exponentials 1,110), P V and S again (1,190), and the two tiles take
// turns. f32 rows take twice the UMMAs (5,900 cycles).
//
// The packed rows of a (sequence, KV head) are its new tokens times the G query heads that share the KV head. A CTA
// takes two tiles of 128 rows (one when there are no more) and walks the keys in tiles of 128:
//   S = Q K^T in TMEM, weights P back into TMEM over S (f16), O += P V in TMEM, all accumulation f32.
// f32 queries are f16 hi + lo in shared memory (S = Qhi K^T + Qlo K^T) and their weights hi + lo in TMEM (P takes
// exactly the 128 columns of its S); 16-bit queries are one f16 and their weights one f16. Rows are scaled by a
// power of two into f16's range first (exact, but for bf16 values below 2^-17 of their row's largest, which lose bits). Roles:
//  * warps 0..7 and 8..15: softmax of one row tile each, two threads per row (64 keys each; two warps more per scheduler
//    hide each other's latencies), which tell each other their largest scores. The reference maximum moves only
//    when a score exceeds it by a factor of 2^8 (weights above 1 are as exact as any in f16), so O is hardly ever rescaled, and
//    the row's own threads do that; the tensor core works on the other row tile meanwhile. A quarter of 16-bit queries'
//    exponentials is computed on the FMA pipe: the special-function unit is what bounds this step.
//  * warps 16..18: the loader. K and V tiles go to a ring of shared-memory stages in the 128-byte-swizzled layout that
//    serves K as a K-major and V as an MN-major operand: tensor copies for f16 pages, registers and an exact conversion to
//    f16 for 8-bit ones (fetched one tile ahead). Scales stay out of the operands: a block's key scale multiplies its
//    scores and its value scale enters the weights' exponent (the sum takes it out again), 16 columns at a time. A row's
//    reference is then the largest score plus log2 of the value scale that it sees: what is rounded off a weight is small beside
//    what the largest of its products adds, not beside the largest scale.
//  * warp 19, an elected lane: issues the UMMAs; PV of one tile and S of its next key tile go back to back.
// Masks only touch the key tiles that need them. Values that no row sees are zeroed by the loader; values that are not
// finite in a tile that some row does not see whole are zeroed too and added by the threads of the rows that see them.
// A cluster of CTAs splits the keys when there are few row tiles and joins over distributed shared memory in rank
// order. Every wait is bounded and gives up once another role has failed.
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>

#include "paged.cuh"
#include "paged_math.cuh"
#include "tc5_core.cuh"
#include "tma_host.h"

namespace cg = cooperative_groups;

namespace neko {

namespace {

constexpr int kRows = 128, kKeys = 128;  // of a tile
constexpr int kSoftWarps = 16, kLoadWarp = 16, kMmaWarp = 19, kThreads = 20 * 32;  // 96 registers a thread
constexpr int kLoaders = 96;
constexpr int kCopyTiles = 2;
constexpr int64_t kCopyBytes = int64_t(1) << 31;
constexpr int kRing = 4;        // key tiles whose scales are kept (at most 5 stages are in flight)
constexpr int kOddRing = 8;     // and their keys with odd values
// Weights are 2^(score (+ log2 of the value scale) - reference + kLift), at most 2^15. What f16 rounds off them, half of 2^-24 with
// hi + lo, is 2^-32 of the largest: little lag of the reference keeps small weights, much saves trips of O through registers (f32
// ragged prompts at a lag of 2^8 678 us, 2^7 693, 2^6 718, 2^4 806).
constexpr float kLazy = 8.0f;   // log2 of how far a score may exceed the reference
constexpr float kLift = 15.0f - kLazy;
// An UMMA's f32 accumulation truncates: each step takes a share off the sum, 3.2e-8 on average (measured on sums of 2,500
// steps, whose common factor was 1 - 2.1e-5; half a unit in the last of 24 places is 4.3e-8 of a mantissa spread evenly over
// the logarithm). What O held before a step loses as a whole, so the sum of the weights, which is rounded to nearest, is made
// to lose as much and the quotient does not keep it - but no more than a key tile adds, since a step that adds nothing truncates
// nothing (one key with all the weight, 262,144 keys: 5e-4 too large otherwise). What is left differs from value to value, about 6e-9 a step: for f32
// queries O leaves TMEM every kFlush key tiles for sums that are rounded to nearest (20,000 keys: an error of 1.3e-6 every 8
// tiles, 2.4e-6 every 16; ragged prompts on 3,000 keys: 669 and 646 us).
constexpr float kDrop = 3.2e-8f;
constexpr int kFlush = 8;
constexpr float kVMin = -60.0f; // the product of a row's likeliest key with a block's scale counts as no less than 2^-60 of the reference
constexpr float kVNone = -126.0f;
constexpr float kGone = -1.0f;

// What the key and value tiles come from: f16 pages, 8-bit pages converted by the loader, or f16 copies of 8-bit pages.
enum Source : int { kF16Pages = 0, kCodes = 1, kCopies = 2 };

struct PromptPlan {
    int ranks;      // CTAs that share a (sequence, KV head, row tile pair): the cluster
    int row_tiles;  // pairs of row tiles per (sequence, KV head)
    int tiles_per;  // row tiles of a CTA: 1 or 2
    int group;      // query heads per KV head
    uint64_t group_inv;  // ceil(2^32 / group): x / group = x * group_inv >> 32 for x below 2^32 / group
    float* flush;        // [slot][HD][256 rows]: sums that have left TMEM (f32 queries; NULL: none do)
    uint32_t* taken;     // [slot]: 1 while a CTA has it (NULL: every CTA has one of its own)
    int slots;           // as many as CTAs run at once, or as there are
};

template <int HD, bool HILO>
struct PL {
    static constexpr int kParts = HILO ? 2 : 1;
    static constexpr int kHalf = kRows * 128;             // bytes of a 128-row, 64-wide f16 tile
    static constexpr int kQTile = kHalf * (HD / 64);      // one part of one row tile
    static constexpr int kStage = kHalf * (HD / 64);
    static constexpr int kQBytes = 2 * kParts * kQTile;
    static constexpr int kStages = HD == 64 ? 5 : HILO ? 3 : 5;
    static constexpr int kStageOff = kQBytes;
    static constexpr int kMiscOff = kStageOff + kStages * kStage;
    static constexpr int kJoinPitch = HD + 4;             // floats of a row's state: values, their unit, sum, its unit
    static constexpr int kSmem = kMiscOff + 3072 - 128;
    static_assert(kSmem <= 227 * 1024, "shared memory");
    static_assert(2 * kRows * kJoinPitch * 4 <= kMiscOff, "the joined states take the operands' place");
    static_assert(kStages <= 5, "the ring of scales");
};

// barriers and small arrays behind the operands
struct Misc {
    uint64_t full[5], empty[5], s_full[2], p_full[2], pv_done[2], drain, land, scanned, q_full;
    uint32_t tmem, fail;
    int slot;                          // of plan.flush; -1: none
    float ks[kRing][8];                // scales of a key tile's blocks of 16 keys; kGone: not resident
    float vs[kRing][8];                // log2 of theirs of the values
    uint32_t whole[kRing];             // every block is resident
    uint32_t odd[kOddRing][4];         // of a key tile that needs masks: keys with values that are not finite
    float most[2][2 * kRows];          // by half of the key tile: the rows' largest scores (with value scales), at the end their
                                       // largest scores without and their sums; before the first tile most[0] is scale / the
                                       // row's power of two
};
static_assert(sizeof(Misc) <= 3072 - 128, "misc");

__device__ __forceinline__ uint64_t v_desc(uint32_t addr) {
    // MN-major, 128-byte swizzle: 64-value blocks 16 KB apart (LBO), groups of 8 keys 1024 bytes apart (SBO)
    return uint64_t((addr >> 4) & 0x3FFF) | (uint64_t(16384 >> 4) << 16) | (uint64_t(1024 >> 4) << 32) |
           (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, 1, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc)
        : "memory");
}
#define NEKO_R32(r)                                                                                                  \
    "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),      \
        "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),       \
        "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),      \
        "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
#define NEKO_REGS32                                                                                                  \
    "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,"  \
    "%29,%30,%31}"
// 32 columns of this thread's TMEM lane; the values are there after ld_wait on the same registers.
__device__ __forceinline__ void ld32(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 " NEKO_REGS32 ", [%32];" : NEKO_R32(r) : "r"(addr));
}
__device__ __forceinline__ void ld_wait(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : NEKO_R32(r)::"memory");
}
__device__ __forceinline__ void st32(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], " NEKO_REGS32 ";" : NEKO_R32(r) : "r"(addr) : "memory");
}
__device__ __forceinline__ void st16(uint32_t addr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void st8(uint32_t addr, const uint32_t* v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), "r"(v[0]), "r"(v[1]),
                 "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}
#define NEKO_R16(r)                                                                                                  \
    "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),      \
        "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
__device__ __forceinline__ void ld16(uint32_t addr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : NEKO_R16(r)
                 : "r"(addr));
}
__device__ __forceinline__ void ld_wait16(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : NEKO_R16(r)::"memory");
}
__device__ __forceinline__ void st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ float max_nan(float x, float y) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
    return r;
}
// 2^x of two numbers (at least 2^-126) off the special-function unit, which is what bounds the softmax: the integer part
// by adding 1.5 * 2^23, a polynomial of degree 4 for the rest (least maximum relative error on [-1/2, 1/2]: 2.6e-6,
// against 2.4e-4 of the f16 that the weight is rounded to).
__device__ __forceinline__ void exp2_poly(float& x, float& y) {
    const uint64_t magic = pack2(12582912.0f, 12582912.0f), less = pack2(-12582912.0f, -12582912.0f), neg = pack2(-1.0f, -1.0f);
    const uint64_t z = pack2(fmaxf(x, -126.0f), fmaxf(y, -126.0f));
    const uint64_t r = add2(z, magic), f = fma2(add2(r, less), neg, z);
    uint64_t p = pack2(0.009570086374878883f, 0.009570086374878883f);
    p = fma2(p, f, pack2(0.055917900055646896f, 0.055917900055646896f));
    p = fma2(p, f, pack2(0.2402474582195282f, 0.2402474582195282f));
    p = fma2(p, f, pack2(0.6931217908859253f, 0.6931217908859253f));
    p = fma2(p, f, pack2(0.9999992847442627f, 0.9999992847442627f));
    float r0, r1, p0, p1;
    unpack2(r, r0, r1), unpack2(p, p0, p1);
    x = __int_as_float(__float_as_int(p0) + (__float_as_int(r0) << 23));
    y = __int_as_float(__float_as_int(p1) + (__float_as_int(r1) << 23));
}
// Bounded wait that also ends once another role has failed; false: give up.
__device__ __forceinline__ bool wait_on(uint64_t* bar, uint32_t parity, volatile uint32_t* fail) {
    for (uint32_t i = 0; i < kMbarMaxTries; i++) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 7) == 7 && *fail) return false;
    }
    *fail = 1;
    set_op_error(kErrMbarTimeout);
    return false;
}
// Bounded wait for what is in flight once a role has given up.
__device__ __forceinline__ void wait_out(uint64_t* bar, uint32_t parity) {
    for (uint32_t i = 0; i < kMbarMaxTries; i++)
        if (mbar_try_wait(bar, parity)) return;
    set_op_error(kErrMbarTimeout);
}
// Whether the four 16-byte words hold f16 values that are not finite; those are zeroed.
__device__ __forceinline__ bool drop_odd(uint4& x) {
    bool odd = false;
    uint32_t* w = reinterpret_cast<uint32_t*>(&x);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if ((w[i] & 0x7c00u) == 0x7c00u) w[i] &= 0xffff0000u, odd = true;
        if ((w[i] & 0x7c000000u) == 0x7c000000u) w[i] &= 0xffffu, odd = true;
    }
    return odd;
}

// The pools as [pages][kv heads * page][hd] f16, read in boxes of a page's tokens x 64 values (f16 pages only).
struct PromptMaps {
    CUtensorMap k, v;
};
__device__ __forceinline__ void copy_box(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
        "[%5];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}

template <int HD, int SRC, bool HILO>
__global__ void __launch_bounds__(kThreads, 1) paged_prompt_kernel(const neko_paged_attention_args a,
                                                                  const PromptPlan plan,
                                                                  const __grid_constant__ PromptMaps maps) {
    constexpr bool kScaled = SRC != kF16Pages, kConvert = SRC == kCodes;
    using L = PL<HD, HILO>;
    extern __shared__ __align__(1024) uint8_t sm[];
    if (smem_u32(sm) & 1023u) {  // the operands' swizzle goes by address bits
        if (threadIdx.x == 0) set_op_error(kErrMisalignedSmem);
        return;
    }
    Misc& ms = *reinterpret_cast<Misc*>(sm + L::kMiscOff);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const neko_paged_cache& c = a.cache;

    // ---- the work of this CTA, the same for its whole cluster but for the rank
    int b = blockIdx.x;
    const int rank = b % plan.ranks;
    b /= plan.ranks;
    const int kvh = b % c.n_kv;
    b /= c.n_kv;
    const int s = b % c.n_seq;
    const int tile = plan.row_tiles - 1 - b / c.n_seq;  // the longest rows first
    const int G = plan.group;
    auto over_g = [&](int x) { return int(uint64_t(uint32_t(x)) * plan.group_inv >> 32); };
    const int row0 = a.q_start ? a.q_start[s] : s;
    const int n = a.q_start ? a.q_start[s + 1] - row0 : 1;
    const int held = max(a.kv_len[s], 0);
    const int len = min(held, c.max_pages * c.page_size);
    if (row0 < 0 || n < 0 || n > a.max_new || row0 + n > a.tokens) {
        if (tid == 0) set_op_error(kErrBadIndex);
        return;
    }
    const int r0 = tile * plan.tiles_per * kRows;
    const int rows = min(n * G - r0, plan.tiles_per * kRows);
    if (rows <= 0) return;
    const int mt = rows > kRows ? 2 : 1;
    const int pos_lo = held - n + over_g(r0), pos_hi = held - n + over_g(r0 + rows - 1);
    const int prefix = a.prefix ? min(max(a.prefix[s], 0), len) : 0;
    const int hi = max(min(len, pos_hi + 1), 0);
    const int lo = a.window && pos_lo >= a.window ? min(pos_lo - a.window + 1, hi) : 0;
    const int t_lo = lo / kKeys, t_hi = (max(hi, prefix > lo ? prefix : 0) + kKeys - 1) / kKeys;
    const int t_pre = min((prefix + kKeys - 1) / kKeys, t_lo);
    const int nt_all = t_pre + max(t_hi - t_lo, 0);
    const int i_begin = int(int64_t(nt_all) * rank / plan.ranks), i_end = int(int64_t(nt_all) * (rank + 1) / plan.ranks);
    const int nt = i_end - i_begin;
    auto key_of = [&](int i) { i += i_begin; return kKeys * (i < t_pre ? i : i - t_pre + t_lo); };
    // every key of the tile is seen by every row between two positions
    auto open = [&](int j0, int p_lo, int p_hi) {
        return j0 + kKeys <= len && ((j0 + kKeys - 1 <= p_lo && (!a.window || p_hi - j0 < a.window)) || j0 + kKeys <= prefix);
    };

    if (tid == 0) {
        for (int i = 0; i < L::kStages; i++) mbar_init(&ms.full[i], kConvert ? kLoaders : 1), mbar_init(&ms.empty[i], 1);
        for (int h = 0; h < 2; h++) mbar_init(&ms.s_full[h], 1), mbar_init(&ms.p_full[h], 256), mbar_init(&ms.pv_done[h], 1);
        mbar_init(&ms.drain, 1), mbar_init(&ms.land, 1), mbar_init(&ms.scanned, kLoaders), mbar_init(&ms.q_full, 32 * kSoftWarps);
        ms.fail = 0;
        for (int i = 0; i < 8; i++) ms.odd[i / 4][i % 4] = 0;  // tiles 0 and 1
        fence_barrier_init();
    }
    if constexpr (HILO) {
        // A slot for this CTA: its own number's in a grid of no more CTAs than slots, else one that is free. There is one for every
        // CTA that runs (the search is bounded all the same), and it begins at the SM's number, where the SM's CTA before this
        // one had its slot: from the block's number on it took 90 us of 770 in all, and with fewer slots than SMs 50 of 165.
        if (tid == 32 * kLoadWarp) {
            int slot = -1;
            if (plan.flush && nt > kFlush) {
                unsigned sm_id;
                asm volatile("mov.u32 %0, %%smid;" : "=r"(sm_id));
                if (!plan.taken) slot = int(blockIdx.x);
                for (int x = 0; x < 2 * plan.slots && slot < 0; x++) {
                    const int y = int((sm_id + unsigned(x)) % unsigned(plan.slots));
                    if (atomicCAS(&plan.taken[y], 0u, 1u) == 0u) slot = y;
                }
            }
            ms.slot = slot;
        }
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ms.tmem)), "r"(512u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ms.tmem;
    volatile uint32_t* fail = &ms.fail;

    // Of a softmax thread's row: log2 of O's unit (the reference), and the sum of the weights with log2 of its unit. Without
    // value scales the two are one; with them the sum's is the largest score of this thread's half of the keys.
    float row_max = -INFINITY, row_sum = 0.0f, sum_max = -INFINITY;
    // f32 queries: this thread's first kept sum (256 floats between columns), and log2 of their unit, which only grows
    float* kept = nullptr;
    float kept_ref = 0.0f, sum_kept = 0.0f;  // and the weights' sum that goes with them
    if (warp >= kLoadWarp && warp < kMmaWarp) {
        // ------------------------------------------------------------------ loader
        const int lt = tid - 32 * kLoadWarp;
        const int32_t* table = c.table + int64_t(s) * c.table_stride;
        const int ps_log = 31 - __clz(c.page_size);
        const int total = 2 * nt;  // items K0 V0 K1 V1 ..
        // lane x < 8: page of the 16 keys from j0 + 16 x, -1: none
        auto pages_of = [&](int j0) {
            const int j = j0 + 16 * lane, slot = j >> ps_log;
            const int p = lane < 8 && j < len && slot < c.max_pages ? table[slot] : -1;
            return p < c.num_pages ? p : -1;
        };
        int pages = nt > 0 ? pages_of(key_of(0)) : -1, pages_next = -1;
        bool ok = true;
        if constexpr (kConvert) {
            constexpr int kRowChunks = HD / 16;             // 16-byte pieces of a key row
            constexpr int kRowsAt = kLoaders / kRowChunks;  // key rows of one round of pieces: 12 or 24
            constexpr int kPer = (kKeys + kRowsAt - 1) / kRowsAt;
            const int piece = lt % kRowChunks, row_in = lt / kRowChunks;
            const int64_t inner = int64_t(kvh) * c.page_size * HD + piece * 16;
            uint4 got[kPer];
            auto fetch = [&](const void* pool, int j0) {
                const uint8_t* base = static_cast<const uint8_t*>(pool) + inner;
                const int64_t at = pages >= 0 ? int64_t(pages) * c.page_stride : -1;
                const int at_lo = int(uint32_t(at)), at_hi = int(at >> 32);
#pragma unroll
                for (int y = 0; y < kPer; y++) {
                    const int r = row_in + y * kRowsAt;
                    const uint32_t o_lo = __shfl_sync(0xffffffffu, at_lo, r >> 4);  // rows past 128: lane 8, no page
                    const int o_hi = __shfl_sync(0xffffffffu, at_hi, r >> 4);
                    const uint8_t* p = base + (int64_t(o_hi) << 32 | o_lo) + (r & (c.page_size - 1)) * HD;
                    got[y] = o_hi >= 0 && r < len - j0 ? ldg_stream(p) : make_uint4(0, 0, 0, 0);
                }
            };
            // Pieces of the second 64 values write their 16-byte halves in the other order: eight lanes, eight bank groups.
            const bool second = piece >= 4;
            const uint32_t place = second ? L::kHalf : 0;
            const int ch0 = piece * 2 % 8 + second, ch1 = piece * 2 % 8 + !second;
            float ks = 0.0f, vs = 0.0f;  // lt < 8: the scales of this thread's block of the tile
            auto scales = [&]() {
                if (lt < 8 && pages >= 0) {
                    ks = c.k_scale[int64_t(pages) * c.scale_stride + kvh];
                    vs = c.v_scale[int64_t(pages) * c.scale_stride + kvh];
                }
            };
            if (nt > 0) {
                scales();
                fetch(c.k_pages, key_of(0));
            }
            for (int x = 0; x < total; x++) {
                const int st = x % L::kStages, i = x >> 1;
                const bool v = x & 1;
                if (x >= L::kStages) {
                    ok = wait_on(&ms.empty[st], ((x / L::kStages) & 1) ^ 1, fail);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                }
                uint8_t* base = sm + L::kStageOff + st * L::kStage + place;
                if (!v) {
                    if (warp == kLoadWarp) {
                        const float vl = lane < 8 && pages >= 0 ? fmaxf(log2f(vs), kVNone) : kVNone;
                        const bool whole = __all_sync(0xffffffffu, lane >= 8 || pages >= 0);
                        if (lane < 8) ms.ks[i % kRing][lane] = pages >= 0 ? fabsf(ks) : kGone, ms.vs[i % kRing][lane] = vl;
                        if (lane == 0) ms.whole[i % kRing] = whole;
                    }
                    // every loader thread is past item x - kStages (the wait above), so none has touched tile i + 2's yet
                    if (lt >= 32 && lt < 36) ms.odd[(i + 2) % kOddRing][lt - 32] = 0;
                    if (i + 1 < nt) pages_next = pages_of(key_of(i + 1));
                } else if (!open(key_of(i), pos_lo, pos_hi)) {  // values that are not numbers leave the operand
#pragma unroll
                    for (int y = 0; y < kPer; y++) {
                        uint32_t* w = reinterpret_cast<uint32_t*>(&got[y]);
                        bool odd = false;
#pragma unroll
                        for (int z = 0; z < 4; z++) {
                            // 0x80 of each byte whose low seven bits are all ones
                            const uint32_t nan = ((w[z] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
                            odd |= nan != 0;
                            w[z] &= ~(nan | (nan - (nan >> 7)));
                        }
                        const int r = row_in + y * kRowsAt;
                        if (odd) atomicOr(&ms.odd[i % kOddRing][r >> 5], 1u << (r & 31));  // r < 128: others are zeros
                    }
                }
#pragma unroll
                for (int y = 0; y < kPer; y++) {
                    const uint32_t ws[4] = {got[y].x, got[y].y, got[y].z, got[y].w};
                    uint32_t f[8];
#pragma unroll
                    for (int z = 0; z < 4; z++) f[2 * z] = e4m3x2_to_f16x2(uint16_t(ws[z])), f[2 * z + 1] = e4m3x2_to_f16x2(uint16_t(ws[z] >> 16));
                    const uint4 a0 = make_uint4(f[0], f[1], f[2], f[3]), a1 = make_uint4(f[4], f[5], f[6], f[7]);
                    const int r = row_in + y * kRowsAt;
                    if ((y + 1) * kRowsAt <= kKeys || r < kKeys) {
                        *reinterpret_cast<uint4*>(base + sw128_off(r, ch0)) = second ? a1 : a0;
                        *reinterpret_cast<uint4*>(base + sw128_off(r, ch1)) = second ? a0 : a1;
                    }
                }
                fence_proxy_async();
                mbar_arrive(&ms.full[st]);
                if (x + 1 < total) {  // the next item's pieces fly while this one is used
                    if (v) {
                        pages = pages_next;
                        scales();
                    }
                    fetch(v ? c.k_pages : c.v_pages, key_of((x + 1) >> 1));
                }
            }
        } else {
            // one warp starts the tensor copies, a lane per page and 64 values; all four look through the tiles that need it
            const int per_page = kKeys / c.page_size, box = lane >> (HD / 64 - 1), half = lane & (HD / 64 - 1);
            const uint32_t box_bytes = uint32_t(c.page_size) * 128;
            const bool carrier = box < per_page;  // at most 16 lanes (8 pages of 16 tokens, two halves)
            int scans = 0;
            int begun = 0;             // items whose copies have been started;
            uint32_t by_land = 0;      // bit x % 32: they complete on `land`, not on `full`;
            bool landing = false;      // `land` has not been seen complete since
            float ks = 0.0f, vs = 0.0f;
            auto scales = [&]() {
                if (SRC == kCopies && warp == kLoadWarp && pages >= 0) {
                    ks = c.k_scale[int64_t(pages) * c.scale_stride + kvh];
                    vs = c.v_scale[int64_t(pages) * c.scale_stride + kvh];
                }
            };
            if (nt > 0) scales();
            for (int x = 0; x < total; x++) {
                const int st = x % L::kStages, i = x >> 1;
                const bool v = x & 1;
                const int j0 = key_of(i);
                uint8_t* base = sm + L::kStageOff + st * L::kStage;
                const bool strict = !open(j0, pos_lo, pos_hi);
                const bool whole = __all_sync(0xffffffffu, lane >= 8 || pages >= 0), scan = v && (strict || !whole);
                if (warp == kLoadWarp) {
                    if (x >= L::kStages) {
                        ok = wait_on(&ms.empty[st], ((x / L::kStages) & 1) ^ 1, fail);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                    }
                    if (!v) {
                        const float vl = SRC == kCopies && lane < 8 && pages >= 0 ? fmaxf(log2f(vs), kVNone) : kVNone;
                        if (lane < 8) ms.ks[i % kRing][lane] = pages < 0 ? kGone : SRC == kCopies ? fabsf(ks) : 1.0f, ms.vs[i % kRing][lane] = vl;
                    }
                    if (!v && lane < 4) ms.odd[(i + 2) % kOddRing][lane] = 0;
                    if (!v && lane == 0) ms.whole[i % kRing] = whole;
                    int page = __shfl_sync(0xffffffffu, pages, carrier ? box << (ps_log - 4) : 31);
                    if (SRC == kCopies && page >= 0) page = s * c.max_pages + (j0 >> ps_log) + box;
                    const uint32_t boxes = __popc(__ballot_sync(0xffffffffu, page >= 0));
                    uint64_t* bar = scan ? &ms.land : &ms.full[st];
                    __syncwarp();  // lane 0's arrival publishes what the other lanes have written above
                    if (lane == 0) mbar_arrive_expect_tx(bar, boxes * box_bytes);
                    __syncwarp();
                    begun = x + 1, landing = scan;
                    by_land = (by_land & ~(1u << (x & 31))) | uint32_t(scan) << (x & 31);
                    if (page >= 0)
                        copy_box(base + half * L::kHalf + box * box_bytes, v ? &maps.v : &maps.k, half * 64, kvh * c.page_size, page, bar);
                }
                if (scan) {
                    ok = wait_on(&ms.land, scans & 1, fail);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    landing = false;
                    // rows that nobody holds are zeroed, values that are not finite taken out
                    uint32_t held_rows = 0;  // lane x < 8: rows of block x that are held
                    if (lane < 8 && pages >= 0) held_rows = uint32_t(min(max(len - j0 - 16 * lane, 0), 16));
                    constexpr int kChunks = HD / 8;  // 16-byte pieces of a key row
#pragma unroll 4
                    for (int k = 0; k < (kKeys * kChunks + kLoaders - 1) / kLoaders; k++) {  // as often for every lane
                        const int y = lt + k * kLoaders, r = y / kChunks, ch = y % kChunks;
                        const uint32_t held16 = __shfl_sync(0xffffffffu, held_rows, (r >> 4) & 7);
                        if (r < kKeys) {
                            uint4* p = reinterpret_cast<uint4*>(base + ch / 8 * L::kHalf + sw128_off(r, ch % 8));
                            uint4 u = (r & 15) < int(held16) ? *p : make_uint4(0, 0, 0, 0);
                            const bool odd = strict && drop_odd(u);
                            if (odd || (r & 15) >= int(held16)) *p = u;
                            if (odd) atomicOr(&ms.odd[i % kOddRing][r >> 5], 1u << (r & 31));
                        }
                    }
                    fence_proxy_async();
                    mbar_arrive(&ms.scanned);
                    if (warp == kLoadWarp) {
                        ok = wait_on(&ms.scanned, scans & 1, fail);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        if (lane == 0) mbar_arrive(&ms.full[st]);
                    }
                    scans++;
                }
                if (!v && i + 1 < nt) pages_next = pages_of(key_of(i + 1));
                if (v) {
                    pages = pages_next;
                    scales();
                }
            }
            // Given up: the copies that are still in flight land (again with a limit) before their place is used otherwise or the
            // CTA leaves.
            if (!ok && warp == kLoadWarp) {
                for (int x = max(begun - L::kStages, 0); x < begun; x++)
                    if (!(by_land >> (x & 31) & 1)) wait_out(&ms.full[x % L::kStages], (x / L::kStages) & 1);
                if (landing) wait_out(&ms.land, scans & 1);
                __syncwarp();
            }
        }
    } else if (warp == kMmaWarp) {
        // ------------------------------------------------------------------ UMMA issue
        // The whole warp walks the loop and one elected lane issues: with the role on a single lane of a divergent warp the
        // operands' descriptors went through vector registers, about 70 cycles an UMMA.
        if (nt > 0) {
            constexpr uint32_t idesc_s = f16_idesc(kRows, kKeys), idesc_o = f16_idesc(kRows, HD) | (1u << 16);
            const uint64_t q_desc = sw128_desc(smem_u32(sm)), k_desc = sw128_desc(smem_u32(sm + L::kStageOff)),
                           vv_desc = v_desc(smem_u32(sm + L::kStageOff));
            auto issue_s = [&](int h, int st) {
                const uint64_t qd = q_desc + uint64_t(h * L::kParts * (L::kQTile >> 4));
                const uint64_t kd = k_desc + uint64_t(st * (L::kStage >> 4));
                if (elect_one()) {
#pragma unroll
                    for (int part = L::kParts - 1; part >= 0; part--)  // the small products first: fewer steps truncate large sums
#pragma unroll
                        for (int k = 0; k < HD / 16; k++) {
                            const uint32_t off = ((k / 4) * L::kHalf + (k % 4) * 32) >> 4;
                            umma_f16(tmem + h * 128, qd + part * (L::kQTile >> 4) + off, kd + off, idesc_s, part < L::kParts - 1 || k > 0);
                        }
                    umma_commit(&ms.s_full[h]);
                }
            };
            auto issue_pv = [&](int h, int st) {
                // weights of keys 16 k ..: each thread's over its own scores; hi + lo: 32-column groups of hi, lo (16 each)
                const uint32_t p = tmem + h * 128, o = tmem + 256 + h * 128;
                const uint64_t vd = vv_desc + uint64_t(st * (L::kStage >> 4));
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < kKeys / 16; k++) {
                        const uint32_t col = HILO ? 32 * (k / 2) + 8 * (k % 2) : 64 * (k / 4) + 8 * (k % 4);
                        umma_ts(o, p + col, vd + k * (2048 >> 4), idesc_o);
                        if constexpr (HILO) umma_ts(o, p + col + 16, vd + k * (2048 >> 4), idesc_o);
                    }
                    umma_commit(&ms.pv_done[h]);
                }
            };
            auto commit = [&](uint64_t* bar) {
                if (elect_one()) umma_commit(bar);
            };
            bool ok = wait_on(&ms.q_full, 0, fail) && wait_on(&ms.full[0], 0, fail);
            ok = __all_sync(0xffffffffu, ok);
            if (ok) {
                for (int h = 0; h < mt; h++) issue_s(h, 0);
                commit(&ms.empty[0]);
            }
            int sv = 1, pv = 0, sk = 2 % L::kStages, pk = 2 / L::kStages;  // stages and phases of V of this tile and K of the next
            auto next = [&](int& st, int& ph) {
                st += 2;
                if (st >= L::kStages) st -= L::kStages, ph ^= 1;
            };
            for (int i = 0; i < nt && ok; i++) {
                ok = wait_on(&ms.full[sv], pv, fail);
                ok = __all_sync(0xffffffffu, ok);
                for (int h = 0; h < mt && ok; h++) {
                    ok = ok && wait_on(&ms.p_full[h], i & 1, fail);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    tc_fence_after();
                    issue_pv(h, sv);
                    if (h == mt - 1) commit(&ms.empty[sv]);
                    if (i + 1 < nt) {
                        if (h == 0) ok = wait_on(&ms.full[sk], pk, fail);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        issue_s(h, sk);
                        if (h == mt - 1) commit(&ms.empty[sk]);
                    }
                }
                next(sv, pv), next(sk, pk);
            }
            commit(&ms.drain);  // nothing is in flight when the TMEM is freed, whatever happened
            wait_out(&ms.drain, 0);
        }
        __syncwarp();
    } else {
        // ------------------------------------------------------------------ queries: eight lanes a row, hd / 8 values each
        constexpr int E = HD / 8;
        const auto load_q = [&](auto* base) {
#pragma unroll 2
            for (int r = warp * 4 + (lane >> 3); r < mt * kRows; r += 4 * kSoftWarps) {
                float x[E];
#pragma unroll
                for (int e = 0; e < E; e++) x[e] = 0.0f;
                if (r < rows) {
                    const int pr = r0 + r, rt = over_g(pr);
                    const auto* p = base + int64_t(row0 + rt) * a.q_token + int64_t(kvh * G + pr - rt * G) * a.q_head + (lane & 7) * E;
                    const bool vec = (reinterpret_cast<uintptr_t>(p) & (sizeof(*p) * 4 - 1)) == 0;
#pragma unroll
                    for (int e = 0; e < E; e += 4) load_row<4>(p + e, vec, *reinterpret_cast<float(*)[4]>(&x[e]));
                }
                float most = 0.0f;
#pragma unroll
                for (int e = 0; e < E; e++) most = fmaxf(most, finite_abs(x[e]));
#pragma unroll
                for (int o = 4; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                const float up = row_up(most);
                const int d = (lane & 7) * E;
                uint8_t* dst = sm + (r / kRows * L::kParts) * L::kQTile + d / 64 * L::kHalf;
#pragma unroll
                for (int e = 0; e < E; e += 8) {
                    uint32_t h2[4], l2[4];
#pragma unroll
                    for (int y = 0; y < 4; y++) split_hilo(x[e + 2 * y] * up, x[e + 2 * y + 1] * up, h2[y], l2[y]);
                    const uint32_t at = sw128_off(r % kRows, (d % 64 + e) / 8);
                    *reinterpret_cast<uint4*>(dst + at) = make_uint4(h2[0], h2[1], h2[2], h2[3]);
                    if constexpr (HILO) *reinterpret_cast<uint4*>(dst + L::kQTile + at) = make_uint4(l2[0], l2[1], l2[2], l2[3]);
                }
                if ((lane & 7) == 0) ms.most[0][r] = a.scale / up;
            }
        };
        if constexpr (HILO) load_q(static_cast<const float*>(a.q));
        else if (a.type == kTF16) load_q(static_cast<const __half*>(a.q));
        else load_q(static_cast<const __nv_bfloat16*>(a.q));
        fence_proxy_async();
        mbar_arrive(&ms.q_full);
    }
    const int half_w = warp / 8, col_w = (warp >> 2) & 1;  // of a softmax warp: row tile and half of the key tile
    const int row_w = half_w * kRows + (warp & 3) * 32 + lane;
    if (warp < kSoftWarps && half_w < mt) {
        // ------------------------------------------------------------------ softmax, two threads per row
        const int h = half_w, r = row_w, pr = r0 + r;
        const uint32_t lanes = uint32_t(32 * (warp & 3)) << 16;
        const uint32_t ts = tmem + lanes + h * 128, to = tmem + lanes + 256 + h * 128 + col_w * (HD / 2);
        const bool real = r < rows;
        const int rt = over_g(pr), qpos = real ? held - n + rt : kNoRow;
        const float slope = a.slopes && real ? a.slopes[kvh * G + pr - rt * G] * kLog2e : 0.0f;
        const int h_lo = held - n + over_g(r0 + h * kRows), h_hi = held - n + over_g(r0 + min(rows, (h + 1) * kRows) - 1);
        const float cap = a.softcap * kLog2e;
        {
            uint32_t z[32];
#pragma unroll
            for (int x = 0; x < 32; x++) z[x] = 0;
#pragma unroll
            for (int x = 0; x < HD / 2; x += 32) st32(to + x, z);
            st_wait();
        }
        wait_on(&ms.q_full, 0, fail);
        __syncwarp();
        // from the accumulator to log2 units, or with a cap to the tanh's argument
        // (and what the scores' own HD / 16 steps truncate)
        const float whole_score = ms.most[0][r] * (1.0f + (HD / 16 + 1) / 2.0f * kDrop);
        const float factor = a.softcap > 0.0f ? whole_score / a.softcap : whole_score * kLog2e;
        // The two warps of 32 rows meet at a named barrier of theirs: no wait of this role ends it early (a wait that gives up
        // has set the fail flag, and every later one returns at once), so both always come to every meeting.
        auto meet = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(1 + 4 * h + (warp & 3)) : "memory"); };
        meet();  // both threads of a row have read its factor before either writes
        for (int i = 0; i < nt; i++) {
            const int j0 = key_of(i);
            const bool open_rows = open(j0, h_lo, h_hi), open_cta = open(j0, pos_lo, pos_hi);
            const float* ksp = ms.ks[i % kRing];
            const float* vsp = ms.vs[i % kRing];
            wait_on(&ms.s_full[h], i & 1, fail);
            __syncwarp();
            tc_fence_after();
            if constexpr (HILO) {
                if (i > 0 && i % kFlush == 0 && ms.slot >= 0) {
                    wait_on(&ms.pv_done[h], (i - 1) & 1, fail);
                    __syncwarp();
                    tc_fence_after();
                    const bool again = kept != nullptr;
                    kept = plan.flush + (int64_t(ms.slot) * HD + col_w * (HD / 2)) * (2 * kRows) + r;
                    const float now = row_max == -INFINITY ? 0.0f : row_max, f = ex2(fminf(kept_ref - now, 0.0f));
                    kept_ref = now;
                    sum_kept += row_sum;
                    row_sum = 0.0f;
#pragma unroll 1
                    for (int x = 0; x < HD / 2; x += 16) {
                        uint32_t o[16];
                        ld16(to + x, o);
                        float was[16];
#pragma unroll
                        for (int y = 0; y < 16; y++) was[y] = again ? kept[(x + y) * (2 * kRows)] : 0.0f;
                        ld_wait16(o);
#pragma unroll
                        for (int y = 0; y < 16; y++) {
                            kept[(x + y) * (2 * kRows)] = fmaf(was[y], f, __uint_as_float(o[y]));
                            o[y] = 0;
                        }
                        st16(to + x, o);
                    }
                    st_wait();
                }
            }
            const bool plain_mask = open_rows && ms.whole[i % kRing];
            const int xv = 2 * i + 1, stv = xv % L::kStages;
            bool odd_tile = false;
            if (!open_cta) {
                wait_on(&ms.full[stv], (xv / L::kStages) & 1, fail);
                __syncwarp();
                const uint32_t* od = ms.odd[i % kOddRing];
                odd_tile = (od[0] | od[1] | od[2] | od[3]) != 0;
            }
            // this thread's half of its row of O times f, and this tile's values that are not finite
            auto fix_o = [&](float f, bool odd) {
                if (i > 0) {
                    wait_on(&ms.pv_done[h], (i - 1) & 1, fail);
                    __syncwarp();
                    tc_fence_after();
                }
#pragma unroll 1
                for (int x = 0; x < HD / 2; x += 16) {
                    uint32_t o[16];
                    ld16(to + x, o);
                    ld_wait16(o);
#pragma unroll
                    for (int y = 0; y < 16; y++) o[y] = __float_as_uint(__uint_as_float(o[y]) * f);
                    if (odd) {
#pragma unroll 1
                        for (int key = 0; key < kKeys; key++) {
                            if (!(ms.odd[i % kOddRing][key >> 5] >> (key & 31) & 1)) continue;
                            const int j = j0 + key, slot = j / c.page_size;
                            if (j >= len || ksp[key >> 4] == kGone) continue;
                            const bool see = (j <= qpos && (!a.window || qpos - j < a.window)) || (j < prefix && qpos != kNoRow);
                            const int64_t at = int64_t(c.table[int64_t(s) * c.table_stride + slot]) * c.page_stride +
                                               (int64_t(kvh) * c.page_size + j % c.page_size) * HD + col_w * (HD / 2) + x;
#pragma unroll
                            for (int y = 0; y < 16; y++) {
                                float v;
                                if constexpr (kScaled) {
                                    v = (static_cast<const uint8_t*>(c.v_pages)[at + y] & 0x7f) == 0x7f ? NAN : 0.0f;
                                } else {
                                    v = __half2float(static_cast<const __half*>(c.v_pages)[at + y]);
                                    if (fabsf(v) <= 65504.0f) v = 0.0f;
                                }
                                if (see) o[y] = __float_as_uint(__uint_as_float(o[y]) + v);
                            }
                        }
                    }
                    st16(to + x, o);
                }
                st_wait();
            };
            if (odd_tile) fix_o(1.0f, true);
            // ---- tiles that need more than the scale: a cap, a bias, masks; 32 scores at a time in a rolled loop, in log2 units
            // back into TMEM
            const float *kb = ksp + 4 * col_w, *vb = vsp + 4 * col_w;  // of this thread's blocks of 16 keys
            const uint32_t tc = ts + 64 * col_w;
            const bool shaped = a.softcap > 0.0f || a.slopes || !plain_mask || a.scale < 0.0f;
            if (shaped) {
#pragma unroll 1
                for (int q = 0; q < 2; q++) {
                    uint32_t u[32];
                    ld32(tc + 32 * q, u);
                    const float f0 = kScaled ? factor * fabsf(kb[2 * q]) : factor, f1 = kScaled ? factor * fabsf(kb[2 * q + 1]) : factor;
                    ld_wait(u);
                    const int jq = j0 + 64 * col_w + 32 * q;
                    float most = 0.0f;
#pragma unroll
                    for (int x = 0; x < 32; x++) {
                        u[x] = __float_as_uint(__uint_as_float(u[x]) * (x < 16 ? f0 : f1));
                        most = max_nan(most, fabsf(__uint_as_float(u[x])));
                    }
                    if (a.softcap > 0.0f) {  // of score / cap
                        if (__all_sync(0xffffffffu, most <= 0.5f)) {
                            // an odd polynomial of degree 9 (largest error on [-1/2, 1/2]: 6.3e-9): two units of the
                            // special functions less than below
#pragma unroll
                            for (int x = 0; x < 32; x += 2) {
                                const uint64_t y = pack2(__uint_as_float(u[x]), __uint_as_float(u[x + 1])), y2 = mul2(y, y);
                                uint64_t p = fma2(y2, pack2(0.016737453639507294f, 0.016737453639507294f), pack2(-0.05276207625865936f, -0.05276207625865936f));
                                p = fma2(p, y2, pack2(0.13320569694042206f, 0.13320569694042206f));
                                p = fma2(p, y2, pack2(-0.3333277702331543f, -0.3333277702331543f));
                                p = fma2(p, y2, pack2(0.9999999403953552f, 0.9999999403953552f));
                                p = mul2(mul2(p, y), pack2(cap, cap));
                                float p0, p1;
                                unpack2(p, p0, p1);
                                u[x] = __float_as_uint(p0), u[x + 1] = __float_as_uint(p1);
                            }
                        } else {
#pragma unroll
                            for (int x = 0; x < 32; x++) {
                                const float y = __uint_as_float(u[x]);
                                u[x] = __float_as_uint(cap * (fabsf(y) <= 0.5f ? tanh_small(y) : tanh_abs(y)));
                            }
                        }
                    }
                    if (a.slopes) {
#pragma unroll
                        for (int x = 0; x < 32; x++) u[x] = __float_as_uint(fmaf(slope, float(jq + x - qpos), __uint_as_float(u[x])));
                    }
                    if (!plain_mask) {
                        // seen: j in [see_lo, see_hi) or j < pre, and the block is resident
                        const int see_hi = min(len, qpos + 1) - jq, see_lo = (a.window && qpos >= a.window ? qpos - a.window + 1 : 0) - jq;
                        const int pre = (real ? prefix : 0) - jq;
                        const bool gone0 = kb[2 * q] == kGone, gone1 = kb[2 * q + 1] == kGone;
#pragma unroll
                        for (int x = 0; x < 32; x++)
                            if (!((x < see_hi && x >= see_lo) || x < pre) || (x < 16 ? gone0 : gone1)) u[x] = 0xff800000u;
                    }
                    st32(tc + 32 * q, u);
                }
                st_wait();
            }
            // ---- this thread's 64 scores and the largest of them, with their blocks' value scales and without
            uint32_t u[2][32];
            ld32(tc, u[0]);
            ld32(tc + 32, u[1]);
            float fb[4];  // what brings them to log2 units
#pragma unroll
            for (int b = 0; b < 4; b++) fb[b] = shaped ? 1.0f : kScaled ? factor * kb[b] : factor;
            ld_wait(u[0]), ld_wait(u[1]);
            float top = -INFINITY, top_score = -INFINITY;
#pragma unroll
            for (int b = 0; b < 4; b++) {
                float m[4];
#pragma unroll
                for (int x = 0; x < 16; x++) {
                    const float v = __uint_as_float(u[b / 2][16 * (b & 1) + x]);
                    m[x & 3] = x < 4 ? v : max_nan(m[x & 3], v);
                }
                const float most = max_nan(max_nan(m[0], m[1]), max_nan(m[2], m[3])) * fb[b];
                top = max_nan(top, kScaled ? most + vb[b] : most);
                if (kScaled) top_score = max_nan(top_score, most);
            }
            if (kScaled && top_score > sum_max && top_score < INFINITY) {
                top_score = ceilf(top_score);
                const float f = ex2(sum_max - top_score);  // from -inf: 0
                sum_max = top_score, row_sum *= f;
                if (HILO) sum_kept *= f;
            }
            // One buffer: this tile's scores exist, so the other thread has handed in its last weights and read this one's.
            ms.most[col_w][r] = top;
            meet();
            top = max_nan(top, ms.most[col_w ^ 1][r]);
            if (!(top < INFINITY)) row_sum = NAN;  // as exp(inf - inf) and exp(NaN) give, whatever computes the weights
            // The reference moves only when a score exceeds it by more than 2^kLazy (the same decision in both warps of a row), and then to
            // that score itself: its weight, often most of the row, is a power of two and f16 takes nothing off it (whole
            // powers of two as references: f16 rows' error 2.9e-4 instead of 2.6e-4).
            const bool up = top > row_max + kLazy && top < INFINITY;  // also from -inf
            if (__any_sync(0xffffffffu, up)) {
                float f = 1.0f;
                if (up) {
                    f = ex2(row_max - top);  // row_max = -inf: nothing there yet, 0
                    row_max = top;
                    if (!kScaled) row_sum *= f;
                    if (!kScaled && HILO) sum_kept *= f;
                }
                if (i > 0) fix_o(f, false);
            }
            // ---- weights, their sum; P over this thread's scores
            const float ref = row_max == -INFINITY ? 0.0f : row_max, sum_ref = sum_max == -INFINITY ? 0.0f : sum_max;
            float sum = 0.0f;
            uint64_t sums[2] = {0, 0};
#pragma unroll
            for (int b = 0; b < 4; b++) {
                const int q = b / 2, g = b & 1;
                // weights of score and scale against the reference: 2^vr times what they add to the sum
                const float vr = kScaled ? fmaxf(vb[b] + (sum_ref - ref), kVMin) : 0.0f, o = (kScaled ? vr - sum_ref : -ref) + kLift;
                const uint64_t ff = pack2(fb[b], fb[b]), off = pack2(o, o);
                if (kScaled) sums[0] = sums[1] = 0;
                [[maybe_unused]] uint32_t lo8[8];
#pragma unroll
                for (int x = 16 * g; x < 16 * g + 16; x += 2) {
                    float z0, z1;
                    unpack2(fma2(pack2(__uint_as_float(u[q][x]), __uint_as_float(u[q][x + 1])), ff, off), z0, z1);
                    if (!HILO && (x & 7) == 6) exp2_poly(z0, z1);
                    else z0 = ex2(z0), z1 = ex2(z1);
                    sums[x / 2 & 1] = add2(sums[x / 2 & 1], pack2(z0, z1));
                    // f16 weights in the scores' registers
                    if constexpr (HILO) split_hilo(z0, z1, u[q][16 * g + (x & 15) / 2], lo8[(x & 15) / 2]);
                    else u[q][x / 2] = h2u(__floats2half2_rn(z0, z1));
                }
                if constexpr (HILO) {
                    st8(tc + 32 * q + 8 * g, &u[q][16 * g]);
                    st8(tc + 32 * q + 16 + 8 * g, lo8);
                } else if (g) {
                    st16(tc + 16 * q, *reinterpret_cast<const uint32_t(*)[16]>(u[q]));
                }
                if (kScaled || b == 3) {  // the sum without the value scale
                    float z0, z1;
                    unpack2(add2(sums[0], sums[1]), z0, z1);
                    sum = kScaled ? fmaf(z0 + z1, ex2(-vr), sum) : z0 + z1;
                }
            }
            constexpr float kSteps = kKeys / 16 * L::kParts;
            row_sum = row_sum - fminf(kSteps * kDrop * row_sum, sum) + fmaf(sum, -(kSteps + 1) / 2 * kDrop, sum);
            st_wait();
            tc_fence_before();
            mbar_arrive(&ms.p_full[h]);
        }
        if (nt > 0) {
            wait_on(&ms.pv_done[h], (nt - 1) & 1, fail);
            __syncwarp();
            tc_fence_after();
        }
        if constexpr (kScaled) {  // the two halves' sums in one unit
            ms.most[col_w][r] = sum_max;
            meet();
            const float both = fmaxf(sum_max, ms.most[col_w ^ 1][r]);
            meet();  // both are read before the sums take their place
            if (sum_max > -INFINITY) {
                const float f = ex2(sum_max - both);
                row_sum *= f;
                if (HILO) sum_kept *= f;
            }
            sum_max = both;
        }
    }
    // ---- the outputs. Alone: through shared memory, once the operands are used up. In a cluster each CTA owns a share of
    // the rows: every CTA pushes its states of them into the owner's shared memory.
    __syncwarp();
    if (HILO) row_sum += sum_kept;
    if (warp < kSoftWarps && half_w < mt) ms.most[col_w][row_w] = row_sum;
    const bool alone = plan.ranks == 1;
    cg::cluster_group cluster = cg::this_cluster();
    if (alone) __syncthreads();
    else cluster.sync();
    float* state = reinterpret_cast<float*>(sm);  // [rank][row of the share][values, maximum, sum]
    const int share = mt * kRows / plan.ranks;
    if (warp < kSoftWarps && half_w < mt) {
        const int r = row_w;
        const uint32_t to = tmem + (uint32_t(32 * (warp & 3)) << 16) + 256 + half_w * 128 + col_w * (HD / 2);
        row_sum += ms.most[col_w ^ 1][r];
        // A row without keys goes by its reference: its sum holds the 2^-126 that exp2_poly gives a masked score (NaN stays).
        const bool none = row_max == -INFINITY && row_sum == row_sum;
        float f = 1.0f;
        if (alone) f = none ? 0.0f : (kScaled && row_max > -INFINITY ? exp2f(row_max - sum_max) : 1.0f) / row_sum;
        const float f_kept = ex2(fminf(kept_ref - (row_max == -INFINITY ? 0.0f : row_max), 0.0f));
        float* mine = (alone ? state : cluster.map_shared_rank(state, r / share)) + (rank * share + r % share) * L::kJoinPitch;
#pragma unroll
        for (int x = 0; x < HD / 2; x += 32) {
            uint32_t w[32];
            ld32(to + x, w);
            ld_wait(w);
            if (HILO && kept) {
#pragma unroll
                for (int y = 0; y < 32; y++) w[y] = __float_as_uint(fmaf(kept[(x + y) * (2 * kRows)], f_kept, __uint_as_float(w[y])));
            }
#pragma unroll
            for (int y = 0; y < 32; y += 4) {
                float4 v = make_float4(__uint_as_float(w[y]) * f, __uint_as_float(w[y + 1]) * f, __uint_as_float(w[y + 2]) * f,
                                       __uint_as_float(w[y + 3]) * f);
                if (alone && none) v = make_float4(0, 0, 0, 0);
                *reinterpret_cast<float4*>(mine + col_w * (HD / 2) + x + y) = v;
            }
        }
        if (!col_w) mine[HD] = row_max, mine[HD + 1] = row_sum, mine[HD + 2] = kScaled ? sum_max : row_max;
    }
    tc_fence_before();
    if (alone) __syncthreads();
    else cluster.sync();
    if (HILO && tid == 32 * kLoadWarp && plan.taken && ms.slot >= 0) {  // every thread has read its sums
        __threadfence();
        atomicExch(&plan.taken[ms.slot], 0u);
    }
    if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    auto put = [&](int r, int d, float4 v) {
        const int pr = r0 + r;
        const int rt = over_g(pr);
        const int64_t off = int64_t(row0 + rt) * a.o_token + int64_t(kvh * G + pr - rt * G) * a.o_head + d;
        const float x[4] = {v.x, v.y, v.z, v.w};
        auto store = [&](auto* p) { store_row<4>(p, (reinterpret_cast<uintptr_t>(p) & (sizeof(*p) * 4 - 1)) == 0, x); };
        if (a.type == kTF32) store(static_cast<float*>(a.out) + off);
        else if (a.type == kTF16) store(static_cast<__half*>(a.out) + off);
        else store(static_cast<__nv_bfloat16*>(a.out) + off);
    };
    if (alone) {
        for (int x = tid; x < rows * (HD / 4); x += kThreads) {
            const int r = x / (HD / 4), d = x % (HD / 4) * 4;
            put(r, d, *reinterpret_cast<const float4*>(state + r * L::kJoinPitch + d));
        }
        return;
    }
    const int mine = min(max(rows - rank * share, 0), share);  // rows that this CTA owns
    for (int x = tid; x < mine * (HD / 4); x += kThreads) {
        const int r = x / (HD / 4), d = x % (HD / 4) * 4;
        float top = -INFINITY, top_sum = -INFINITY, sum = 0.0f;
        for (int w = 0; w < plan.ranks; w++) {
            const float* st = state + (w * share + r) * L::kJoinPitch;
            top = fmaxf(top, st[HD]), top_sum = fmaxf(top_sum, st[HD + 2]);
        }
        const float ref = top == -INFINITY ? 0.0f : top, sum_ref = top_sum == -INFINITY ? 0.0f : top_sum;
        float4 v = make_float4(0, 0, 0, 0);
        for (int w = 0; w < plan.ranks; w++) {
            const float* st = state + (w * share + r) * L::kJoinPitch;
            const float f = ex2(st[HD] - ref);
            const float4 o = *reinterpret_cast<const float4*>(st + d);
            sum = fmaf(kScaled ? ex2(st[HD + 2] - sum_ref) : f, st[HD + 1], sum), v.x = fmaf(f, o.x, v.x), v.y = fmaf(f, o.y, v.y), v.z = fmaf(f, o.z, v.z), v.w = fmaf(f, o.w, v.w);
        }
        const float f = (kScaled ? exp2f(ref - sum_ref) : 1.0f) / sum;
        put(rank * share + r, d, sum == 0.0f ? make_float4(0, 0, 0, 0) : make_float4(v.x * f, v.y * f, v.z * f, v.w * f));
    }
}

// f16 copies of the 8-bit pages that the sequences hold: block (s, i) of the copies is page table[s][i], codes without
// their scales (exact). A CTA per (sequence, page, K or V).
__global__ void __launch_bounds__(256) paged_copies_kernel(const neko_paged_attention_args a, uint4* copies) {
    const neko_paged_cache& c = a.cache;
    const int slot = blockIdx.x, s = blockIdx.y, v = blockIdx.z;
    const int page = c.table[int64_t(s) * c.table_stride + slot];
    if (int64_t(slot) * c.page_size >= a.kv_len[s] || page < 0 || page >= c.num_pages) return;
    const int pieces = c.n_kv * c.page_size * c.head_dim / 16;
    const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(v ? c.v_pages : c.k_pages) + int64_t(page) * c.page_stride);
    uint4* dst = copies + (int64_t(v) * c.n_seq * c.max_pages + int64_t(s) * c.max_pages + slot) * pieces * 2;
    for (int i0 = threadIdx.x; i0 < pieces; i0 += 4 * 256) {
        uint4 w[4];
#pragma unroll
        for (int y = 0; y < 4; y++)
            if (i0 + 256 * y < pieces) w[y] = ldg_stream(src + i0 + 256 * y);
#pragma unroll
        for (int y = 0; y < 4; y++) {
            if (i0 + 256 * y >= pieces) break;
            const uint32_t ws[4] = {w[y].x, w[y].y, w[y].z, w[y].w};
            uint32_t f[8];
#pragma unroll
            for (int z = 0; z < 4; z++) f[2 * z] = e4m3x2_to_f16x2(uint16_t(ws[z])), f[2 * z + 1] = e4m3x2_to_f16x2(uint16_t(ws[z] >> 16));
            dst[2 * (i0 + 256 * y)] = make_uint4(f[0], f[1], f[2], f[3]);
            dst[2 * (i0 + 256 * y) + 1] = make_uint4(f[4], f[5], f[6], f[7]);
        }
    }
}

template <int HD, int SRC, bool HILO>
cudaError_t go(const neko_paged_attention_args& a, const PromptPlan& p, int64_t items, const __half* copies, cudaStream_t st) {
    using L = PL<HD, HILO>;
    const neko_paged_cache& c = a.cache;
    auto* fn = paged_prompt_kernel<HD, SRC, HILO>;
    if (cudaError_t e = ensure_dyn_smem(fn, L::kSmem); e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(items * p.ranks));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = L::kSmem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = unsigned(p.ranks);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = p.ranks > 1 ? 1 : 0;
    PromptMaps maps = {};
    if (SRC != kCodes) {
        const int64_t rows = int64_t(c.n_kv) * c.page_size, own = rows * HD, pages = int64_t(c.n_seq) * c.max_pages;
        const bool copy = SRC == kCopies;
        if (!encode_f16_pages(&maps.k, copy ? copies : c.k_pages, HD, rows, copy ? pages : c.num_pages, (copy ? own : c.page_stride) * 2, c.page_size) ||
            !encode_f16_pages(&maps.v, copy ? copies + pages * own : c.v_pages, HD, rows, copy ? pages : c.num_pages, (copy ? own : c.page_stride) * 2, c.page_size))
            return cudaErrorNotSupported;
    }
    return cudaLaunchKernelEx(&cfg, fn, a, p, maps);
}

template <int HD, int SRC>
cudaError_t by_type(const neko_paged_attention_args& a, const PromptPlan& p, int64_t items, const __half* copies, cudaStream_t st) {
    return a.type == NEKO_T_F32 ? go<HD, SRC, true>(a, p, items, copies, st) : go<HD, SRC, false>(a, p, items, copies, st);
}

template <int HD>
cudaError_t by_pages(const neko_paged_attention_args& a, const PromptPlan& p, int64_t items, cudaStream_t st) {
    const neko_paged_cache& c = a.cache;
    if (c.type != NEKO_T_E4M3) return by_type<HD, kF16Pages>(a, p, items, nullptr, st);
    // Each CTA would convert its keys again: from kCopyTiles CTAs per (sequence, KV head) on, they are converted once,
    // if the copies stay below kCopyBytes. Not copied and copied, f32 rows: 2 CTAs each (8 x 2,048 keys, 256 tokens) 128 and
    // 113 us, (4 x 8,192) 238 and 201; 6 each (1 x 8,192, 768 tokens) 349 and 239. One each gains less (16 x 4,096 keys,
    // 128 tokens: 256 and 238), for copies that are twice the cache.
    const int64_t bytes = 2 * int64_t(c.n_seq) * c.max_pages * c.n_kv * c.page_size * HD * 2;
    if (p.row_tiles < kCopyTiles || bytes > kCopyBytes) return by_type<HD, kCodes>(a, p, items, nullptr, st);
    void* mem = nullptr;
    if (scratch_alloc(&mem, size_t(bytes), st) != cudaSuccess) {  // a cache that fills the GPU: every CTA converts its own
        cudaGetLastError();
        return by_type<HD, kCodes>(a, p, items, nullptr, st);
    }
    cudaError_t e = launch_ex(paged_copies_kernel, dim3(unsigned(c.max_pages), unsigned(c.n_seq), 2), dim3(256), 0, st, false, a,
                              static_cast<uint4*>(mem));
    if (e == cudaSuccess) e = by_type<HD, kCopies>(a, p, items, static_cast<const __half*>(mem), st);
    cudaFreeAsync(mem, st);
    return e;
}

// How many clusters of 1 << log CTAs run at once on the current device (a CTA fills an SM; an SM left over in its GPC stays
// idle). Asked once per device; threads that ask at the same time get the same answer.
template <int HD>
int clusters_at_once(int log) {
    static std::atomic<int> known[64][4];
    int dev = 0;
    cudaGetDevice(&dev);
    std::atomic<int>& slot = known[dev & 63][log];
    if (const int n = slot.load(std::memory_order_relaxed)) return n;
    int n = num_sms();
    if (log > 0) {
        auto* fn = paged_prompt_kernel<HD, kCodes, true>;
        cudaLaunchConfig_t cfg = {};
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 1u << log;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.gridDim = dim3(1u << log);
        cfg.blockDim = dim3(kThreads);
        cfg.dynamicSmemBytes = PL<HD, true>::kSmem;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        if (ensure_dyn_smem(fn, PL<HD, true>::kSmem) != cudaSuccess || cudaOccupancyMaxActiveClusters(&n, fn, &cfg) != cudaSuccess || n <= 0) {
            cudaGetLastError();
            n = std::max(1, num_sms() >> (log + 1));
        }
    }
    slot.store(n, std::memory_order_relaxed);
    return n;
}

// Row tiles of a CTA and CTAs of a cluster: what takes the least time by the measured cost of 128 keys (one and two row
// tiles, in tenths of a microsecond), of a CTA's start and of the join. Two row tiles share a CTA's keys and its tensor core
// (one prompt of 768 f32 tokens on 8,192 keys, 8 KV heads: one row tile each 239 us, two in clusters of 2 159); one is
// better where that fills SMs (512 bf16 tokens on 2,048 keys: 30.4 us, two in clusters of 4 33.7). Without clusters 64 f32 tokens
// on 8,192 keys take 207 us, with clusters of 8 39; 16 clusters of 8 do not run at once and 90 us become 62 with 8 of them.
template <int HD>
int64_t split(PromptPlan& p, int64_t tiles, int64_t heads, int64_t key_tiles, bool f32) {
    const int64_t step[2] = {f32 ? 34 : 23, f32 ? 41 : 26}, start = 80, join[2] = {50, 150};
    int64_t best = INT64_MAX, items = 0;
    for (int two = 0; two < (tiles > 1 ? 2 : 1); two++) {
        const int64_t row_tiles = (tiles + two) / (1 + two), n = heads * row_tiles;
        for (int log = 0; log < 4 && (log == 0 || key_tiles >= (1 << log)); log++) {
            const int64_t at_once = clusters_at_once<HD>(log), rounds = (n + at_once - 1) / at_once;
            const int64_t time = rounds * (start + ((key_tiles + (1 << log) - 1) >> log) * step[two] + (log ? join[two] : 0));
            if (time >= best) continue;
            best = time, items = n;
            p.tiles_per = 1 + two, p.row_tiles = int(row_tiles), p.ranks = 1 << log;
        }
    }
    return items;
}

template <int HD>
cudaError_t by_source(const neko_paged_attention_args& a, cudaStream_t st) {
    const neko_paged_cache& c = a.cache;
    const int64_t rows = int64_t(a.max_new) * (a.n_head / c.n_kv);
    PromptPlan p;
    p.group = a.n_head / c.n_kv;
    p.group_inv = ((uint64_t(1) << 32) + p.group - 1) / p.group;
    const int64_t key_tiles = (int64_t(c.max_pages) * c.page_size + kKeys - 1) / kKeys;
    const int64_t items = split<HD>(p, (rows + kRows - 1) / kRows, int64_t(c.n_seq) * c.n_kv, key_tiles, a.type == NEKO_T_F32);
    if (items * p.ranks > 0x7fffffff) return cudaErrorInvalidConfiguration;
    p.flush = nullptr, p.taken = nullptr;
    p.slots = int(std::min<int64_t>(items * p.ranks, num_sms()));
    void* flush = nullptr;
    if (a.type == NEKO_T_F32 && key_tiles > int64_t(p.ranks) * kFlush) {
        const bool shared = items * p.ranks > p.slots;
        const size_t bytes = size_t(p.slots) * 2 * kRows * HD * 4;  // at most 19 MB
        if (cudaError_t e = scratch_alloc(&flush, bytes + size_t(p.slots) * 4, st); e != cudaSuccess) return e;
        p.flush = static_cast<float*>(flush);
        if (shared) {
            p.taken = reinterpret_cast<uint32_t*>(static_cast<char*>(flush) + bytes);
            if (cudaError_t e = cudaMemsetAsync(p.taken, 0, size_t(p.slots) * 4, st); e != cudaSuccess) {
                cudaFreeAsync(flush, st);
                return e;
            }
        }
    }
    const cudaError_t e = by_pages<HD>(a, p, items, st);
    if (flush) cudaFreeAsync(flush, st);
    return e;
}

}  // namespace

cudaError_t launch_paged_prompt(const neko_paged_attention_args& a, cudaStream_t st) {
    return a.cache.head_dim == 64 ? by_source<64>(a, st) : by_source<128>(a, st);
}

}  // namespace neko
