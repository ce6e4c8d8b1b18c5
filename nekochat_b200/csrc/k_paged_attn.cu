// Attention of few query rows over a paged cache (neko_op_paged_attention): decode steps, short continuations, small
// prompts, and every head dim of 32.
//
// Bound by memory: on contexts of one length 5.6 TB/s from 8-bit pages and 6.5 TB/s from f16 ones (74 x 8,192 tokens, 87 and
// 101 % of the measured copy rate; the value scales' exponents cost the former 5 %), 5.2 TB/s on 128 ragged contexts up to
// 8,192 tokens (232 us); small calls by latency.
//
// The packed rows of a (sequence, KV head) are its new tokens times the G query heads that share the KV head, so a key
// is read once for all of them. Every warp owns groups of 16 keys and works alone (no barrier until the end): scores
// S^T = K q^T and O^T += V^T P^T on mma.sync m16n8k16 with keys / head dims as the MMA's 16 rows and the query rows as
// its 8 columns. The order of the summed index is free as long as both operands agree, so the fragments come straight
// from global memory: lane (g, t) holds, for K, 16-byte pieces t, t + 4, .. of key rows g and g + 8, and for V the
// pieces g, g + 8, .. of key rows 2t, 2t + 1, 2t + 8, 2t + 9; neither K nor V passes through shared memory. 8-bit codes
// become f16 in registers (exact), keys' scales multiply the scores, values' scales enter the weights' exponent: a row's
// reference is the largest score plus log2 of the value scale that it sees, and the sum of its weights has the largest score
// as a unit of its own, so what f16 rounds off a weight is small beside the largest of the row's products. P reaches the
// second product by transposing 8 x 8 tiles in registers (movmatrix).
// f32 queries are two columns each, f16 hi and lo (22 bits; scores are the columns' sum), and so are their weights P;
// 16-bit queries one f16 column, weights one f16. Rows are scaled by a power of two into f16's range first (exact, but for
// bf16 values below 2^-17 of their row's largest, which lose bits).
// All groups of all items, in order, are dealt out in equal shares to the warps that the GPU holds at a time, whatever
// the lengths; each CTA adds up the sequences' groups itself (the lengths are on the device only). A warp goes through
// its share item by item, its start-up hidden behind the other warps of its SM: nothing waits for a CTA's other warps
// until all are done, when the parts of an item meet in shared memory. What several CTAs share is joined from their parts
// by a second small kernel, in order, so results do not depend on timing.
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "paged.cuh"
#include "paged_math.cuh"

namespace cg = cooperative_groups;

namespace neko {

namespace {

__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
    uint32_t d;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(sel));
    return d;
}
// The bits of a word's values that are not finite (8-bit codes: NaN).
template <bool Q8>
__device__ __forceinline__ uint32_t odd_lanes(uint32_t w) {
    if constexpr (Q8) {
        const uint32_t nan = ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
        return nan | (nan - (nan >> 7));
    } else {
        return ((w & 0x7c00u) == 0x7c00u ? 0xffffu : 0u) | ((w & 0x7c000000u) == 0x7c000000u ? 0xffff0000u : 0u);
    }
}

// Words (4 bytes) of one key row that a lane holds: K (a quarter of the row) and V (an eighth).
template <int HD, bool Q8>
struct Words {
    static constexpr int kRow = HD * (Q8 ? 1 : 2);
    static constexpr int kK = kRow / 16, kV = kRow / 32;
};

// N words in pieces of up to 16 bytes, piece i at p + i * step bytes.
template <int N>
__device__ __forceinline__ void load_words(const uint8_t* p, int step, uint32_t (&w)[N]) {
    if constexpr (N == 1) {
        asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(w[0]) : "l"(p));
    } else if constexpr (N == 2) {
        asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
    } else {
#pragma unroll
        for (int i = 0; i < N / 4; i++) {
            const uint4 v = ldg_stream(p + i * step);
            w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
        }
    }
}

constexpr int kWarps = 8, kThreads = 32 * kWarps;
// CTAs per SM, by the registers that a key group in flight takes.
template <int HD, bool Q8, int NT>
constexpr int kCtas = NT == 1 && (Q8 || HD <= 64) ? 2 : 1;

struct DecodePlan {
    int group;            // query heads per KV head
    uint64_t group_inv;   // ceil(2^32 / group): x / group = x * group_inv >> 32 for x below 2^32 / group
    uint32_t page_16;     // page stride in 16-byte units
    int page_log;
    float* part;          // [row tile][2 * CTAs][rows][HD + 4]: rows' states (NULL where a row tile has one CTA)
    int4* desc;           // [row tile][CTAs]: an item that starts in the CTA and ends in a later one
    int tile0;            // first row tile of the launch
    int ranks_log;        // of the clusters of the small variant
};

// Columns of an MMA: 8 rows (16-bit queries) or 4 (f32: hi and lo columns).
template <int HD, bool HILO, int NT>
struct Tile {
    static constexpr int kRowsPer = HILO ? 4 : 8;
    static constexpr int kRows = NT * kRowsPer;
    static constexpr int kLaneRows = HILO ? 1 : 2;  // rows per lane and column tile
    static constexpr int kPitch = HD + 4;           // floats of a row's state: values, log2 of their unit, sum, log2 of its unit
    static constexpr int kState = kRows * kPitch;
    // dynamic shared memory: the warps' two states, what they are, warp totals, groups before each sequence
    static constexpr int kMetaOff = 2 * kWarps * kState * 4;
    static constexpr int kScanOff = kMetaOff + 2 * kWarps * 16;
    static constexpr int kPreOff = kScanOff + 16 * 4;
    static size_t smem(int n_seq) { return kPreOff + size_t(n_seq + 1) * 4; }
    static size_t smem_small() { return kPreOff + size_t(kState) * 4; }  // the CTA's part in place of the groups
};

// What a row tile of a sequence sees, the same for all its KV heads.
struct Span {
    int row0, n, held, len, prefix, rows, pos_lo, pos_hi, hi, lo, g_lo, g_pre, ng;
};
template <int kRows>
__device__ __forceinline__ Span span_of(const neko_paged_attention_args& a, const DecodePlan& plan, int s, int tile) {
    Span v;
    v.row0 = a.q_start ? a.q_start[s] : s;
    v.n = a.q_start ? a.q_start[s + 1] - v.row0 : 1;
    v.held = max(a.kv_len[s], 0);
    v.len = min(v.held, a.cache.max_pages << plan.page_log);
    v.prefix = a.prefix ? min(max(a.prefix[s], 0), v.len) : 0;
    if (v.row0 < 0 || v.n < 0 || v.n > a.max_new || v.row0 + v.n > a.tokens) {
        set_op_error(kErrBadIndex);
        v.n = 0;
    }
    auto over_g = [&](int x) { return int(uint64_t(uint32_t(x)) * plan.group_inv >> 32); };
    const int r0 = tile * kRows;
    v.rows = max(min(v.n * plan.group - r0, kRows), 0);
    v.pos_lo = v.held - v.n + over_g(r0), v.pos_hi = v.held - v.n + over_g(r0 + max(v.rows, 1) - 1);
    // keys some row of the tile sees: [0, pre) and [lo, hi), as groups of 16
    v.hi = max(min(v.len, v.pos_hi + 1), 0);
    v.lo = a.window && v.pos_lo >= a.window ? min(v.pos_lo - a.window + 1, v.hi) : 0;
    const int g_hi = (max(v.hi, v.prefix > v.lo ? v.prefix : 0) + 15) / 16;
    v.g_lo = v.lo / 16;
    v.g_pre = min((v.prefix + 15) / 16, v.g_lo);  // prefix groups before g_lo
    // rows that see nothing still get a group, without a page, so that some CTA writes their zeros
    v.ng = v.rows > 0 ? max(v.g_pre + max(g_hi - v.g_lo, 0), 1) : 0;
    return v;
}

// log2 of a code's value where the scale is x: exact for powers of two, which the append writes.
__device__ __forceinline__ float log2_scale(float x) {
    const uint32_t b = __float_as_uint(x);
    float e = __uint_as_float(0x4b000000u | b >> 23) - (8388608.0f + 127.0f);  // 2^23 + the exponent's field
    if (b & 0x7fffffu) e = log2f(x);
    return fmaxf(e, -126.0f);
}
// What turns values in units of 2^top over a sum in units of 2^top_sum into the quotient (nothing seen: there are no values).
__device__ __forceinline__ float over_sum(float top, float sum, float top_sum) {
    return sum == 0.0f ? 0.0f : (top > -INFINITY ? exp2f(top - top_sum) : 1.0f) / sum;
}
// v * f to four values of a packed row of the output.
template <bool HILO>
__device__ __forceinline__ void put_row(const neko_paged_attention_args& a, const DecodePlan& plan, int row0, int kvh, int pr, int d,
                                        float4 v, float f) {
    const int rt = int(uint64_t(uint32_t(pr)) * plan.group_inv >> 32);
    const int64_t off = int64_t(row0 + rt) * a.o_token + int64_t(kvh * plan.group + pr - rt * plan.group) * a.o_head + d;
    const float x[4] = {v.x * f, v.y * f, v.z * f, v.w * f};
    auto store = [&](auto* p) { store_row<4>(p, (reinterpret_cast<uintptr_t>(p) & (sizeof(*p) * 4 - 1)) == 0, x); };
    if constexpr (HILO) store(static_cast<float*>(a.out) + off);
    else if (a.type == kTF16) store(static_cast<__half*>(a.out) + off);
    else store(static_cast<__nv_bfloat16*>(a.out) + off);
}

template <int HD, bool Q8, bool HILO, int NT, bool CL>
__global__ void __launch_bounds__(kThreads, kCtas<HD, Q8, NT>) paged_decode_kernel(const neko_paged_attention_args a,
                                                                                const DecodePlan plan) {
    using TL = Tile<HD, HILO, NT>;
    using W = Words<HD, Q8>;
    constexpr int kSteps = HD / 16;
    // Weights are 2^(score + log2 of the value scale - reference + kLift), at most 2^15. What f16 rounds off them, half of 2^-24
    // with hi + lo, is 2^-36 of the largest; the reference lags by 2^kLazy at most. A row's likeliest key times a block's scale
    // counts as no less than 2^kLeast of the reference.
    constexpr float kLazy = 4.0f, kLift = 11.0f, kLeast = -60.0f;
    constexpr float kNone = -3.0e38f;  // of what has seen nothing: a number, so that differences need no questions
    extern __shared__ __align__(16) float sm[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const neko_paged_cache& c = a.cache;
    const int tile = plan.tile0 + blockIdx.y, G = plan.group, n_kv = c.n_kv;
    uint8_t* smb = reinterpret_cast<uint8_t*>(sm);
    int4* meta = reinterpret_cast<int4*>(smb + TL::kMetaOff);  // item, 1 starts | 2 ends, row0, rows; item -1: none
    int* totals = reinterpret_cast<int*>(smb + TL::kScanOff);
    int* pre = reinterpret_cast<int*>(smb + TL::kPreOff);
    auto over_g = [&](int x) { return int(uint64_t(uint32_t(x)) * plan.group_inv >> 32); };

    // ---- this warp's equal share of the groups of 16 keys
    const int cta = blockIdx.x;
    int s = 0, kvh = 0, cnt = 1;
    int64_t total, warps, x = 0, x_end = 0;
    if (lane < 2) meta[2 * warp + lane].x = -1;
    __syncwarp();
    if constexpr (CL) {
        // of one item: the cluster's
        s = blockIdx.x >> plan.ranks_log, kvh = blockIdx.z;
        cnt = span_of<TL::kRows>(a, plan, s, tile).ng;
        total = cnt, warps = min(int64_t(kWarps) << plan.ranks_log, total);
        const int gw = (blockIdx.x & ((1 << plan.ranks_log) - 1)) * kWarps + warp;
        if (gw < warps) x = total * gw / warps, x_end = total * (gw + 1) / warps;
    } else {
        // of all (sequence, KV head) items', in order: groups before each sequence, added up
        int carry = 0;
        for (int base = 0; base < c.n_seq; base += kThreads) {
            const int sq = base + tid;
            int y = sq < c.n_seq ? span_of<TL::kRows>(a, plan, sq, tile).ng : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int z = __shfl_up_sync(0xffffffffu, y, o);
                if (lane >= o) y += z;
            }
            if (lane == 31) totals[warp] = y;
            __syncthreads();
            int before = carry;
#pragma unroll
            for (int w = 0; w < kWarps; w++) {
                if (w < warp) before += totals[w];
                carry += totals[w];
            }
            if (sq < c.n_seq) pre[sq + 1] = before + y;
            __syncthreads();
        }
        if (tid == 0) pre[0] = 0;
        __syncthreads();
        total = int64_t(carry) * n_kv;
        warps = max(min(int64_t(gridDim.x) * kWarps, total), int64_t(1));
        const int gw = cta * kWarps + warp;
        if (gw < warps) x = total * gw / warps, x_end = total * (gw + 1) / warps;
        if (x < x_end) {
            int a0 = 0, a1 = c.n_seq;  // pre[a0] * n_kv <= x < pre[a1] * n_kv
            while (a1 - a0 > 1) {
                const int mid = (a0 + a1) >> 1;
                if (int64_t(pre[mid]) * n_kv <= x) a0 = mid;
                else a1 = mid;
            }
            s = a0;
            cnt = pre[s + 1] - pre[s];
            kvh = int(uint32_t(x - int64_t(pre[s]) * n_kv) / uint32_t(cnt));
        }
    }
    int starts_last = -1;  // the CTA where the item that starts in this warp and does not end in it does
#pragma unroll 1
    while (x < x_end) {
        const int64_t item = CL ? 0 : int64_t(pre[s]) * n_kv + int64_t(kvh) * cnt;  // its first group
        const int k_begin = int(x - item), k_end = int(min(int64_t(cnt), x_end - item));
        const Span sp = span_of<TL::kRows>(a, plan, s, tile);
        const int row0 = sp.row0, n = sp.n, held = sp.held, len = sp.len, prefix = sp.prefix, rows = sp.rows;
        const int pos_lo = sp.pos_lo, pos_hi = sp.pos_hi, hi = sp.hi, lo = sp.lo, g_lo = sp.g_lo, g_pre = sp.g_pre;
        const int r0 = tile * TL::kRows;

        // ---- keys and values: fragments straight from the pages
        const int32_t* table = c.table + int64_t(s) * c.table_stride;
        constexpr int kB = Q8 ? 1 : 2;
        const int in_page = (1 << plan.page_log) - 1;
        const int64_t head_off = (int64_t(kvh) << plan.page_log) * HD * kB;
        const uint8_t* kp = static_cast<const uint8_t*>(c.k_pages) + head_off + g * W::kRow + t * (W::kK >= 4 ? 16 : W::kK * 4);
        const uint8_t* vp = static_cast<const uint8_t*>(c.v_pages) + head_off + 2 * t * W::kRow + g * (W::kV >= 4 ? 16 : W::kV * 4);
        const float *ksp = c.k_scale + kvh, *vsp = c.v_scale + kvh;
        auto key_of = [&](int k) { return 16 * (k < g_pre ? k : k - g_pre + g_lo); };  // first key of a group
        auto page_of = [&](int k) {
            const int slot = key_of(k) >> plan.page_log;
            const int p = k < k_end && slot < c.max_pages ? table[slot] : -1;
            return p < c.num_pages ? p : -1;
        };
        uint32_t kw[2][W::kK], vw[4][W::kV];
        float ks = 1.0f, vs = 1.0f;
        auto place = [&](int page, int j0) {
            return (uint64_t(uint32_t(page)) * plan.page_16 << 4) + uint32_t((j0 & in_page) * W::kRow);
        };
        auto load_k = [&](int page, int j0) {
            const uint8_t* p = kp + place(page, j0);
            load_words(p, 64, kw[0]);
            load_words(p + 8 * W::kRow, 64, kw[1]);
            if constexpr (Q8) ks = ksp[int64_t(page) * c.scale_stride];
        };
        auto load_v = [&](int page, int j0) {
            const uint8_t* p = vp + place(page, j0);
            load_words(p, 128, vw[0]);
            load_words(p + W::kRow, 128, vw[1]);
            load_words(p + 8 * W::kRow, 128, vw[2]);
            load_words(p + 9 * W::kRow, 128, vw[3]);
            if constexpr (Q8) vs = vsp[int64_t(page) * c.scale_stride];
        };
        // the V^T fragments of dims' tiles: word w gives one (f16) or two (8-bit) tiles of 16 dims
        auto v_frag = [&](int tile_i, uint32_t (&f)[4]) {
            if constexpr (Q8) {
                const int w = tile_i >> 1;
                const uint32_t sel = tile_i & 1 ? 0x7362u : 0x5140u;
                const uint32_t x = prmt(vw[0][w], vw[1][w], sel), y = prmt(vw[2][w], vw[3][w], sel);
                f[0] = e4m3x2_to_f16x2(uint16_t(x)), f[1] = e4m3x2_to_f16x2(uint16_t(x >> 16));
                f[2] = e4m3x2_to_f16x2(uint16_t(y)), f[3] = e4m3x2_to_f16x2(uint16_t(y >> 16));
            } else {
                f[0] = prmt(vw[0][tile_i], vw[1][tile_i], 0x5410u), f[1] = prmt(vw[0][tile_i], vw[1][tile_i], 0x7632u);
                f[2] = prmt(vw[2][tile_i], vw[3][tile_i], 0x5410u), f[3] = prmt(vw[2][tile_i], vw[3][tile_i], 0x7632u);
            }
        };
        // K and V of a group are in flight as soon as their registers are free: K of the next from the end of this one's
        // scores, V from the end of its P V. The first group's fly while the queries are read.
        int k = k_begin;
        int page = page_of(k), next_page = page_of(k + 1);
        if (page >= 0) {
            load_k(page, key_of(k));
            load_v(page, key_of(k));
        }

        // ---- queries as B fragments: for each step of 16 dims this lane's four of column g
        uint32_t qf[NT][kSteps][2];
        float qscale[NT][TL::kLaneRows];  // of this lane's score columns: scale * the row's power of two (* log2 e without a cap)
        int qpos[NT][TL::kLaneRows];
        float slope[NT][TL::kLaneRows];
        const float unit = a.softcap > 0.0f ? a.scale : a.scale * kLog2e;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int r = nt * TL::kRowsPer + (HILO ? g >> 1 : g);
            float q[kSteps][4];
            float most = 0.0f;
#pragma unroll
            for (int i = 0; i < kSteps; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) q[i][e] = 0.0f;
            if (r < rows) {
                const int rt = over_g(r0 + r);
                const int64_t off = int64_t(row0 + rt) * a.q_token + int64_t(kvh * G + r0 + r - rt * G) * a.q_head;
                auto fetch = [&](auto* p) {
                    const bool vec = (reinterpret_cast<uintptr_t>(p) & (sizeof(*p) * 4 - 1)) == 0;
#pragma unroll
                    for (int i = 0; i < kSteps; i++) {
                        // one word of an 8-bit row, two words of an f16 row
                        const int d = Q8 ? (W::kK >= 4 ? 64 * (i / 4) + 16 * t + 4 * (i % 4) : 8 * t + 4 * i) : 32 * (i / 2) + 8 * t + 4 * (i % 2);
                        load_row<4>(p + d, vec, q[i]);
                    }
                };
                if constexpr (HILO) fetch(static_cast<const float*>(a.q) + off);
                else if (a.type == kTF16) fetch(static_cast<const __half*>(a.q) + off);
                else fetch(static_cast<const __nv_bfloat16*>(a.q) + off);
#pragma unroll
                for (int i = 0; i < kSteps; i++)
#pragma unroll
                    for (int e = 0; e < 4; e++) most = fmaxf(most, finite_abs(q[i][e]));
            }
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
            const float up = row_up(most);
#pragma unroll
            for (int i = 0; i < kSteps; i++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    uint32_t hi2 = h2u(__floats2half2_rn(q[i][2 * h] * up, q[i][2 * h + 1] * up)), lo2 = 0;
                    if constexpr (HILO) split_hilo(q[i][2 * h] * up, q[i][2 * h + 1] * up, hi2, lo2);
                    qf[nt][i][h] = HILO && (g & 1) ? lo2 : hi2;
                }
            const float down = unit / up;
#pragma unroll
            for (int y = 0; y < TL::kLaneRows; y++) {
                const int rr = HILO ? t : 2 * t + y, r2 = nt * TL::kRowsPer + rr, rt = over_g(r0 + r2);
                qscale[nt][y] = __shfl_sync(0xffffffffu, down, (HILO ? 2 * rr : rr) * 4);
                qpos[nt][y] = r2 < rows ? held - n + rt : kNoRow;
                slope[nt][y] = a.slopes && r2 < rows ? a.slopes[kvh * G + r0 + r2 - rt * G] * kLog2e : 0.0f;
            }
        }

        float acc[NT][kSteps][4];
        float m[NT][TL::kLaneRows], l[NT][TL::kLaneRows];  // largest score and sum of the weights against it
        float u[NT][TL::kLaneRows];                        // reference less kLift: the accumulators' unit (8-bit values)
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
            for (int i = 0; i < kSteps; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) acc[nt][i][e] = 0.0f;
#pragma unroll
            for (int r = 0; r < TL::kLaneRows; r++) m[nt][r] = u[nt][r] = kNone, l[nt][r] = 0.0f;
        }
        const float inv_cap = a.softcap > 0.0f ? 1.0f / a.softcap : 0.0f;

#pragma unroll 1
        for (; k < k_end; k++) {
            const int j0 = key_of(k), j1 = key_of(k + 1);
            const int after = page_of(k + 2);
            if (page < 0) {
                page = next_page, next_page = after;
                if (page >= 0) {
                    load_k(page, j1);
                    load_v(page, j1);
                }
                continue;
            }
            // ---- scores
            float sc[NT][4];
#pragma unroll
            for (int i = 0; i < kSteps; i++) {
                uint32_t f[4];
                if constexpr (Q8) {
                    f[0] = e4m3x2_to_f16x2(uint16_t(kw[0][i])), f[1] = e4m3x2_to_f16x2(uint16_t(kw[1][i]));
                    f[2] = e4m3x2_to_f16x2(uint16_t(kw[0][i] >> 16)), f[3] = e4m3x2_to_f16x2(uint16_t(kw[1][i] >> 16));
                } else {
                    f[0] = kw[0][2 * i], f[1] = kw[1][2 * i], f[2] = kw[0][2 * i + 1], f[3] = kw[1][2 * i + 1];
                }
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    if (i == 0) mma16816_z(sc[nt], f, qf[nt][i][0], qf[nt][i][1]);
                    else mma16816(sc[nt], f, qf[nt][i][0], qf[nt][i][1]);
                }
            }
            const float ks_now = ks;
            page = next_page, next_page = after;
            if (page >= 0) load_k(page, j1);
            // ---- scale, cap, bias, masks
            // open: every key of the group is seen by every row of the tile
            const bool open = (j0 + 16 <= prefix) || (j0 + 15 <= pos_lo && j0 + 16 <= len && (!a.window || pos_hi - j0 < a.window));
            uint32_t seen_bits = 0;  // per lane: (nt, row, key) -> seen
            float z[NT][TL::kLaneRows][2];
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int r = 0; r < TL::kLaneRows; r++) {
                    const float f = qscale[nt][r] * ks_now;
#pragma unroll
                    for (int h = 0; h < 2; h++) z[nt][r][h] = (HILO ? sc[nt][2 * h] + sc[nt][2 * h + 1] : sc[nt][2 * h + r]) * f;
                }
            if (a.softcap > 0.0f) {
                float most = 0.0f;
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int r = 0; r < TL::kLaneRows; r++)
#pragma unroll
                        for (int h = 0; h < 2; h++) most = fmaxf(most, fabsf(z[nt][r][h] *= inv_cap));
                const bool small = __all_sync(0xffffffffu, most <= 0.5f);
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int r = 0; r < TL::kLaneRows; r++)
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const float y = z[nt][r][h];
                            z[nt][r][h] = a.softcap * kLog2e * (small || fabsf(y) <= 0.5f ? tanh_small(y) : tanh_abs(y));
                        }
            }
            if (a.slopes) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int r = 0; r < TL::kLaneRows; r++)
#pragma unroll
                        for (int h = 0; h < 2; h++) z[nt][r][h] = fmaf(slope[nt][r], float(j0 + g + 8 * h - qpos[nt][r]), z[nt][r][h]);
            }
            if (!open) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int r = 0; r < TL::kLaneRows; r++)
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const int j = j0 + g + 8 * h, at = qpos[nt][r];
                            const bool see = (j < len && j <= at && (!a.window || at - j < a.window)) || (j < prefix && at != kNoRow);
                            if (see) seen_bits |= 1u << (nt * 4 + r * 2 + h);
                            else z[nt][r][h] = -INFINITY;
                        }
            }
            // ---- running maxima (moved only by more than 2^kLazy: weights above 1 are as exact)
            const float lv = Q8 ? log2_scale(vs) : 0.0f;
            bool up = false;
            float top[NT][TL::kLaneRows];
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int r = 0; r < TL::kLaneRows; r++) {
                    float x = fmaxf(z[nt][r][0], z[nt][r][1]);
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                    top[nt][r] = x;
                    up |= x > m[nt][r] + kLazy || (Q8 && x + lv > u[nt][r] + (kLift + kLazy));
                }
            if (__any_sync(0xffffffffu, up)) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    float f[TL::kLaneRows];
#pragma unroll
                    for (int r = 0; r < TL::kLaneRows; r++) {
                        f[r] = 1.0f;
                        if (top[nt][r] > m[nt][r] + kLazy) {
                            const float fm = ex2(m[nt][r] - top[nt][r]);  // from kNone: 0
                            m[nt][r] = top[nt][r];
                            l[nt][r] *= fm;
                            if (!Q8) f[r] = fm;
                        }
                        if (Q8 && top[nt][r] + lv > u[nt][r] + (kLift + kLazy)) {
                            const float next = top[nt][r] + lv - kLift;
                            f[r] = ex2(u[nt][r] - next);
                            u[nt][r] = next;
                        }
                    }
#pragma unroll
                    for (int i = 0; i < kSteps; i++)
#pragma unroll
                        for (int e = 0; e < 4; e++) acc[nt][i][e] *= f[HILO ? 0 : e & 1];
                }
            }
            // ---- weights as B fragments
            uint32_t pf[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                float p[2][TL::kLaneRows];
#pragma unroll
                for (int r = 0; r < TL::kLaneRows; r++) {
                    // 2^vr: what a weight against the reference is of what it adds to the sum
                    const float vr = Q8 ? fmaxf(lv + (m[nt][r] - u[nt][r]), kLeast + kLift) : kLift, off = vr - m[nt][r];
                    p[0][r] = ex2(z[nt][r][0] + off), p[1][r] = ex2(z[nt][r][1] + off);
                    l[nt][r] = Q8 ? fmaf(p[0][r] + p[1][r], ex2(-vr), l[nt][r]) : l[nt][r] + (p[0][r] + p[1][r]);
                }
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    uint32_t hl;
                    if constexpr (HILO) {
                        const float x = p[h][0];
                        const __half hi1 = __float2half_rn(x);
                        hl = h2u(__halves2half2(hi1, __float2half_rn(x - __half2float(hi1))));
                    } else {
                        hl = h2u(__floats2half2_rn(p[h][0], p[h][1]));
                    }
                    pf[nt][h] = movmatrix(hl);
                }
            }
            // ---- P V
            if (!open) {
                // Values that no row of the tile sees are zeroed (they may hold anything); values that only some rows see
                // and that are not finite join the accumulators of the rows that see them, key by key.
                bool odd = false;
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const int j = j0 + 2 * t + (x & 1) + 8 * (x >> 1);
                    const bool dead = !((j < hi && j >= lo) || j < prefix);
#pragma unroll
                    for (int w = 0; w < W::kV; w++) {
                        if (dead) vw[x][w] = 0;
                        odd |= odd_lanes<Q8>(vw[x][w]) != 0;
                    }
                }
                if (__any_sync(0xffffffffu, odd)) {
#pragma unroll 1
                    for (int key = 0; key < 16; key++) {
                        // who sees this key: the lanes that hold its scores say so
                        const uint32_t bits = __shfl_sync(0xffffffffu, seen_bits, (key & 7) * 4 + t) >> (key >> 3);
                        const int mine = (key >> 3) * 2 + (key & 1);
                        const bool here = (key & 7) >> 1 == t;
                        uint32_t keep[4][W::kV];
#pragma unroll
                        for (int x = 0; x < 4; x++)
#pragma unroll
                            for (int w = 0; w < W::kV; w++) {
                                keep[x][w] = vw[x][w];
                                const uint32_t mask = here && x == mine ? odd_lanes<Q8>(vw[x][w]) : 0u;
                                vw[x][w] &= mask;
                                keep[x][w] &= ~mask;
                            }
#pragma unroll
                        for (int i = 0; i < kSteps; i++) {
                            uint32_t f[4];
                            v_frag(i, f);
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) {
                                float d[4];
                                mma16816_z(d, f, pf[nt][0], pf[nt][1]);
#pragma unroll
                                for (int e = 0; e < 4; e++) {
                                    const int r = HILO ? 0 : e & 1;
                                    if (bits >> (nt * 4 + r * 2) & 1u) acc[nt][i][e] += d[e];
                                }
                            }
                        }
#pragma unroll
                        for (int x = 0; x < 4; x++)
#pragma unroll
                            for (int w = 0; w < W::kV; w++) vw[x][w] = keep[x][w];
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < kSteps; i++) {
                uint32_t f[4];
                v_frag(i, f);
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    if constexpr (HILO) {
                        // added outside the MMA, which truncates: on the accumulator itself every group took 3e-8 off it
                        // (an error of 1.6e-5 on 150 x 18,000 keys, 6.4e-7 this way in the same time; 16-bit results do not see it)
                        float d[4];
                        mma16816_z(d, f, pf[nt][0], pf[nt][1]);
#pragma unroll
                        for (int e = 0; e < 4; e++) acc[nt][i][e] += d[e];
                    } else {
                        mma16816(acc[nt][i], f, pf[nt][0], pf[nt][1]);
                    }
                }
            }
            if (page >= 0) load_v(page, j1);
        }

        // ---- an item of this warp's own to the output, a part of one to shared memory
        const bool first = k_begin == 0, ends = k_end == cnt;
        float* st0 = sm + (2 * warp + first) * TL::kState;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
            for (int r = 0; r < TL::kLaneRows; r++) {
                float sum = l[nt][r];
                sum += __shfl_xor_sync(0xffffffffu, sum, 4);
                sum += __shfl_xor_sync(0xffffffffu, sum, 8);
                sum += __shfl_xor_sync(0xffffffffu, sum, 16);
                const int row = nt * TL::kRowsPer + (HILO ? t : 2 * t + r);
                float* st = st0 + row * TL::kPitch;
                if (g == 0) *reinterpret_cast<float4*>(st + HD) = make_float4(Q8 ? u[nt][r] : m[nt][r], sum, m[nt][r], 0.0f);
#pragma unroll
                for (int i = 0; i < kSteps; i++) {
                    float2 v;
                    v.x = HILO ? acc[nt][i][0] + acc[nt][i][1] : acc[nt][i][r];
                    v.y = HILO ? acc[nt][i][2] + acc[nt][i][3] : acc[nt][i][2 + r];
                    const int d = Q8 ? (HD / 8) * g + 2 * i : W::kV >= 4 ? 64 * (i / 4) + 8 * g + 2 * (i % 4) : 4 * g + 2 * i;
                    *reinterpret_cast<float2*>(st + d) = v;
                }
            }
        }
        __syncwarp();
        if (!CL && first && ends) {
            for (int y = lane; y < rows * (HD / 4); y += 32) {
                const int row = y / (HD / 4), d = y % (HD / 4) * 4;
                const float* st = st0 + row * TL::kPitch;
                const float4 of = *reinterpret_cast<const float4*>(st + HD);
                put_row<HILO>(a, plan, row0, kvh, r0 + row, d, *reinterpret_cast<const float4*>(st + d), over_sum(of.x, of.y, of.z));
            }
            __syncwarp();
        } else if (lane == 0) {
            meta[2 * warp + first] = make_int4(s * n_kv + kvh, (first ? 1 : 0) | (ends ? 2 : 0), row0, rows);
        }
        if (first && !ends) starts_last = int((((item + cnt) * warps - 1) / total) / kWarps);
        x = item + k_end;
        if (!CL && x < x_end && ++kvh == n_kv) {
            kvh = 0;
            do s++;
            while (pre[s + 1] == pre[s]);
            cnt = pre[s + 1] - pre[s];
        }
    }
    __syncthreads();
    if constexpr (CL) {
        // ---- the warps' parts joined in each CTA, the CTAs' over distributed shared memory, in order
        cg::cluster_group cluster = cg::this_cluster();
        const Span sp = span_of<TL::kRows>(a, plan, s, tile);
        const int ranks = 1 << plan.ranks_log, rank = blockIdx.x & (ranks - 1);
        float* mine = reinterpret_cast<float*>(smb + TL::kPreOff);
        auto join = [&](int row, int d, int parts, auto part, float& top, float& sum, float& top_sum) {
            top = top_sum = -INFINITY, sum = 0.0f;
            for (int i = 0; i < parts; i++)
                if (const float* st = part(i)) {
                    const float4 of = *reinterpret_cast<const float4*>(st + row * TL::kPitch + HD);
                    top = fmaxf(top, of.x), top_sum = fmaxf(top_sum, of.z);
                }
            const float ref = top == -INFINITY ? 0.0f : top, sum_ref = top_sum == -INFINITY ? 0.0f : top_sum;
            float4 v = make_float4(0, 0, 0, 0);
            for (int i = 0; i < parts; i++) {
                const float* st = part(i);
                if (!st) continue;
                st += row * TL::kPitch;
                const float4 o = *reinterpret_cast<const float4*>(st + d), of = *reinterpret_cast<const float4*>(st + HD);
                const float f = ex2(of.x - ref);
                sum = fmaf(ex2(of.z - sum_ref), of.y, sum);
                v.x = fmaf(f, o.x, v.x), v.y = fmaf(f, o.y, v.y), v.z = fmaf(f, o.z, v.z), v.w = fmaf(f, o.w, v.w);
            }
            return v;
        };
        for (int y = tid; y < sp.rows * (HD / 4); y += kThreads) {
            const int row = y / (HD / 4), d = y % (HD / 4) * 4;
            float top, sum, top_sum;
            const float4 v = join(row, d, 2 * kWarps, [&](int i) { return meta[i].x >= 0 ? sm + i * TL::kState : nullptr; }, top, sum, top_sum);
            if (ranks == 1) {
                put_row<HILO>(a, plan, sp.row0, kvh, tile * TL::kRows + row, d, v, over_sum(top, sum, top_sum));
            } else {
                *reinterpret_cast<float4*>(mine + row * TL::kPitch + d) = v;
                if (d == 0) *reinterpret_cast<float4*>(mine + row * TL::kPitch + HD) = make_float4(top, sum, top_sum, 0.0f);
            }
        }
        if (ranks == 1) return;
        cluster.sync();
        for (int y = rank * kThreads + tid; y < sp.rows * (HD / 4); y += kThreads * ranks) {
            const int row = y / (HD / 4), d = y % (HD / 4) * 4;
            float top, sum, top_sum;
            const float4 v = join(row, d, ranks, [&](int i) -> const float* { return cluster.map_shared_rank(mine, i); }, top, sum, top_sum);
            put_row<HILO>(a, plan, sp.row0, kvh, tile * TL::kRows + row, d, v, over_sum(top, sum, top_sum));
        }
        cluster.sync();  // no CTA leaves while another reads its part
        return;
    }
    // ---- parts of the same item joined over the warps, 32 pieces of four values a warp: to the output, or as one of this CTA's (at most
    // two) parts
    if (starts_last > cta && lane == 0) plan.desc[int64_t(tile) * gridDim.x + cta] = make_int4(s, kvh, starts_last, meta[2 * warp + 1].z);
    const int4 mine = lane < 2 * kWarps ? meta[lane] : make_int4(-1, 0, 0, 0);
    const uint32_t valid = __ballot_sync(0xffffffffu, mine.x >= 0);
    // lanes that hold the first part of an item here: the part before theirs belongs to another
    const uint32_t below = valid & ((1u << lane) - 1u);
    const int item_before = __shfl_sync(0xffffffffu, mine.x, below ? 31 - __clz(below) : lane);
    const uint32_t heads = __ballot_sync(0xffffffffu, mine.x >= 0 && (!below || item_before != mine.x));
    bool open_item = false;
    int turn = 0;  // 32 output pieces at a time go round the warps
    for (uint32_t left = heads; left; left &= left - 1) {  // the same in every warp
        const int b = __ffs(left) - 1;
        const uint32_t rest = left & (left - 1);
        const uint32_t in = valid & ~((1u << b) - 1u) & (rest ? (rest & (0u - rest)) - 1u : 0xffffffffu);
        const int last_part = 31 - __clz(in);
        const int flags = (__shfl_sync(0xffffffffu, mine.y, b) & 1) | (__shfl_sync(0xffffffffu, mine.y, last_part) & 2);
        open_item |= flags == 1;
        const int item_id = __shfl_sync(0xffffffffu, mine.x, b), row0 = __shfl_sync(0xffffffffu, mine.z, b), rows = __shfl_sync(0xffffffffu, mine.w, b);
        float* part = plan.part + ((int64_t(tile) * gridDim.x + cta) * 2 + (flags & 1)) * TL::kState;
        for (int y0 = 0; y0 < rows * (HD / 4); y0 += 32) {
            const int y = y0 + lane;
            if (turn++ % kWarps != warp || y >= rows * (HD / 4)) continue;
            const int row = y / (HD / 4), d = y % (HD / 4) * 4, at = row * TL::kPitch;
            float top = -INFINITY, top_sum = -INFINITY, sum = 0.0f;
            float4 v = make_float4(0, 0, 0, 0);
            for (uint32_t w = in; w;) {  // four parts at a time
                float uw[4], lw[4], mw[4];
                float4 o[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float* st = sm + (w ? __ffs(w) - 1 : b) * TL::kState + at;
                    const float4 of = *reinterpret_cast<const float4*>(st + HD);
                    uw[i] = w ? of.x : -INFINITY, lw[i] = of.y, mw[i] = w ? of.z : -INFINITY;
                    o[i] = *reinterpret_cast<const float4*>(st + d);
                    w &= w - 1;
                }
                const float now = fmaxf(top, fmaxf(fmaxf(uw[0], uw[1]), fmaxf(uw[2], uw[3])));
                const float now_sum = fmaxf(top_sum, fmaxf(fmaxf(mw[0], mw[1]), fmaxf(mw[2], mw[3])));
                const float ref = now == -INFINITY ? 0.0f : now, sum_ref = now_sum == -INFINITY ? 0.0f : now_sum, was = ex2(top - ref);
                sum *= ex2(top_sum - sum_ref), v.x *= was, v.y *= was, v.z *= was, v.w *= was;
                top = now, top_sum = now_sum;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float f = ex2(uw[i] - ref);
                    sum = fmaf(ex2(mw[i] - sum_ref), lw[i], sum);
                    v.x = fmaf(f, o[i].x, v.x), v.y = fmaf(f, o[i].y, v.y), v.z = fmaf(f, o[i].z, v.z), v.w = fmaf(f, o[i].w, v.w);
                }
            }
            if (flags == 3) {
                put_row<HILO>(a, plan, row0, item_id % n_kv, tile * TL::kRows + row, d, v, over_sum(top, sum, top_sum));
            } else {
                *reinterpret_cast<float4*>(part + at + d) = v;
                if (d == 0) *reinterpret_cast<float4*>(part + at + HD) = make_float4(top, sum, top_sum, 0.0f);
            }
        }
    }
    if (!open_item && tid == 0 && plan.desc) plan.desc[int64_t(tile) * gridDim.x + cta] = make_int4(-1, 0, 0, 0);
    pdl_trigger();
}

// Joins the parts of the items that several CTAs share, in their order: block x the item that starts in the decode
// kernel's CTA x.
template <int HD, bool HILO, int NT>
__global__ void __launch_bounds__(128) paged_join_kernel(const neko_paged_attention_args a, const DecodePlan plan, int ctas) {
    using TL = Tile<HD, HILO, NT>;
    pdl_wait();
    const int tile = blockIdx.y, cta = blockIdx.x;
    const int4 d4 = plan.desc[int64_t(tile) * ctas + cta];
    if (d4.x < 0) return;
    const int s = d4.x, kvh = d4.y, last = d4.z, row0 = d4.w;
    const int n = a.q_start ? a.q_start[s + 1] - row0 : 1;
    const int rows = min(n * plan.group - tile * TL::kRows, TL::kRows);
    const float* base = plan.part + (int64_t(tile) * ctas + cta) * 2 * TL::kState;
    // part 0 is the CTA's second slot, the others the first slots of the CTAs after it
    auto part = [&](int i) { return base + (i == 0 ? 1 : 2 * i) * int64_t(TL::kState); };
    const int parts = last - cta + 1;
    for (int y = threadIdx.x; y < rows * (HD / 4); y += 128) {
        const int row = y / (HD / 4), d = y % (HD / 4) * 4, at = row * TL::kPitch;
        float top = -INFINITY, top_sum = -INFINITY, sum = 0.0f;
        float4 v = make_float4(0, 0, 0, 0);
        for (int i0 = 0; i0 < parts; i0 += 8) {  // eight parts' loads in flight
            float uw[8], lw[8], mw[8];
            float4 o[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const bool in = i0 + i < parts;
                const float* p = part(in ? i0 + i : 0) + at;
                const float4 of = in ? *reinterpret_cast<const float4*>(p + HD) : make_float4(-INFINITY, 0.0f, -INFINITY, 0.0f);
                uw[i] = of.x, lw[i] = of.y, mw[i] = of.z;
                o[i] = in ? *reinterpret_cast<const float4*>(p + d) : make_float4(0, 0, 0, 0);
            }
            float now = top, now_sum = top_sum;
#pragma unroll
            for (int i = 0; i < 8; i++) now = fmaxf(now, uw[i]), now_sum = fmaxf(now_sum, mw[i]);
            const float ref = now == -INFINITY ? 0.0f : now, sum_ref = now_sum == -INFINITY ? 0.0f : now_sum, old = ex2(top - ref);
            sum *= ex2(top_sum - sum_ref), top = now, top_sum = now_sum;
            v.x *= old, v.y *= old, v.z *= old, v.w *= old;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float f = ex2(uw[i] - ref);
                sum = fmaf(ex2(mw[i] - sum_ref), lw[i], sum);
                v.x = fmaf(f, o[i].x, v.x), v.y = fmaf(f, o[i].y, v.y), v.z = fmaf(f, o[i].z, v.z), v.w = fmaf(f, o[i].w, v.w);
            }
        }
        put_row<HILO>(a, plan, row0, kvh, tile * TL::kRows + row, d, v, over_sum(top, sum, top_sum));
    }
}

// Few items of few keys: a cluster of CTAs each, about two groups of 16 keys for every warp, which need neither scratch memory
// nor the second kernel (one chat, 777 keys: 12 us a call, 8.4 on the GPU, against 16 and 10.4). 0: not that few, else the CTAs
// of a cluster. Where an SM holds one CTA, clusters of 8 find no room side by side (4: 13.8 us, 8: 23.3).
int small_ranks(int64_t items, int64_t per_item, int64_t room) {
    const int most = room > num_sms() ? 8 : 4;
    int ranks = 1;
    while (ranks < most && per_item > 16 * ranks && items * ranks * 2 <= room) ranks *= 2;
    return items * ranks <= room && per_item <= 64 * ranks ? ranks : 0;
}

template <int HD, bool Q8, bool HILO, int NT>
cudaError_t go(const neko_paged_attention_args& a, cudaStream_t st) {
    using TL = Tile<HD, HILO, NT>;
    const neko_paged_cache& c = a.cache;
    DecodePlan p;
    p.group = a.n_head / c.n_kv;
    p.group_inv = ((uint64_t(1) << 32) + p.group - 1) / p.group;
    p.page_16 = uint32_t(c.page_stride * (Q8 ? 1 : 2) / 16);
    p.page_log = 31 - __builtin_clz(c.page_size);
    p.ranks_log = 0;
    p.tile0 = 0;
    const int64_t row_tiles = (int64_t(a.max_new) * p.group + TL::kRows - 1) / TL::kRows;
    // as many CTAs for each row tile as the GPU holds at a time, or a group of 16 keys for each warp where the cache has room for
    // fewer. Prompts on heads of 32 have thousands of row tiles: no more than 16 times what the GPU holds in all, which bounds the
    // parts (40 MB, two states a CTA), and none where that is one CTA each.
    const int64_t groups = int64_t(c.max_pages) * c.page_size / 16 * c.n_kv * c.n_seq;
    const int64_t items = int64_t(c.n_kv) * c.n_seq;
    const int64_t per_item = int64_t(c.max_pages) * c.page_size / 16, room = int64_t(num_sms()) * kCtas<HD, Q8, NT>;
    const int ctas = int(std::max<int64_t>(1, std::min({room, std::max(groups, items) / kWarps, 16 * room / row_tiles})));
    const size_t part_bytes = size_t(row_tiles) * ctas * 2 * TL::kState * 4, desc_bytes = size_t(row_tiles) * ctas * sizeof(int4);
    if (const int ranks = c.n_kv <= 65535 ? small_ranks(items * row_tiles, per_item, room) : 0) {
        auto* small = paged_decode_kernel<HD, Q8, HILO, NT, true>;
        if (cudaError_t e = ensure_dyn_smem(small, TL::smem_small()); e != cudaSuccess) return e;
        p.ranks_log = 31 - __builtin_clz(ranks);
        p.part = nullptr, p.desc = nullptr;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(unsigned(c.n_seq * ranks), unsigned(row_tiles), unsigned(c.n_kv));
        cfg.blockDim = dim3(kThreads);
        cfg.dynamicSmemBytes = TL::smem_small();
        cfg.stream = st;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = unsigned(ranks);
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = ranks > 1 ? 1 : 0;
        return cudaLaunchKernelEx(&cfg, small, a, p);
    }
    auto* fn = paged_decode_kernel<HD, Q8, HILO, NT, false>;
    const size_t smem = TL::smem(c.n_seq);
    cudaError_t e = ensure_dyn_smem(fn, smem);
    if (e != cudaSuccess) return e;
    if (ctas == 1) {  // nothing is shared
        p.part = nullptr, p.desc = nullptr;
        for (int64_t left = row_tiles; left > 0 && e == cudaSuccess; left -= 65535, p.tile0 += 65535)
            e = launch_ex(fn, dim3(1, unsigned(std::min<int64_t>(left, 65535))), dim3(kThreads), smem, st, false, a, p);
        return e;
    }
    void* mem = nullptr;
    if ((e = scratch_alloc(&mem, part_bytes + desc_bytes, st)) != cudaSuccess) return e;
    p.part = static_cast<float*>(mem);
    p.desc = reinterpret_cast<int4*>(static_cast<char*>(mem) + part_bytes);
    e = launch_ex(fn, dim3(unsigned(ctas), unsigned(row_tiles)), dim3(kThreads), smem, st, false, a, p);
    if (e == cudaSuccess)
        e = launch_ex(paged_join_kernel<HD, HILO, NT>, dim3(unsigned(ctas), unsigned(row_tiles)), dim3(128), 0, st, true, a, p, ctas);
    cudaFreeAsync(mem, st);
    return e;
}

template <int HD, bool Q8>
cudaError_t by_rows(const neko_paged_attention_args& a, cudaStream_t st) {
    const int64_t rows = int64_t(a.max_new) * (a.n_head / a.cache.n_kv);
    if (a.type == NEKO_T_F32) return rows <= 4 ? go<HD, Q8, true, 1>(a, st) : go<HD, Q8, true, 2>(a, st);
    return rows <= 8 ? go<HD, Q8, false, 1>(a, st) : go<HD, Q8, false, 2>(a, st);
}

// Whether a row tile each of more items than SMs costs the tensor cores' kernel, which runs one CTA per SM, more in CTA starts
// than this kernel takes in all: both by measured costs in nanoseconds (a CTA's start, 128 keys; a row tile's pass, an item and its
// groups of 16 keys). f32 rows, 448 items: 32 rows on 24 keys 55 us there, 44 here, on 128 keys 57 and 64; 2,048 items:
// 20 rows on 64 keys 196 and 85, on 512 keys 301 and 315. Of 304 measured shapes the rule makes 79 faster, up to 2.9 times, and 6 of
// 160 items up to 17 % slower.
bool starts(int64_t items, int64_t rows, int64_t per_item, bool f32) {
    const int64_t rounds = (items + num_sms() - 1) / num_sms(), tile = f32 ? 8 : 16, tiles = (rows + tile - 1) / tile;
    if (rounds == 1 || rows > 128) return false;
    const int64_t there = 5000 + rounds * (8000 + (per_item + 7) / 8 * (f32 ? 3400 : 2300));
    const int64_t here = 12000 + tiles * ((f32 ? 3000 : 2000) + items * (per_item + 5) * (f32 ? 13 : 18) / 10);
    return here < there;
}

}  // namespace

cudaError_t launch_paged_attention(const neko_paged_attention_args& a, cudaStream_t st) {
    // Rows past 16 go to the tensor cores' kernel (8 x 4,000 f16 keys, f32 rows: 16 rows 61 us each way, 20 rows 62 against 90),
    // but not where this one's small variant takes them (64 rows on 600 keys: 12 us against 22) nor up to 32 rows on many 8-bit
    // keys, which that one would convert for few rows (48 x 2,000 keys: 252 us against 316, 16-bit rows 139 against 277; of fewer
    // than 8,192 groups of 16 keys, 5,000 keys: 43 against 35), nor many short contexts: starts() below. Head dim 32 stays here.
    const neko_paged_cache& c = a.cache;
    const int64_t rows = int64_t(a.max_new) * (a.n_head / c.n_kv), items = int64_t(c.n_seq) * c.n_kv;
    if (rows > kPromptRows && c.head_dim >= 64) {
        const int64_t per_item = int64_t(c.max_pages) * c.page_size / 16, tile = a.type == NEKO_T_F32 ? 8 : 16;
        const bool many = c.type == NEKO_T_E4M3 && rows <= 2 * kPromptRows && items * per_item >= 8192;
        if (!many && !small_ranks(items * ((rows + tile - 1) / tile), per_item, num_sms()) &&
            !starts(items, rows, per_item, a.type == NEKO_T_F32))
            return launch_paged_prompt(a, st);
    }
    const bool q8 = a.cache.type == NEKO_T_E4M3;
    switch (a.cache.head_dim) {
        case 32: return q8 ? by_rows<32, true>(a, st) : by_rows<32, false>(a, st);
        case 64: return q8 ? by_rows<64, true>(a, st) : by_rows<64, false>(a, st);
        default: return q8 ? by_rows<128, true>(a, st) : by_rows<128, false>(a, st);
    }
}

}  // namespace neko
