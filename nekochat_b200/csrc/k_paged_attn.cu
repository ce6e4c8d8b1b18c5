// Attention of few query rows over a paged cache (neko_op_paged_attention): decode steps, short continuations and,
// one tile of rows after the other, anything else.
//
// The packed rows of a (sequence, KV head) are its new tokens times the G query heads that share the KV head, so a key
// is read once for all of them. Every warp owns groups of 16 keys and works alone (no barrier until the end): scores
// S^T = K q^T and O^T += V^T P^T on mma.sync m16n8k16 with keys / head dims as the MMA's 16 rows and the query rows as
// its 8 columns. The order of the summed index is free as long as both operands agree, so the fragments come straight
// from global memory: lane (g, t) holds, for K, 16-byte pieces t, t + 4, .. of key rows g and g + 8, and for V the
// pieces g, g + 8, .. of key rows 2t, 2t + 1, 2t + 8, 2t + 9; neither K nor V passes through shared memory. 8-bit codes
// become f16 in registers (exact), keys' scales multiply the scores, values' scales the group's P V before it joins
// the f32 accumulator. P reaches the second product by transposing 8 x 8 tiles in registers (movmatrix).
// f32 queries are two columns each, f16 hi and lo (22 bits; scores are the columns' sum), and so are their weights P;
// 16-bit queries one exact f16 column, weights one f16. Rows are scaled by a power of two into f16's range first.
// Each warp keeps its own running maximum and sum; warps meet in shared memory at the end, and the CTAs that share a
// (sequence, KV head) form a thread-block cluster and meet over distributed shared memory, in rank order, so no
// scratch memory is needed and results do not depend on timing.
#include <cooperative_groups.h>

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

// CTAs of 8 warps per SM, by the registers that a key group in flight takes.
template <int kWarps, int HD, bool Q8, int NT>
constexpr int kCtas = kWarps == 16 ? 1 : NT == 1 && (Q8 || HD <= 64) ? 2 : 1;

struct DecodePlan {
    int ranks_log;        // log2 of the CTAs per (sequence, KV head, row tile): the cluster
    int group;            // query heads per KV head
    uint64_t group_inv;   // ceil(2^32 / group): x / group = x * group_inv >> 32 for x below 2^32 / group
    uint32_t page_16;     // page stride in 16-byte units
    int page_log;
};

// Columns of an MMA: 8 rows (16-bit queries) or 4 (f32: hi and lo columns).
template <int HD, bool Q8, bool HILO, int NT, int kWarps>
struct Tile {
    static constexpr int kRowsPer = HILO ? 4 : 8;
    static constexpr int kRows = NT * kRowsPer;
    static constexpr int kLaneRows = HILO ? 1 : 2;  // rows per lane and column tile
    static constexpr int kPitch = HD + 4;
    // dynamic shared memory (floats): per warp and row maximum, sum, accumulator; then the CTA's
    static constexpr int kState = kRows * (kPitch + 2);
    static constexpr size_t kSmem = size_t(kWarps + 1) * kState * 4;
};

template <int HD, bool Q8, bool HILO, int NT, int kWarps>
__global__ void __launch_bounds__(32 * kWarps, kCtas<kWarps, HD, Q8, NT>) paged_decode_kernel(
    const neko_paged_attention_args a, const DecodePlan plan) {
    using TL = Tile<HD, Q8, HILO, NT, kWarps>;
    using W = Words<HD, Q8>;
    constexpr int kSteps = HD / 16;
    extern __shared__ __align__(16) float sm[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const neko_paged_cache& c = a.cache;
    const int ranks = 1 << plan.ranks_log;
    const int rank = blockIdx.x & (ranks - 1), s = blockIdx.x >> plan.ranks_log, kvh = blockIdx.y, tile = blockIdx.z;
    const int G = plan.group;
    auto over_g = [&](int x) { return int(uint64_t(uint32_t(x)) * plan.group_inv >> 32); };

    // the sequence: everything below is the same for all CTAs of the cluster
    const int row0 = a.q_start ? a.q_start[s] : s;
    const int n = a.q_start ? a.q_start[s + 1] - row0 : 1;
    const int held = max(a.kv_len[s], 0), len = min(held, c.max_pages << plan.page_log);
    const int prefix = a.prefix ? min(max(a.prefix[s], 0), len) : 0;
    if (row0 < 0 || n < 0 || n > a.max_new || row0 + n > a.tokens) {
        if (tid == 0) set_device_error(kErrBadIndex);
        return;
    }
    const int r0 = tile * TL::kRows;  // first packed row of this tile
    const int rows = min(n * G - r0, TL::kRows);
    if (rows <= 0) return;
    const int pos_lo = held - n + over_g(r0), pos_hi = held - n + over_g(r0 + rows - 1);
    // keys some row of the tile sees: [0, pre) and [lo, hi), as groups of 16
    const int hi = max(min(len, pos_hi + 1), 0);
    const int lo = a.window ? min(max(pos_lo - a.window + 1, 0), hi) : 0;
    const int g_lo = lo / 16, g_hi = (max(hi, prefix > lo ? prefix : 0) + 15) / 16;
    const int g_pre = min((prefix + 15) / 16, g_lo);  // prefix groups before g_lo
    const int ng = g_pre + max(g_hi - g_lo, 0);
    const int k_begin = int(int64_t(ng) * rank >> plan.ranks_log), k_end = int(int64_t(ng) * (rank + 1) >> plan.ranks_log);

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
    int k = k_begin + warp;
    int page = page_of(k), next_page = page_of(k + kWarps);
    if (page >= 0) {
        load_k(page, key_of(k));
        load_v(page, key_of(k));
    }

    // ---- queries as B fragments
    uint32_t qf[NT][kSteps][2];
    float qscale[NT][TL::kLaneRows];  // of this lane's score columns: scale * the row's power of two (* log2 e without a cap)
    int qpos[NT][TL::kLaneRows];
    float slope[NT][TL::kLaneRows];
    const float unit = a.softcap > 0.0f ? a.scale : a.scale * kLog2e;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        const int r = r0 + nt * TL::kRowsPer + (HILO ? g >> 1 : g);
        float x[kSteps][4];
        float most = 0.0f;
#pragma unroll
        for (int i = 0; i < kSteps; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) x[i][e] = 0.0f;
        if (r < n * G) {
            const int rt = over_g(r);
            const int64_t off = int64_t(row0 + rt) * a.q_token + int64_t(kvh * G + r - rt * G) * a.q_head;
            auto fetch = [&](auto* p) {
                const bool vec = (reinterpret_cast<uintptr_t>(p) & (sizeof(*p) * 4 - 1)) == 0;
#pragma unroll
                for (int i = 0; i < kSteps; i++) {
                    // the four dims of step i: one word of an 8-bit row, two words of an f16 row
                    const int d = Q8 ? (W::kK >= 4 ? 64 * (i / 4) + 16 * t + 4 * (i % 4) : 8 * t + 4 * i)
                                     : 32 * (i / 2) + 8 * t + 4 * (i % 2);
                    load_row<4>(p + d, vec, x[i]);
                }
            };
            if constexpr (HILO) fetch(static_cast<const float*>(a.q) + off);
            else if (a.type == kTF16) fetch(static_cast<const __half*>(a.q) + off);
            else fetch(static_cast<const __nv_bfloat16*>(a.q) + off);
#pragma unroll
            for (int i = 0; i < kSteps; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) most = fmaxf(most, finite_abs(x[i][e]));
        }
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        const float up = row_up(most);
#pragma unroll
        for (int i = 0; i < kSteps; i++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                uint32_t hi2, lo2;
                split_hilo(x[i][2 * h] * up, x[i][2 * h + 1] * up, hi2, lo2);
                qf[nt][i][h] = HILO && (g & 1) ? lo2 : hi2;
            }
        const float down = unit / up;
#pragma unroll
        for (int x2 = 0; x2 < TL::kLaneRows; x2++) {
            const int rr = HILO ? t : 2 * t + x2;  // this lane's score row within the column tile
            qscale[nt][x2] = __shfl_sync(0xffffffffu, down, (HILO ? 2 * rr : rr) * 4);
            const int pr = r0 + nt * TL::kRowsPer + rr, rt = over_g(pr);
            qpos[nt][x2] = pr < n * G ? held - n + rt : kNoRow;
            slope[nt][x2] = a.slopes && pr < n * G ? a.slopes[kvh * G + pr - rt * G] * kLog2e : 0.0f;
        }
    }

    float acc[NT][kSteps][4];
    float m[NT][TL::kLaneRows], l[NT][TL::kLaneRows];
    float vref = 0.0f;  // the value scale that the accumulators are in units of
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
        for (int i = 0; i < kSteps; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) acc[nt][i][e] = 0.0f;
#pragma unroll
        for (int r = 0; r < TL::kLaneRows; r++) m[nt][r] = -INFINITY, l[nt][r] = 0.0f;
    }
    const float inv_cap = a.softcap > 0.0f ? 1.0f / a.softcap : 0.0f;

    for (; k < k_end; k += kWarps) {
        const int j0 = key_of(k), j1 = key_of(k + kWarps);
        const int after = page_of(k + 2 * kWarps);
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
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int r = 0; r < TL::kLaneRows; r++)
#pragma unroll
                    for (int h = 0; h < 2; h++) z[nt][r][h] = a.softcap * kLog2e * tanh_abs(z[nt][r][h] * inv_cap);
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
        // ---- running maximum (moved only by more than 2^8: weights up to that are as exact) and value scale
        const float vs_now = vs;
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
                up |= x > m[nt][r] + 8.0f;
            }
        const bool v_up = Q8 && vs_now > 16.0f * vref;
        if (__any_sync(0xffffffffu, up) || v_up) {
            float fv = 1.0f;
            if (v_up) {
                fv = __fdividef(vref, vs_now);
                vref = vs_now;
            }
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                float f[TL::kLaneRows];
#pragma unroll
                for (int r = 0; r < TL::kLaneRows; r++) {
                    f[r] = 1.0f;
                    if (top[nt][r] > m[nt][r] + 8.0f) {
                        f[r] = ex2(m[nt][r] - top[nt][r]);  // from -inf: 0
                        m[nt][r] = top[nt][r];
                        l[nt][r] *= f[r];
                    }
                    f[r] *= fv;
                }
#pragma unroll
                for (int i = 0; i < kSteps; i++)
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[nt][i][e] *= f[HILO ? 0 : e & 1];
            }
        }
        // ---- weights as B fragments, in units of the reference scale
        uint32_t pf[NT][2];
        const float ratio = Q8 ? (vref > 0.0f ? __fdividef(vs_now, vref) : 0.0f) : 1.0f;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            float p[2][TL::kLaneRows];
#pragma unroll
            for (int r = 0; r < TL::kLaneRows; r++) {
                const float ref = m[nt][r] == -INFINITY ? 0.0f : m[nt][r];
                p[0][r] = ex2(z[nt][r][0] - ref), p[1][r] = ex2(z[nt][r][1] - ref);
                l[nt][r] += p[0][r] + p[1][r];
            }
#pragma unroll
            for (int h = 0; h < 2; h++) {
                uint32_t hl;
                if constexpr (HILO) {
                    const float x = p[h][0] * ratio;
                    const __half hi1 = __float2half_rn(x);
                    hl = h2u(__halves2half2(hi1, __float2half_rn(x - __half2float(hi1))));
                } else {
                    hl = h2u(__floats2half2_rn(p[h][0] * ratio, p[h][1] * ratio));
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
            for (int nt = 0; nt < NT; nt++) mma16816(acc[nt][i], f, pf[nt][0], pf[nt][1]);
        }
        if (page >= 0) load_v(page, j1);
    }

    // ---- the warps' states to shared memory: [row](max, sum, values)
    float* mine = sm + warp * TL::kState;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
        for (int r = 0; r < TL::kLaneRows; r++) {
            float sum = l[nt][r];
            sum += __shfl_xor_sync(0xffffffffu, sum, 4);
            sum += __shfl_xor_sync(0xffffffffu, sum, 8);
            sum += __shfl_xor_sync(0xffffffffu, sum, 16);
            const int row = nt * TL::kRowsPer + (HILO ? t : 2 * t + r);
            float* st = mine + row * (TL::kPitch + 2);
            if (g == 0) st[0] = m[nt][r], st[1] = sum;
#pragma unroll
            for (int i = 0; i < kSteps; i++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const float v = (HILO ? acc[nt][i][2 * h] + acc[nt][i][2 * h + 1] : acc[nt][i][2 * h + r]) * (Q8 ? vref : 1.0f);
                    const int d = Q8 ? (HD / 8) * g + 2 * i + h
                                     : (W::kV >= 4 ? 64 * (i / 4) + 8 * g + 2 * (i % 4) + h : 4 * g + 2 * i + h);
                    st[2 + d] = v;
                }
        }
    }
    __syncthreads();
    // ---- joined over the warps
    const bool alone = ranks == 1;
    float* cta = sm + kWarps * TL::kState;
    auto put = [&](int row, int d, float v) {
        const int pr = r0 + row, rt = over_g(pr);
        const int64_t off = int64_t(row0 + rt) * a.o_token + int64_t(kvh * G + pr - rt * G) * a.o_head + d;
        if (a.type == kTF32) static_cast<float*>(a.out)[off] = v;
        else if (a.type == kTF16) static_cast<__half*>(a.out)[off] = __float2half_rn(v);
        else static_cast<__nv_bfloat16*>(a.out)[off] = __float2bfloat16_rn(v);
    };
    auto join = [&](int row, int d, int count, auto state, float& top, float& sum) {
        top = -INFINITY;
        for (int w = 0; w < count; w++) top = fmaxf(top, state(w)[0]);
        const float ref = top == -INFINITY ? 0.0f : top;
        sum = 0.0f;
        float v = 0.0f;
        for (int w = 0; w < count; w++) {
            const float* st = state(w);
            const float f = ex2(st[0] - ref);
            sum += f * st[1];
            v += f * st[2 + d];
        }
        return v;
    };
    for (int x = tid; x < rows * HD; x += 32 * kWarps) {
        const int row = x / HD, d = x % HD;
        float top, sum;
        const float v = join(row, d, kWarps, [&](int w) { return sm + w * TL::kState + row * (TL::kPitch + 2); }, top, sum);
        if (alone) {
            put(row, d, sum == 0.0f ? 0.0f : v / sum);
        } else {
            float* st = cta + row * (TL::kPitch + 2);
            if (d == 0) st[0] = top, st[1] = sum;
            st[2 + d] = v;
        }
    }
    if (alone) return;
    // ---- joined over the cluster, each CTA a share of the outputs
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    const int share = (rows * HD + ranks - 1) >> plan.ranks_log;
    for (int x = rank * share + tid; x < min(rows * HD, (rank + 1) * share); x += 32 * kWarps) {
        const int row = x / HD, d = x % HD;
        float top, sum;
        const float v = join(row, d, ranks,
                             [&](int w) { return cluster.map_shared_rank(cta, w) + row * (TL::kPitch + 2); }, top, sum);
        put(row, d, sum == 0.0f ? 0.0f : v / sum);
    }
    cluster.sync();  // no CTA leaves while another reads its state
}

template <int HD, bool Q8, bool HILO, int NT, int kWarps>
cudaError_t go(const neko_paged_attention_args& a, int ranks, cudaStream_t st) {
    using TL = Tile<HD, Q8, HILO, NT, kWarps>;
    const neko_paged_cache& c = a.cache;
    DecodePlan p;
    p.group = a.n_head / c.n_kv;
    p.group_inv = ((uint64_t(1) << 32) + p.group - 1) / p.group;
    p.ranks_log = 31 - __builtin_clz(ranks);
    p.page_16 = uint32_t(c.page_stride * (Q8 ? 1 : 2) / 16);
    p.page_log = 31 - __builtin_clz(c.page_size);
    const int64_t row_tiles = (int64_t(a.max_new) * p.group + TL::kRows - 1) / TL::kRows;
    if (row_tiles > 65535 || c.n_kv > 65535 || int64_t(c.n_seq) * ranks > 0x7fffffff) return cudaErrorInvalidConfiguration;
    auto* fn = paged_decode_kernel<HD, Q8, HILO, NT, kWarps>;
    cudaError_t e = ensure_dyn_smem(fn, TL::kSmem);
    if (e != cudaSuccess) return e;
    if (ranks > 8 && (e = cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1)) != cudaSuccess)
        return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(c.n_seq * ranks), unsigned(c.n_kv), unsigned(row_tiles));
    cfg.blockDim = dim3(32 * kWarps);
    cfg.dynamicSmemBytes = TL::kSmem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = unsigned(ranks);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ranks > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, fn, a, p);
}

// CTAs that share a (sequence, KV head, row tile): enough for two CTAs of 8 warps on every SM, as long as each warp
// keeps two groups of 16 keys. Where 16 of them do not fill the GPU, CTAs of 16 warps.
template <int HD, bool Q8, bool HILO, int NT>
cudaError_t by_work(const neko_paged_attention_args& a, cudaStream_t st) {
    const neko_paged_cache& c = a.cache;
    const int64_t rows = int64_t(a.max_new) * (a.n_head / c.n_kv), kRows = Tile<HD, Q8, HILO, NT, 8>::kRows;
    const int64_t items = int64_t(c.n_seq) * c.n_kv * ((rows + kRows - 1) / kRows);
    const int64_t groups = int64_t(c.max_pages) * c.page_size / 16;
    int ranks = 1;
    while (ranks < 16 && items * ranks < 2 * num_sms() && groups > 16 * ranks) ranks *= 2;
    if (NT == 1 && ranks == 16 && items * 16 <= num_sms() && groups > 32 * ranks)
        return go<HD, Q8, HILO, NT, NT == 1 ? 16 : 8>(a, ranks, st);
    return go<HD, Q8, HILO, NT, 8>(a, ranks, st);
}

template <int HD, bool Q8>
cudaError_t by_rows(const neko_paged_attention_args& a, cudaStream_t st) {
    const int64_t rows = int64_t(a.max_new) * (a.n_head / a.cache.n_kv);
    if (a.type == NEKO_T_F32) return rows <= 4 ? by_work<HD, Q8, true, 1>(a, st) : by_work<HD, Q8, true, 2>(a, st);
    return rows <= 8 ? by_work<HD, Q8, false, 1>(a, st) : by_work<HD, Q8, false, 2>(a, st);
}

}  // namespace

cudaError_t launch_paged_attention(const neko_paged_attention_args& a, cudaStream_t st) {
    const int64_t rows = int64_t(a.max_new) * (a.n_head / a.cache.n_kv);
    if (rows > kPromptRows && a.cache.head_dim >= 64) return launch_paged_prompt(a, st);
    const bool q8 = a.cache.type == NEKO_T_E4M3;
    switch (a.cache.head_dim) {
        case 32: return q8 ? by_rows<32, true>(a, st) : by_rows<32, false>(a, st);
        case 64: return q8 ? by_rows<64, true>(a, st) : by_rows<64, false>(a, st);
        default: return q8 ? by_rows<128, true>(a, st) : by_rows<128, false>(a, st);
    }
}

}  // namespace neko
