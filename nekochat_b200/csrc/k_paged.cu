// Appending keys and values to a paged cache (neko_op_paged_append): per-head RMSNorm of q and k, rotary position
// embedding, one rounding to the cache's type. The engine's counterpart is rope.comp + kv_store.comp on a contiguous
// f16 cache (qwen3_model.cpp:249-254, cpu_ops.cpp:513-542); pages, 8-bit blocks, partial and interleaved rotations
// have none.
//
// A unit of work is the (at most page_size) new tokens that one sequence puts into one page, for one head of q, k or
// v: an 8-bit block's scale depends on all of them, so one owner sees them all, holds them in registers and needs no
// atomics.
//  * Steps (a few new tokens per sequence): a warp per unit, head_dim / 32 consecutive values a lane; latency is all.
//  * Prompts: a CTA per (sequence, page) and group of heads. A lane holds eight values of a token, both members of four
//    rotation pairs, so the rotation needs no exchange and its cosines stay in registers from head to head; the next
//    head's values fly while this one's are worked on. Ragged prompts of 14,364 bf16 tokens, 32 + 16 heads of 128, 8-bit
//    cache: 94 us, 3.5 TB/s (55 % of the measured copy rate; issue slots bound it: 136 warp instructions a row at first,
//    packed f32 pairs and eight values a lane since); 4,001 f32 tokens, f16 cache: 15 us, 4.1 TB/s.
#include <algorithm>
#include <type_traits>

#include "paged.cuh"
#include "paged_math.cuh"

namespace neko {

namespace {

// Starts count as no more than this: no page and no row of the rotation table is there, and positions stay within 31 bits (the
// new tokens of a call are fewer than 2^24, 65,535 pages).
constexpr int kFarthest = 1 << 30;

constexpr int kFewTokens = 4;  // tokens of a unit in the step kernel

constexpr int kSlots = 4;  // tokens of a lane in the prompt kernel (2: 32 warps per SM instead of 16, 115 us against 92 on ragged prompts)

struct AppendPlan {
    int units;    // head rows: n_head + 2 n_kv (n_head = 0 without q)
    int per_cta;  // of them for one CTA
    int page_log;
};

// x c + y s, the same bits in both kernels.
__device__ __forceinline__ float turned(float x, float y, float c, float s) { return __fmaf_rn(x, c, __fmul_rn(y, s)); }

// The smallest power of two (at least 2^-100) with which `most` is at most 448 = 1.75 * 2^8.
__device__ __forceinline__ float block_scale(float most) {
    const uint32_t bits = __float_as_uint(most);
    const int e = int(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return __uint_as_float(uint32_t(max(e, kScaleMinExp) + 127) << 23);
}
// Codes that a block held before, times a ratio of scales (a power of two below 1).
__device__ __forceinline__ void recode(uint8_t* blk, int count, float ratio, int thread, int threads) {
    uint32_t* w = reinterpret_cast<uint32_t*>(blk);
    for (int k = thread; k < count / 4; k += threads) {
        const uint32_t v = w[k], f0 = e4m3x2_to_f16x2(uint16_t(v)), f1 = e4m3x2_to_f16x2(uint16_t(v >> 16));
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&f0)), b = __half22float2(*reinterpret_cast<const __half2*>(&f1));
        w[k] = uint32_t(f32x2_to_e4m3x2(a.x * ratio, a.y * ratio)) | uint32_t(f32x2_to_e4m3x2(b.x * ratio, b.y * ratio)) << 16;
    }
}

template <typename T, int HD, bool Q8>
__global__ void __launch_bounds__(128) paged_append_step_kernel(const neko_paged_append_args a, const AppendPlan plan) {
    constexpr int E = HD / 32;  // values per lane and token
    const int lane = threadIdx.x & 31;
    const int unit = blockIdx.y * 4 + (threadIdx.x >> 5), s = blockIdx.x, chunk = blockIdx.z;
    if (unit >= plan.units) return;

    const neko_paged_cache& c = a.cache;
    const int row0 = a.q_start ? a.q_start[s] : s;
    const int n = a.q_start ? a.q_start[s + 1] - row0 : 1;
    const int start = min(a.start[s], kFarthest);
    if (row0 < 0 || n < 0 || n > a.max_new || row0 + n > a.tokens) {  // outside the planned rows
        if (lane == 0) set_op_error(kErrBadIndex);
        return;
    }
    const bool live = start >= 0;
    const int ps = c.page_size;
    // token range [i0, i1) of this unit
    const int first = live ? start >> plan.page_log : 0, off0 = live ? start & (ps - 1) : 0;
    const int i0 = max(0, chunk * ps - off0), i1 = min(n, (chunk + 1) * ps - off0);
    if (i0 >= i1) return;
    const int slot = first + chunk;
    const int page = live && slot < c.max_pages ? c.table[int64_t(s) * c.table_stride + slot] : -1;
    const int nh = a.q ? a.n_head : 0;
    const int kind = unit < nh ? 0 : unit < nh + c.n_kv ? 1 : 2;  // q, k, v
    const int head = kind == 0 ? unit : kind == 1 ? unit - nh : unit - nh - c.n_kv;
    const T* src = static_cast<const T*>(kind == 0 ? a.q : kind == 1 ? a.k : a.v);
    const int64_t ts = kind == 0 ? a.q_token : kind == 1 ? a.k_token : a.v_token;
    const int64_t hs = kind == 0 ? a.q_head : kind == 1 ? a.k_head : a.v_head;
    src += int64_t(head) * hs + lane * E;
    const bool vec = ((reinterpret_cast<uintptr_t>(src) | (uintptr_t(ts) * sizeof(T))) & (sizeof(T) * E - 1)) == 0;
    const float* gain = kind == 0 ? a.q_gain : kind == 1 ? a.k_gain : nullptr;
    const bool turn = kind != 2 && a.rot > 0;

    // every token's values, in registers
    float x[kFewTokens][E];
#pragma unroll
    for (int r = 0; r < kFewTokens; r++) {
        if (i0 + r < i1) load_row<E>(src + int64_t(row0 + i0 + r) * ts, vec, x[r]);
        else
#pragma unroll
            for (int e = 0; e < E; e++) x[r][e] = 0.0f;
    }
    float g[E];
    if (gain) load_row<E>(gain + lane * E, false, g);
    float old = 0.0f;
    float* sp = nullptr;
    const int o0 = chunk == 0 ? off0 : 0;  // the first new token's place in the page
    const bool resident = page >= 0 && page < c.num_pages;
    if (Q8 && kind != 0 && resident) {
        sp = (kind == 1 ? c.k_scale : c.v_scale) + int64_t(page) * c.scale_stride + head;
        if (o0 > 0) old = *sp;
    }

    const int half = a.rot >> 1;
    // this lane's first rotation index and its partner lane
    const int d0 = lane * E;
    const bool in_rot = turn && d0 < a.rot;
    const int j0 = a.interleaved ? d0 >> 1 : d0 < half ? d0 : d0 - half;
    const bool upper = a.interleaved ? (E == 1 && (lane & 1)) : d0 >= half;
    const int partner = a.interleaved ? (E == 1 ? lane ^ 1 : lane) : in_rot ? (upper ? lane - half / E : lane + half / E) : lane;

#pragma unroll
    for (int r = 0; r < kFewTokens; r++) {
        const int i = i0 + r;
        if (i >= i1) break;  // uniform over the warp
        if (gain) {
            float ss = 0.0f;
#pragma unroll
            for (int e = 0; e < E; e++) ss += x[r][e] * x[r][e];
            const float rstd = rsqrt_near(warp_sum(ss) * (1.0f / HD) + a.eps);
#pragma unroll
            for (int e = 0; e < E; e++) x[r][e] = x[r][e] * rstd * g[e];
        }
        if (turn) {
            const int pos = start + i;
            float y[E];
#pragma unroll
            for (int e = 0; e < E; e++) y[e] = __shfl_sync(0xffffffffu, x[r][e], partner);
            if (in_rot && live && pos < a.cs_rows) {
                const float2* cs = reinterpret_cast<const float2*>(a.cs) + int64_t(pos) * half + j0;
                if (a.interleaved && E > 1) {
#pragma unroll
                    for (int e = 0; e < E / 2; e++) {
                        const float2 t = cs[e];
                        const float p = x[r][2 * e], q = x[r][2 * e + 1];
                        x[r][2 * e] = turned(p, q, t.x, -t.y);
                        x[r][2 * e + 1] = turned(q, p, t.x, t.y);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < E; e++) {
                        const float2 t = cs[e];
                        x[r][e] = turned(x[r][e], y[e], t.x, upper ? t.y : -t.y);
                    }
                }
            }
        }
    }

    if (kind == 0) {
        T* dst = static_cast<T*>(a.q_out) + int64_t(head) * a.o_head + lane * E;
        const bool ov = ((reinterpret_cast<uintptr_t>(dst) | (uintptr_t(a.o_token) * sizeof(T))) & (sizeof(T) * E - 1)) == 0;
#pragma unroll
        for (int r = 0; r < kFewTokens; r++) {
            if (i0 + r >= i1) break;
            if (!live)
#pragma unroll
                for (int e = 0; e < E; e++) x[r][e] = 0.0f;
            store_row<E>(dst + int64_t(row0 + i0 + r) * a.o_token, ov, x[r]);
        }
        return;
    }

    // keys and values
    if (!live) return;
    int i_end = i1;
    if (a.rot > 0 && start + i1 > a.cs_rows) {  // positions past the rotation table are not stored
        i_end = max(i0, a.cs_rows - start);
        if (lane == 0) set_op_error(kErrBadIndex);
    }
    if (i_end <= i0 || !resident) return;
    const int64_t base = int64_t(page) * c.page_stride + int64_t(head) * ps * HD;
    if constexpr (!Q8) {
        __half* dst = static_cast<__half*>(kind == 1 ? c.k_pages : c.v_pages) + base + lane * E;
#pragma unroll
        for (int r = 0; r < kFewTokens; r++) {
            if (i0 + r >= i_end) break;
            store_row<E>(dst + (o0 + r) * HD, true, x[r]);
        }
    } else {
        float most = 0.0f;
#pragma unroll
        for (int r = 0; r < kFewTokens; r++) {
            if (i0 + r >= i_end) break;
#pragma unroll
            for (int e = 0; e < E; e++) most = fmaxf(most, finite_abs(x[r][e]));
        }
        float scale = block_scale(warp_max(most));
        uint8_t* blk = static_cast<uint8_t*>(kind == 1 ? c.k_pages : c.v_pages) + base;
        if (o0 > 0) {
            if (old > scale) scale = old;
            else if (old < scale) recode(blk, o0 * HD, old / scale, lane, 32);
        }
        if (lane == 0) *sp = scale;
        const float inv = 1.0f / scale;  // exact: a power of two
#pragma unroll
        for (int r = 0; r < kFewTokens; r++) {
            if (i0 + r >= i_end) break;
            uint8_t* dst = blk + (o0 + r) * HD + lane * E;
            if constexpr (E == 4) {
                *reinterpret_cast<uint32_t*>(dst) = uint32_t(f32x2_to_e4m3x2(x[r][0] * inv, x[r][1] * inv)) |
                                                    uint32_t(f32x2_to_e4m3x2(x[r][2] * inv, x[r][3] * inv)) << 16;
            } else if constexpr (E == 2) {
                *reinterpret_cast<uint16_t*>(dst) = f32x2_to_e4m3x2(x[r][0] * inv, x[r][1] * inv);
            } else {
                *dst = uint8_t(f32x2_to_e4m3x2(x[r][0] * inv, 0.0f));
            }
        }
    }
}

// Four values of type T at p.
template <typename T>
struct Four {
    using V = typename std::conditional<sizeof(T) == 4, uint4, uint2>::type;
    alignas(sizeof(V)) T v[4];
};
template <typename T>
__device__ __forceinline__ void get4(const T* p, bool vec, Four<T>& f) {
    if (vec) {
        *reinterpret_cast<typename Four<T>::V*>(f.v) = *reinterpret_cast<const typename Four<T>::V*>(p);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) f.v[i] = p[i];
    }
}

// Values 2 h and 2 h + 1 as an f32 pair.
template <typename T>
__device__ __forceinline__ uint64_t pair_of(const Four<T>& f, int h) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const uint32_t w = reinterpret_cast<const uint32_t*>(f.v)[h];
        return pack2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    } else if constexpr (std::is_same<T, __half>::value) {
        const float2 v = __half22float2(reinterpret_cast<const __half2*>(f.v)[h]);
        return pack2(v.x, v.y);
    } else {
        return pack2(f.v[2 * h], f.v[2 * h + 1]);
    }
}
template <typename T>
__device__ __forceinline__ void put4(T* p, bool vec, uint64_t x, uint64_t y) {
    float v[4];
    unpack2(x, v[0], v[1]), unpack2(y, v[2], v[3]);
    Four<T> f;
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        reinterpret_cast<__nv_bfloat162*>(f.v)[0] = __floats2bfloat162_rn(v[0], v[1]);
        reinterpret_cast<__nv_bfloat162*>(f.v)[1] = __floats2bfloat162_rn(v[2], v[3]);
    } else if constexpr (std::is_same<T, __half>::value) {
        reinterpret_cast<__half2*>(f.v)[0] = __floats2half2_rn(v[0], v[1]);
        reinterpret_cast<__half2*>(f.v)[1] = __floats2half2_rn(v[2], v[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) f.v[i] = v[i];
    }
    if (vec) {
        *reinterpret_cast<typename Four<T>::V*>(p) = *reinterpret_cast<const typename Four<T>::V*>(f.v);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) p[i] = f.v[i];
    }
}

template <typename T, int HD, bool Q8>
__global__ void __launch_bounds__(512) paged_append_kernel(const neko_paged_append_args a, const AppendPlan plan) {
    constexpr int kLanes = HD / 8, kRowsPer = 32 / kLanes;  // lanes per token, tokens per warp and slot
    __shared__ uint32_t red[2][32];
    __shared__ __align__(16) float gains[2][HD];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int s = blockIdx.x, chunk = blockIdx.z;
    const int u0 = blockIdx.y * plan.per_cta, u1 = min(plan.units, u0 + plan.per_cta);

    const neko_paged_cache& c = a.cache;
    const int row0 = a.q_start ? a.q_start[s] : s;
    const int n = a.q_start ? a.q_start[s + 1] - row0 : 1;
    const int start = min(a.start[s], kFarthest);
    if (row0 < 0 || n < 0 || n > a.max_new || row0 + n > a.tokens) {  // outside the planned rows
        if (threadIdx.x == 0) set_op_error(kErrBadIndex);
        return;
    }
    const bool live = start >= 0;
    const int ps = c.page_size;
    const int first = live ? start >> plan.page_log : 0, off0 = live ? start & (ps - 1) : 0;
    const int i0 = max(0, chunk * ps - off0), count = min(n, (chunk + 1) * ps - off0) - i0;  // tokens of this page
    if (count <= 0) return;
    const int slot0 = first + chunk;
    const int page = live && slot0 < c.max_pages ? c.table[int64_t(s) * c.table_stride + slot0] : -1;
    const int o0 = chunk == 0 ? off0 : 0;  // the first new token's place in the page
    const int pos0 = start + i0;           // and its position
    int stored = page >= 0 && page < c.num_pages ? count : 0;  // tokens that are stored: none past the rotation table
    if (live && a.rot > 0 && pos0 + count > a.cs_rows) {
        stored = min(stored, max(0, a.cs_rows - pos0));
        if (threadIdx.x == 0) set_op_error(kErrBadIndex);
    }
    const int nh = a.q ? a.n_head : 0;

    // this lane's eight values: four at da, four at db. Half layout: pairs (j, j + rot / 2), then the rest of the head, whose
    // values stay as they are (not turned by 0: an infinity or NaN beside would reach them); interleaved: eight in a row.
    const int l = lane % kLanes, half = a.rot >> 1;
    int da = 8 * l, db = 8 * l + 4;
    bool in_rot = 8 * l < a.rot;
    if (!a.interleaved && a.rot) {
        const int j = 4 * l;
        in_rot = j < half;
        da = in_rot ? j : a.rot + j - half;
        db = in_rot ? j + half : a.rot + (HD - a.rot) / 2 + j - half;
    }
    int tok[kSlots];  // this lane's token in each slot, from i0
    uint64_t cs[kSlots][2], sn[kSlots][2];  // cosines and sines of the four pairs, two and two
    bool turns[kSlots];                     // past the rotation table, and beyond `rot`, nothing does
#pragma unroll
    for (int z = 0; z < kSlots; z++) {
        tok[z] = (z * warps + warp) * kRowsPer + lane / kLanes;
        const int pos = pos0 + tok[z];
        const bool turn = in_rot && live && tok[z] < count && pos < a.cs_rows;
        turns[z] = turn;
        const float4* p = reinterpret_cast<const float4*>(a.cs + (turn ? int64_t(pos) * a.rot + 8 * l : 0));
        const float4 t0 = turn ? p[0] : make_float4(1, 0, 1, 0), t1 = turn ? p[1] : make_float4(1, 0, 1, 0);
        cs[z][0] = pack2(t0.x, t0.z), cs[z][1] = pack2(t1.x, t1.z);
        sn[z][0] = pack2(t0.y, t0.w), sn[z][1] = pack2(t1.y, t1.w);
    }
    const bool all_turn = a.rot == HD && live && pos0 + count <= a.cs_rows;
    if (a.k_gain) {
        for (int d = threadIdx.x; d < HD; d += blockDim.x) {
            if (a.q) gains[0][d] = a.q_gain[d];
            gains[1][d] = a.k_gain[d];
        }
        __syncthreads();
    }

    const T* src = nullptr;  // i0's row of the unit that is fetched next
    int64_t head_step = 0;
    int off[kSlots], out_off[kSlots];  // of this lane's tokens' rows (the host has checked that 128 rows fit 31 bits)
    bool vec = false;
    const bool out_vec = ((reinterpret_cast<uintptr_t>(a.q_out) | (uintptr_t(a.o_token | a.o_head) * sizeof(T))) & (sizeof(T) * 4 - 1)) == 0;
#pragma unroll
    for (int z = 0; z < kSlots; z++) out_off[z] = tok[z] * int(a.o_token);
    auto kind_of = [&](int u) { return u < nh ? 0 : u < nh + c.n_kv ? 1 : 2; };  // q, k, v
    auto head_of = [&](int u, int kind) { return kind == 0 ? u : kind == 1 ? u - nh : u - nh - c.n_kv; };
    Four<T> next[kSlots][2] = {};
    auto fetch = [&](int u) {
        if (u == u0 || u == nh || u == nh + c.n_kv) {
            const int kind = kind_of(u);
            const int64_t ts = kind == 0 ? a.q_token : kind == 1 ? a.k_token : a.v_token;
            head_step = kind == 0 ? a.q_head : kind == 1 ? a.k_head : a.v_head;
            src = static_cast<const T*>(kind == 0 ? a.q : kind == 1 ? a.k : a.v) + head_of(u, kind) * head_step + (row0 + i0) * ts;
            vec = ((reinterpret_cast<uintptr_t>(src) | (uintptr_t(ts | head_step) * sizeof(T))) & (sizeof(T) * 4 - 1)) == 0;
#pragma unroll
            for (int z = 0; z < kSlots; z++) off[z] = tok[z] * int(ts);
        }
#pragma unroll
        for (int z = 0; z < kSlots; z++)
            if (tok[z] < count) {
                get4(src + off[z] + da, vec, next[z][0]);
                get4(src + off[z] + db, vec, next[z][1]);
            }
        src += head_step;
    };
    fetch(u0);
#pragma unroll 1
    for (int u = u0; u < u1; u++) {
        const int kind = kind_of(u), head = head_of(u, kind);
        uint64_t x[kSlots][4];  // value pairs
#pragma unroll
        for (int z = 0; z < kSlots; z++)
#pragma unroll
            for (int e = 0; e < 4; e++) x[z][e] = pair_of(next[z][e / 2], e & 1);
        if (u + 1 < u1) fetch(u + 1);
        if (kind != 0 && stored == 0) continue;  // the same for the whole CTA
        float old = 0.0f;
        float* sp = nullptr;
        if (Q8 && kind != 0) {
            sp = (kind == 1 ? c.k_scale : c.v_scale) + int64_t(page) * c.scale_stride + head;
            if (o0 > 0) old = *sp;
        }
        if (kind != 2 && a.k_gain) {
            const ulonglong2 ga = *reinterpret_cast<const ulonglong2*>(&gains[kind][da]), gb = *reinterpret_cast<const ulonglong2*>(&gains[kind][db]);
            float ss[kSlots];
#pragma unroll
            for (int z = 0; z < kSlots; z++) {
                uint64_t t = mul2(x[z][0], x[z][0]);
#pragma unroll
                for (int e = 1; e < 4; e++) t = fma2(x[z][e], x[z][e], t);
                float t0, t1;
                unpack2(t, t0, t1);
                ss[z] = t0 + t1;
            }
#pragma unroll
            for (int o = kLanes / 2; o > 0; o >>= 1)
#pragma unroll
                for (int z = 0; z < kSlots; z++) ss[z] += __shfl_xor_sync(0xffffffffu, ss[z], o);
#pragma unroll
            for (int z = 0; z < kSlots; z++) {
                const float rstd = rsqrt_near(ss[z] * (1.0f / HD) + a.eps);
                const uint64_t r2 = pack2(rstd, rstd);
                x[z][0] = mul2(mul2(x[z][0], r2), ga.x), x[z][1] = mul2(mul2(x[z][1], r2), ga.y);
                x[z][2] = mul2(mul2(x[z][2], r2), gb.x), x[z][3] = mul2(mul2(x[z][3], r2), gb.y);
            }
        }
        if (kind != 2 && a.rot) {
            auto turn = [&](auto all) {
#pragma unroll
                for (int z = 0; z < kSlots; z++) {
                    if (!decltype(all)::value && !turns[z]) continue;
                    if (a.interleaved) {
#pragma unroll
                        for (int e = 0; e < 4; e++) {  // pair e: its two values are one register pair
                            float p, q, c0, c1, s0, s1;
                            unpack2(x[z][e], p, q), unpack2(cs[z][e / 2], c0, c1), unpack2(sn[z][e / 2], s0, s1);
                            const float co = e & 1 ? c1 : c0, si = e & 1 ? s1 : s0;
                            x[z][e] = pack2(turned(p, q, co, -si), turned(q, p, co, si));
                        }
                    } else {
                        const uint64_t minus = pack2(-1.0f, -1.0f);
#pragma unroll
                        for (int e = 0; e < 2; e++) {  // pairs 2 e and 2 e + 1
                            const uint64_t p = x[z][e], q = x[z][2 + e];
                            x[z][e] = fma2(p, cs[z][e], mul2(q, mul2(sn[z][e], minus)));
                            x[z][2 + e] = fma2(q, cs[z][e], mul2(p, sn[z][e]));
                        }
                    }
                }
            };
            // Where the whole head turns at every position, whatever rows past `count` hold turns too: no predicate a value
            // (ragged prompts 95.7 us, 97.6 with one).
            if (all_turn) turn(std::true_type());
            else turn(std::false_type());
        }
        if (kind == 0) {
            T* dst = static_cast<T*>(a.q_out) + head * a.o_head + (row0 + i0) * a.o_token;
#pragma unroll
            for (int z = 0; z < kSlots; z++) {
                if (tok[z] >= count) continue;
                if (!live) x[z][0] = x[z][1] = x[z][2] = x[z][3] = 0;
                put4(dst + out_off[z] + da, out_vec, x[z][0], x[z][1]);
                put4(dst + out_off[z] + db, out_vec, x[z][2], x[z][3]);
            }
            continue;
        }
        const int64_t base = int64_t(page) * c.page_stride + int64_t(head) * ps * HD + o0 * HD;
        if constexpr (!Q8) {
            __half* dst = static_cast<__half*>(kind == 1 ? c.k_pages : c.v_pages) + base;
#pragma unroll
            for (int z = 0; z < kSlots; z++) {
                if (tok[z] >= stored) continue;
                put4(dst + tok[z] * HD + da, true, x[z][0], x[z][1]);
                put4(dst + tok[z] * HD + db, true, x[z][2], x[z][3]);
            }
        } else {
            // the largest finite magnitude, as bits
            uint32_t most = 0;
#pragma unroll
            for (int z = 0; z < kSlots; z++)
                if (tok[z] < stored)
#pragma unroll
                    for (int e = 0; e < 4; e++) most = max(most, max(uint32_t(x[z][e]) & 0x7fffffffu, uint32_t(x[z][e] >> 32) & 0x7fffffffu));
            if (most >= 0x7f800000u) {  // infinities or NaN among them
                most = 0;
#pragma unroll
                for (int z = 0; z < kSlots; z++)
                    if (tok[z] < stored)
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            const uint32_t m = uint32_t(x[z][e / 2] >> (32 * (e & 1))) & 0x7fffffffu;
                            if (m < 0x7f800000u) most = max(most, m);
                        }
            }
            most = __reduce_max_sync(0xffffffffu, most);
            if (lane == 0) red[u & 1][warp] = most;
            __syncthreads();  // also: every thread has read the old scale
            float scale = block_scale(__uint_as_float(__reduce_max_sync(0xffffffffu, lane < warps ? red[u & 1][lane] : 0u)));
            float inv = __uint_as_float((254u << 23) - __float_as_uint(scale));  // of a power of two
            uint8_t* blk = static_cast<uint8_t*>(kind == 1 ? c.k_pages : c.v_pages) + base;
            if (o0 > 0) {
                if (old > scale) scale = old, inv = 1.0f / old;
                else if (old < scale) recode(blk - o0 * HD, o0 * HD, old * inv, threadIdx.x, blockDim.x);
            }
            if (threadIdx.x == 0) *sp = scale;
            const uint64_t inv2 = pack2(inv, inv);
#pragma unroll
            for (int z = 0; z < kSlots; z++) {
                if (tok[z] >= stored) continue;
#pragma unroll
                for (int y = 0; y < 2; y++) {
                    float v0, v1, v2, v3;
                    unpack2(mul2(x[z][2 * y], inv2), v0, v1), unpack2(mul2(x[z][2 * y + 1], inv2), v2, v3);
                    *reinterpret_cast<uint32_t*>(blk + tok[z] * HD + (y ? db : da)) =
                        uint32_t(f32x2_to_e4m3x2(v0, v1)) | uint32_t(f32x2_to_e4m3x2(v2, v3)) << 16;
                }
            }
        }
    }
}

template <typename T, int HD, bool Q8>
cudaError_t go(const neko_paged_append_args& a, cudaStream_t st) {
    AppendPlan p;
    const int ps = a.cache.page_size;
    p.page_log = 31 - __builtin_clz(ps);
    const int64_t chunks = (int64_t(a.max_new) + ps - 2) / ps + 1;  // an unaligned start can touch one page more
    p.units = (a.q ? a.n_head : 0) + 2 * a.cache.n_kv;
    p.per_cta = 1;
    if (a.max_new <= kFewTokens) {
        if (chunks > 65535 || (p.units + 3) / 4 > 65535) return cudaErrorInvalidConfiguration;
        return launch_ex(paged_append_step_kernel<T, HD, Q8>, dim3(unsigned(a.cache.n_seq), unsigned(p.units + 3) / 4, unsigned(chunks)),
                         dim3(128), 0, st, false, a, p);
    }
    const int warps = std::max(1, ps * (HD / 8) / (32 * kSlots));
    // heads per CTA: up to 8, which share the loads of the cosines (ragged prompts of 14,364 tokens: 92 us, with 4 heads
    // 97), as long as every SM gets 24 warps (a prompt of 4,001 tokens on 12 heads: 4 heads 12.5 us, 8 heads 14.8)
    while (p.per_cta < 8 && a.cache.n_seq * chunks * ((p.units + 2 * p.per_cta - 1) / (2 * p.per_cta)) * warps >= 24 * num_sms()) p.per_cta *= 2;
    const int groups = (p.units + p.per_cta - 1) / p.per_cta;
    if (chunks > 65535 || groups > 65535) return cudaErrorInvalidConfiguration;
    return launch_ex(paged_append_kernel<T, HD, Q8>, dim3(unsigned(a.cache.n_seq), unsigned(groups), unsigned(chunks)), dim3(32 * warps), 0,
                     st, false, a, p);
}

template <typename T>
cudaError_t by_shape(const neko_paged_append_args& a, cudaStream_t st) {
    const bool q8 = a.cache.type == NEKO_T_E4M3;
    switch (a.cache.head_dim) {
        case 32: return q8 ? go<T, 32, true>(a, st) : go<T, 32, false>(a, st);
        case 64: return q8 ? go<T, 64, true>(a, st) : go<T, 64, false>(a, st);
        default: return q8 ? go<T, 128, true>(a, st) : go<T, 128, false>(a, st);
    }
}

}  // namespace

cudaError_t launch_paged_append(const neko_paged_append_args& args, cudaStream_t st) {
    neko_paged_append_args a = args;
    a.cs_rows = std::min(a.cs_rows, kFarthest);
    return a.type == NEKO_T_F32   ? by_shape<float>(a, st)
           : a.type == NEKO_T_F16 ? by_shape<__half>(a, st)
                                  : by_shape<__nv_bfloat16>(a, st);
}

}  // namespace neko
