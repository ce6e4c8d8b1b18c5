// Appending keys and values to a paged cache (neko_op_paged_append): per-head RMSNorm of q and k, rotary position
// embedding, one rounding to the cache's type. The engine's counterpart is rope.comp + kv_store.comp on a contiguous
// f16 cache (qwen3_model.cpp:249-254, cpu_ops.cpp:513-542); pages, 8-bit blocks, partial and interleaved rotations
// have none.
//
// A unit of work is the (at most page_size) new tokens that one sequence puts into one page, for one head of q, k or
// v: an 8-bit block's scale depends on all of them, so one owner sees them all and no atomics are needed. A unit is
// taken by one warp (few new tokens) or by eight (prompts); every lane holds head_dim / 32 consecutive values of a
// token, all tokens of the warp in registers, so a value is read once whatever the scale turns out to be. The
// rotation's partner comes from a shuffle (rot a multiple of 8) and the squares' sum from five.
#include <type_traits>

#include "paged.cuh"

namespace neko {

namespace {

constexpr int kFewTokens = 4;  // tokens a single-warp unit holds

struct AppendPlan {
    int chunks;  // pages a sequence's new tokens can touch
    int units;   // head rows: n_head + 2 n_kv (n_head = 0 without q)
};

template <typename T, int HD, bool Q8, int WU, int RPW>
__global__ void __launch_bounds__(WU == 1 ? 128 : 32 * WU) paged_append_kernel(const neko_paged_append_args a,
                                                                              const AppendPlan plan) {
    constexpr int E = HD / 32;  // values per lane and token
    __shared__ float red[WU];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int upb = WU == 1 ? 4 : 1;  // units per block
    const int ublocks = (plan.units + upb - 1) / upb;
    int b = blockIdx.x;
    const int unit = (b % ublocks) * upb + (WU == 1 ? warp : 0);
    b /= ublocks;
    const int chunk = b % plan.chunks, s = b / plan.chunks;
    if (unit >= plan.units) return;
    const int wu = WU == 1 ? 0 : warp;  // this warp's index in its unit

    const neko_paged_cache& c = a.cache;
    const int row0 = a.q_start ? a.q_start[s] : s;
    int n = a.q_start ? a.q_start[s + 1] - row0 : 1;
    if (row0 < 0 || n < 0 || n > a.max_new || row0 + n > a.tokens) {  // outside the planned rows
        if (threadIdx.x == 0) set_device_error(kErrBadIndex);
        return;
    }
    const int start = a.start[s];
    const bool live = start >= 0;
    const int ps = c.page_size;
    // token range [i0, i1) of this unit
    const int first = live ? start / ps : 0, off0 = live ? start % ps : 0;
    const int i0 = max(0, chunk * ps - off0), i1 = min(n, (chunk + 1) * ps - off0);
    if (i0 >= i1) return;
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
    float x[RPW][E];
#pragma unroll
    for (int r = 0; r < RPW; r++) {
        const int i = i0 + wu + r * WU;
        if (i < i1) load_row<E>(src + int64_t(row0 + i) * ts, vec, x[r]);
        else
#pragma unroll
            for (int e = 0; e < E; e++) x[r][e] = 0.0f;
    }
    float g[E];
    if (gain) load_row<E>(gain + lane * E, false, g);

    const int half = a.rot >> 1;
    // this lane's first rotation index and its partner lane
    const int d0 = lane * E;
    const bool in_rot = turn && d0 < a.rot;
    const int j0 = a.interleaved ? d0 >> 1 : d0 < half ? d0 : d0 - half;
    const bool upper = a.interleaved ? (E == 1 && (lane & 1)) : d0 >= half;
    const int partner = a.interleaved ? (E == 1 ? lane ^ 1 : lane) : in_rot ? (upper ? lane - half / E : lane + half / E) : lane;

#pragma unroll
    for (int r = 0; r < RPW; r++) {
        const int i = i0 + wu + r * WU;
        if (i >= i1) break;  // uniform over the warp
        if (gain) {
            float ss = 0.0f;
#pragma unroll
            for (int e = 0; e < E; e++) ss += x[r][e] * x[r][e];
            const float rstd = 1.0f / sqrtf(warp_sum(ss) / float(HD) + a.eps);
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
                        x[r][2 * e] = p * t.x - q * t.y;
                        x[r][2 * e + 1] = q * t.x + p * t.y;
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < E; e++) {
                        const float2 t = cs[e];
                        x[r][e] = upper ? x[r][e] * t.x + y[e] * t.y : x[r][e] * t.x - y[e] * t.y;
                    }
                }
            }
        }
    }

    if (kind == 0) {
        T* dst = static_cast<T*>(a.q_out) + int64_t(head) * a.o_head + lane * E;
        const bool ov = ((reinterpret_cast<uintptr_t>(dst) | (uintptr_t(a.o_token) * sizeof(T))) & (sizeof(T) * E - 1)) == 0;
#pragma unroll
        for (int r = 0; r < RPW; r++) {
            const int i = i0 + wu + r * WU;
            if (i >= i1) break;
            if (!live)
#pragma unroll
                for (int e = 0; e < E; e++) x[r][e] = 0.0f;
            store_row<E>(dst + int64_t(row0 + i) * a.o_token, ov, x[r]);
        }
        return;
    }

    // keys and values
    if (!live) return;
    int i_end = i1;
    if (a.rot > 0 && start + i1 > a.cs_rows) {  // positions past the rotation table are not stored
        i_end = max(i0, a.cs_rows - start);
        if (lane == 0) set_device_error(kErrBadIndex);
    }
    if (i_end <= i0) return;
    const int slot = first + chunk;
    const int page = slot < c.max_pages ? c.table[int64_t(s) * c.table_stride + slot] : -1;
    if (page < 0 || page >= c.num_pages) return;  // not resident
    const int o0 = chunk == 0 ? off0 : 0;          // the first new token's place in the page
    const int64_t base = int64_t(page) * c.page_stride + int64_t(head) * ps * HD;
    if constexpr (!Q8) {
        __half* dst = static_cast<__half*>(kind == 1 ? c.k_pages : c.v_pages) + base + lane * E;
#pragma unroll
        for (int r = 0; r < RPW; r++) {
            const int i = i0 + wu + r * WU;
            if (i >= i_end) break;
            store_row<E>(dst + (o0 + i - i0) * HD, true, x[r]);
        }
    } else {
        float most = 0.0f;
#pragma unroll
        for (int r = 0; r < RPW; r++) {
            if (i0 + wu + r * WU >= i_end) break;
#pragma unroll
            for (int e = 0; e < E; e++) {
                const float m = fabsf(x[r][e]);
                if (m <= 3.402823466e38f) most = fmaxf(most, m);  // finite ones only
            }
        }
        most = warp_max(most);
        if constexpr (WU > 1) {
            if (lane == 0) red[wu] = most;
            __syncthreads();
            most = red[0];
#pragma unroll
            for (int w = 1; w < WU; w++) most = fmaxf(most, red[w]);
        }
        // smallest 2^e with most <= 448 * 2^e: 448 = 1.75 * 2^8
        const uint32_t bits = __float_as_uint(most);
        int e2 = int(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
        e2 = max(e2, kScaleMinExp);  // zeros and subnormals too
        float scale = __uint_as_float(uint32_t(e2 + 127) << 23);
        float* sp = (kind == 1 ? c.k_scale : c.v_scale) + int64_t(page) * c.scale_stride + head;
        uint8_t* blk = static_cast<uint8_t*>(kind == 1 ? c.k_pages : c.v_pages) + base;
        if (o0 > 0) {
            const float old = *sp;
            if (old > scale) {
                scale = old;
            } else if (old < scale) {  // the tokens held before move to the larger scale
                const float ratio = old / scale;
                uint32_t* w = reinterpret_cast<uint32_t*>(blk);
                for (int k = wu * 32 + lane; k < o0 * HD / 4; k += 32 * WU) {
                    const uint32_t v = w[k];
                    uint32_t f0 = e4m3x2_to_f16x2(uint16_t(v)), f1 = e4m3x2_to_f16x2(uint16_t(v >> 16));
                    const float2 a0 = __half22float2(*reinterpret_cast<__half2*>(&f0));
                    const float2 a1 = __half22float2(*reinterpret_cast<__half2*>(&f1));
                    w[k] = uint32_t(f32x2_to_e4m3x2(a0.x * ratio, a0.y * ratio)) |
                           uint32_t(f32x2_to_e4m3x2(a1.x * ratio, a1.y * ratio)) << 16;
                }
            }
            if constexpr (WU > 1) __syncthreads();  // every warp has read the old scale
        }
        if (wu == 0 && lane == 0) *sp = scale;
        const float inv = 1.0f / scale;  // exact: a power of two
#pragma unroll
        for (int r = 0; r < RPW; r++) {
            const int i = i0 + wu + r * WU;
            if (i >= i_end) break;
            uint8_t* dst = blk + (o0 + i - i0) * HD + lane * E;
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

template <typename T, int HD, bool Q8>
cudaError_t go(const neko_paged_append_args& a, cudaStream_t st) {
    AppendPlan p;
    const int ps = a.cache.page_size;
    p.chunks = (a.max_new + ps - 2) / ps + 1;  // an unaligned start can touch one page more
    p.units = (a.q ? a.n_head : 0) + 2 * a.cache.n_kv;
    const bool few = a.max_new <= kFewTokens;
    const int64_t blocks = int64_t(a.cache.n_seq) * p.chunks * (few ? (p.units + 3) / 4 : p.units);
    if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
    const dim3 grid{unsigned(blocks)};
    if (few) return launch_ex(paged_append_kernel<T, HD, Q8, 1, kFewTokens>, grid, dim3(128), 0, st, false, a, p);
    if (ps == 16) return launch_ex(paged_append_kernel<T, HD, Q8, 8, 2>, grid, dim3(256), 0, st, false, a, p);
    if (ps == 32) return launch_ex(paged_append_kernel<T, HD, Q8, 8, 4>, grid, dim3(256), 0, st, false, a, p);
    if (ps == 64) return launch_ex(paged_append_kernel<T, HD, Q8, 8, 8>, grid, dim3(256), 0, st, false, a, p);
    return launch_ex(paged_append_kernel<T, HD, Q8, 8, 16>, grid, dim3(256), 0, st, false, a, p);
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

cudaError_t launch_paged_append(const neko_paged_append_args& a, cudaStream_t st) {
    return a.type == NEKO_T_F32   ? by_shape<float>(a, st)
           : a.type == NEKO_T_F16 ? by_shape<__half>(a, st)
                                  : by_shape<__nv_bfloat16>(a, st);
}

}  // namespace neko
