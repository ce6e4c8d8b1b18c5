// Moving what a paged cache holds, in all its planes (keys and values of every layer) by one launch: whole pages
// (neko_op_paged_copy) and tokens of a sequence (neko_op_paged_compact).
#include <algorithm>

#include "paged.cuh"

namespace neko {

namespace {

constexpr int kCopyThreads = 256, kPieces = 4;  // 16-byte pieces that a thread has in flight

// A CTA for each 16 KB of a page and plane: bound by memory, every thread's loads come before its stores. 301 pages of 64 tokens, 8 e4m3
// heads of 128, 72 planes: 427 us, 6.65 TB/s of reads and writes, the measured copy rate; 3 f16 pages in 56 planes 6 us.
__global__ void __launch_bounds__(kCopyThreads) paged_copy_kernel(const neko_paged_planes c, const int32_t* __restrict__ src,
                                                                 const int32_t* __restrict__ dst, int chunks, int pieces, int size) {
    const int pair = blockIdx.x / chunks, chunk = blockIdx.x % chunks, plane = blockIdx.y;
    const int from = src[pair], to = dst[pair];
    if (from < 0 || from >= c.num_pages || to < 0 || to >= c.num_pages || from == to) return;
    uint8_t* base = static_cast<uint8_t*>(c.pages) + plane * c.plane_stride * size;
    const uint4* s = reinterpret_cast<const uint4*>(base + from * c.page_stride * size);
    uint4* d = reinterpret_cast<uint4*>(base + to * c.page_stride * size);
    const int i0 = chunk * kCopyThreads * kPieces + threadIdx.x;
    uint4 v[kPieces];
#pragma unroll
    for (int k = 0; k < kPieces; k++)
        if (i0 + k * kCopyThreads < pieces) v[k] = s[i0 + k * kCopyThreads];
#pragma unroll
    for (int k = 0; k < kPieces; k++)
        if (i0 + k * kCopyThreads < pieces) d[i0 + k * kCopyThreads] = v[k];
    if (c.type == kTE4M3 && chunk == 0) {
        float* scale = c.scale + plane * c.scale_plane;
        for (int h = threadIdx.x; h < c.n_kv; h += kCopyThreads) scale[to * c.scale_stride + h] = scale[from * c.scale_stride + h];
    }
}

// Codes times a ratio of scales, four at a time.
__device__ __forceinline__ uint32_t recode4(uint32_t v, float ratio) {
    const uint32_t f0 = e4m3x2_to_f16x2(uint16_t(v)), f1 = e4m3x2_to_f16x2(uint16_t(v >> 16));
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&f0)), b = __half22float2(*reinterpret_cast<const __half2*>(&f1));
    return uint32_t(f32x2_to_e4m3x2(a.x * ratio, a.y * ratio)) | uint32_t(f32x2_to_e4m3x2(b.x * ratio, b.y * ratio)) << 16;
}
__device__ __forceinline__ uint4 recode16(uint4 v, float ratio) {
    if (ratio == 1.0f) return v;
    return make_uint4(recode4(v.x, ratio), recode4(v.y, ratio), recode4(v.z, ratio), recode4(v.w, ratio));
}

// A warp for each (sequence, head, plane). Paths ascend, so no token goes to a later place than it comes from, and none that is
// still to be read has been written over: a group of tokens is read into registers, then written, then the next. 8-bit: one
// target page after the other, for its scale is that of all the tokens that end in it; those come from it or from later pages, whose
// scales are still the old ones.
// Bound by latency: path, table, scales and tokens one after the other, with little in each warp (64 sequences of up to 16 nodes,
// 72 planes of 8 e4m3 heads, memory cold: 50 us; 4 CTAs an SM at 116 registers 63, 8 at 64 registers 54).
constexpr int kWarps = 4, kBatch = 4, kStay = 4;  // warps of a CTA; pieces of tokens, and of tokens that stay, that a lane has in flight
constexpr int kAtOnce = 6;                          // CTAs of an SM: 80 registers a thread
template <int HD, bool Q8>
__global__ void __launch_bounds__(32 * kWarps, kAtOnce) paged_compact_kernel(const neko_paged_planes c, const int32_t* __restrict__ start_of,
                                                                  const int32_t* __restrict__ path_of, int64_t path_stride,
                                                                  const int32_t* __restrict__ count_of, int max_count, int page_log) {
    constexpr int kRow = HD * (Q8 ? 1 : 2), kLanes = kRow / 16, kPer = 32 / kLanes,  // bytes of a token, lanes, tokens of a group's step
                  kB = kBatch < 32 / kPer ? kBatch : 32 / kPer;
    const int lane = threadIdx.x & 31, head = blockIdx.y * kWarps + (threadIdx.x >> 5), s = blockIdx.x, plane = blockIdx.z;
    if (head >= c.n_kv) return;
    const int32_t* path = path_of + int64_t(s) * path_stride;
    const int start = min(start_of[s], 1 << 30), count = count_of[s];
    if (count > max_count) {
        if (lane == 0) set_op_error(kErrBadIndex);
        return;
    }
    if (start < 0 || count <= 0) return;
    const int32_t* table = c.table + int64_t(s) * c.table_stride;
    const int in_page = (1 << page_log) - 1;
    uint8_t* pool = static_cast<uint8_t*>(c.pages) + (plane * c.plane_stride + (int64_t(head) << page_log) * HD) * (Q8 ? 1 : 2);
    float* scales = Q8 ? c.scale + plane * c.scale_plane + head : nullptr;
    auto page_at = [&](int pos) {
        const int slot = pos >> page_log;
        const int p = pos >= 0 && slot < c.max_pages ? table[slot] : -1;
        return p < c.num_pages ? p : -1;
    };
    auto row_at = [&](int page, int pos) { return pool + page * c.page_stride * (Q8 ? 1 : 2) + (pos & in_page) * kRow; };
    // where token k comes from; -1: nowhere
    auto source_of = [&](int k) {
        const int x = path[k];
        return x >= 0 && x <= (1 << 30) ? start + x : -1;
    };
    for (int k0 = 0; k0 < count;) {
        // Tokens of one target page. What says where they come from is read by a lane for each of 32 tokens, and the tokens of the
        // first batch before anything waits for the scales.
        const int k1 = min(count, k0 + (in_page + 1) - ((start + k0) & in_page));
        const int to_page = page_at(start + k0);
        if (to_page >= 0) {
            int from = -1, page = -1;
            [[maybe_unused]] float mine = 0.0f;  // the scale of the lane's token's page
            auto look = [&](int kb) {
                from = kb + lane < k1 ? source_of(kb + lane) : -1;
                page = page_at(from);
                if constexpr (Q8) mine = page >= 0 ? scales[page * c.scale_stride] : 0.0f;
            };
            uint4 v[kB];
            // the batch's tokens kb + kk ..: bits of those that there are
            auto load = [&](int kb, int kk) {
                int got = 0;
#pragma unroll
                for (int b = 0; b < kB; b++) {
                    const int i = kk + b * kPer + lane / kLanes, f = __shfl_sync(0xffffffffu, from, i), p = __shfl_sync(0xffffffffu, page, i);
                    if (p < 0 || (!Q8 && f == start + kb + i)) continue;
                    if (f == start + kb + i) got |= 256 << b;  // stays where it is
                    v[b] = *reinterpret_cast<const uint4*>(row_at(p, f) + lane % kLanes * 16), got |= 1 << b;
                }
                return got;
            };
            look(k0);
            int got = load(k0, 0);
            [[maybe_unused]] float scale = 0.0f;
            if constexpr (Q8) {
                const int stay = k0 == 0 ? start & in_page : 0;  // tokens of this page before the moved ones
                const float old = scales[to_page * c.scale_stride];
                bool any = stay || page >= 0;
                scale = stay ? fmaxf(old, mine) : mine;
                for (int k = k0 + 32 + lane; k < k1; k += 32) {
                    const int p = page_at(source_of(k));
                    if (p >= 0) scale = fmaxf(scale, scales[p * c.scale_stride]), any = true;
                }
                scale = warp_max(scale);
                any = __any_sync(0xffffffffu, any);
                if (any && stay && scale > old) {
                    uint4* w = reinterpret_cast<uint4*>(row_at(to_page, 0));
                    const float ratio = old / scale;
                    for (int i = lane; i < stay * kLanes; i += 32 * kStay) {
                        uint4 x[kStay];
#pragma unroll
                        for (int b = 0; b < kStay; b++)
                            if (i + 32 * b < stay * kLanes) x[b] = w[i + 32 * b];
#pragma unroll
                        for (int b = 0; b < kStay; b++)
                            if (i + 32 * b < stay * kLanes) w[i + 32 * b] = recode16(x[b], ratio);
                    }
                }
                if (!any) scale = old;
            }
            for (int kb = k0; kb < k1; kb += 32) {
                if (kb > k0) look(kb);
                for (int kk = 0; kk < min(32, k1 - kb); kk += kPer * kB) {
                    if (kb > k0 || kk) got = load(kb, kk);
                    __syncwarp();
#pragma unroll
                    for (int b = 0; b < kB; b++) {
                        const int i = kk + b * kPer + lane / kLanes;
                        [[maybe_unused]] const float x = __shfl_sync(0xffffffffu, mine, i);
                        if (!(got >> b & 1)) continue;
                        if constexpr (Q8) {
                            if ((got >> b & 256) && x >= scale) continue;
                            v[b] = recode16(v[b], x < scale ? x / scale : 1.0f);
                        }
                        *reinterpret_cast<uint4*>(row_at(to_page, start + kb + i) + lane % kLanes * 16) = v[b];
                    }
                    __syncwarp();
                }
            }
            if constexpr (Q8) {
                if (lane == 0) scales[to_page * c.scale_stride] = scale;
                __syncwarp();
            }
        }
        k0 = k1;
    }
}

template <int HD>
cudaError_t go(const neko_paged_planes& c, const int32_t* start, const int32_t* path, int64_t path_stride, const int32_t* count, int max_count,
               cudaStream_t st) {
    const dim3 grid(unsigned(c.n_seq), unsigned(c.n_kv + kWarps - 1) / kWarps, unsigned(c.planes));
    auto* fn = c.type == NEKO_T_E4M3 ? paged_compact_kernel<HD, true> : paged_compact_kernel<HD, false>;
    return launch_ex(fn, grid, dim3(32 * kWarps), 0, st, false, c, start, path, path_stride, count, max_count, 31 - __builtin_clz(c.page_size));
}

}  // namespace

cudaError_t launch_paged_copy(const neko_paged_planes& c, const int32_t* src, const int32_t* dst, int n, cudaStream_t st) {
    const int size = c.type == NEKO_T_E4M3 ? 1 : 2;
    const int64_t pieces = int64_t(c.n_kv) * c.page_size * c.head_dim * size / 16, chunks = (pieces + kCopyThreads * kPieces - 1) / (kCopyThreads * kPieces);
    if (pieces > 0x7fffffff || chunks * n > 0x7fffffff) return cudaErrorInvalidConfiguration;
    return launch_ex(paged_copy_kernel, dim3(unsigned(chunks * n), unsigned(c.planes)), dim3(kCopyThreads), 0, st, false, c, src, dst, int(chunks),
                     int(pieces), size);
}

cudaError_t launch_paged_compact(const neko_paged_planes& c, const int32_t* start, const int32_t* path, int64_t path_stride,
                                 const int32_t* count, int max_count, cudaStream_t st) {
    switch (c.head_dim) {
        case 32: return go<32>(c, start, path, path_stride, count, max_count, st);
        case 64: return go<64>(c, start, path, path_stride, count, max_count, st);
        default: return go<128>(c, start, path, path_stride, count, max_count, st);
    }
}

}  // namespace neko
