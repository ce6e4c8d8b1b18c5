// The paged key/value cache's kernels' arguments and small device helpers (k_paged.cu, k_paged_attn.cu).
#pragma once
#include <cuda_bf16.h>

#include "mma_frag.cuh"
#include "neko_common.cuh"
#include "neko_internal.h"

namespace neko {

enum PagedType : int { kTF32 = NEKO_T_F32, kTF16 = NEKO_T_F16, kTBF16 = NEKO_T_BF16, kTE4M3 = NEKO_T_E4M3 };
constexpr int kScaleMinExp = -100;  // scale of a block of zeros: 2^-100

// depth (NULL: none) [tokens]: the new tokens are nodes of a tree, turned by their depths instead of their places.
cudaError_t launch_paged_append(const neko_paged_append_args& a, const int32_t* depth, cudaStream_t st);
// tree (NULL: none): the new tokens are nodes of a tree, positions go by depth and what they see of one another by masks.
cudaError_t launch_paged_attention(const neko_paged_attention_args& a, const neko_tree* tree, cudaStream_t st);
// The tcgen05 kernel, head dim 64 or 128; launch_paged_attention says when (packed rows: new tokens x query heads per KV head).
cudaError_t launch_paged_prompt(const neko_paged_attention_args& a, const neko_tree* tree, cudaStream_t st);
constexpr int kPromptRows = 16;
cudaError_t launch_paged_compact(const neko_paged_planes& c, const int32_t* start, const int32_t* path, int64_t path_stride,
                                 const int32_t* count, int max_count, cudaStream_t st);
cudaError_t launch_paged_copy(const neko_paged_planes& c, const int32_t* src, const int32_t* dst, int n, cudaStream_t st);
cudaError_t launch_tree_masks(const int32_t* parent, const int32_t* q_start, int n_seq, int tokens, int max_new, uint64_t* mask, int words,
                              int32_t* depth, cudaStream_t st);
cudaError_t launch_tree_accept(const int32_t* chosen, const int32_t* draft, const int32_t* parent, const int32_t* q_start, int n_seq,
                               int tokens, int max_new, int32_t* path, int32_t* count, int32_t* token, cudaStream_t st);
cudaError_t launch_sample_rows(const neko_sample_rows_args& a, cudaStream_t st);

// What a kernel of these operators could not do (kErr*) goes to a word of their own, which neko_op_status reads: a model's
// steps read and clear the other one, and would fail for an operator's arguments.
extern __device__ unsigned g_op_error;
__device__ inline void set_op_error(unsigned code) { atomicCAS(&g_op_error, 0u, code); }

// Two e4m3 codes as exact f16 (0x7F / 0xFF: NaN).
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint16_t c) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(c));
    return r;
}
// lo -> bits 0-7, hi -> bits 8-15, to nearest even, beyond +-448 (infinities too) to +-448, NaN to NaN.
__device__ __forceinline__ uint16_t f32x2_to_e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// Where node i of a sequence of n nodes stands, counted from its first: its depth, within [0, n).
__device__ __forceinline__ int tree_depth(const neko_tree& tr, int row0, int i, int n) {
    return tr.depth ? min(max(tr.depth[row0 + i], 0), n - 1) : 0;
}
// Bits [o, o + 32) of a row's mask, zeros where it has none.
__device__ __forceinline__ uint32_t tree_bits(const neko_tree& tr, int row, int o) {
    const uint32_t* m = reinterpret_cast<const uint32_t*>(tr.mask + int64_t(row) * tr.words);
    const int w = o >> 5, end = 2 * tr.words;
    const uint32_t lo = w >= 0 && w < end ? m[w] : 0u, hi = w + 1 >= 0 && w + 1 < end ? m[w + 1] : 0u;
    return __funnelshift_r(lo, hi, o & 31);
}

// N consecutive values of a row as f32; vec: the address is aligned to the N values' size.
template <int N, typename T>
__device__ __forceinline__ void load_row(const T* p, bool vec, float (&x)[N]) {
    if constexpr (sizeof(T) * N == 16 || sizeof(T) * N == 8 || sizeof(T) * N == 4) {
        if (vec) {
            using V = typename std::conditional<sizeof(T) * N == 16, uint4,
                                                typename std::conditional<sizeof(T) * N == 8, uint2, uint32_t>::type>::type;
            alignas(16) T v[N];
            *reinterpret_cast<V*>(v) = *reinterpret_cast<const V*>(p);
#pragma unroll
            for (int i = 0; i < N; i++) x[i] = float(v[i]);
            return;
        }
    }
#pragma unroll
    for (int i = 0; i < N; i++) x[i] = float(p[i]);
}
template <int N, typename T>
__device__ __forceinline__ void store_row(T* p, bool vec, const float (&x)[N]) {
    alignas(16) T v[N];
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = T(x[i]);
    if constexpr (sizeof(T) * N == 16 || sizeof(T) * N == 8 || sizeof(T) * N == 4) {
        if (vec) {
            using V = typename std::conditional<sizeof(T) * N == 16, uint4,
                                                typename std::conditional<sizeof(T) * N == 8, uint2, uint32_t>::type>::type;
            *reinterpret_cast<V*>(p) = *reinterpret_cast<const V*>(v);
            return;
        }
    }
#pragma unroll
    for (int i = 0; i < N; i++) p[i] = v[i];
}

}  // namespace neko
