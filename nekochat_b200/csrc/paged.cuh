// The paged key/value cache's kernels' arguments and small device helpers (k_paged.cu, k_paged_attn.cu).
#pragma once
#include <cuda_bf16.h>

#include "mma_frag.cuh"
#include "neko_common.cuh"
#include "neko_internal.h"

namespace neko {

enum PagedType : int { kTF32 = NEKO_T_F32, kTF16 = NEKO_T_F16, kTBF16 = NEKO_T_BF16, kTE4M3 = NEKO_T_E4M3 };
constexpr int kScaleMinExp = -100;  // scale of a block of zeros: 2^-100

cudaError_t launch_paged_append(const neko_paged_append_args& a, cudaStream_t st);
cudaError_t launch_paged_attention(const neko_paged_attention_args& a, cudaStream_t st);
// The tcgen05 kernel, head dim 64 or 128; launch_paged_attention says when (packed rows: new tokens x query heads per KV head).
cudaError_t launch_paged_prompt(const neko_paged_attention_args& a, cudaStream_t st);
constexpr int kPromptRows = 16;

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
