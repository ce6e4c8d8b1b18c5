// Bookkeeping of trees of drafted tokens (neko_op_tree_masks, neko_op_tree_accept): a CTA for each sequence, its nodes in shared
// memory. Both are bound by latency: a chain of dependent reads as long as the tree is deep, in shared memory instead of L2 (12 nodes:
// 4.7 us for both kernels from a graph; 128 trees of 17 to 64: 6.5). Each node walks to its root, so a line of n nodes costs the masks
// n / 128 such walks one after the other: 512 nodes 0.14 ms, 4,096 7.7 ms.
#include <algorithm>

#include "paged.cuh"

namespace neko {

namespace {

constexpr int kThreads = 128;

// The sequence's first row and its number of nodes; false: it is left out, with more than max_new or rows that are not there.
__device__ __forceinline__ bool rows_of(const int32_t* q_start, int s, int tokens, int max_new, int& row0, int& n) {
    row0 = q_start[s], n = q_start[s + 1] - row0;
    return row0 >= 0 && n >= 0 && n <= max_new && row0 <= tokens - n;
}
// The same; false: none, or left out (reported, n < 0).
__device__ __forceinline__ bool nodes_of(const int32_t* q_start, int s, int tokens, int max_new, int& row0, int& n) {
    if (!rows_of(q_start, s, tokens, max_new, row0, n)) {
        if (threadIdx.x == 0) set_op_error(kErrBadIndex);
        n = -1;
    }
    return n > 0;
}

// A thread for each node walks up to the root. Parents come before their children, so the bits of the node's words come from the
// last to the first: each word is written once, from a register. The CTAs behind the sequences' set the rows of no sequence to
// zero, which costs less than a fill before the kernel. Where the starts go down somewhere, sequences that are there may lie among the
// rows that are to be cleared: each row is looked for in all of them then.
__global__ void __launch_bounds__(kThreads) tree_masks_kernel(const int32_t* __restrict__ parent, const int32_t* __restrict__ q_start, int n_seq,
                                                             int tokens, int max_new, uint64_t* __restrict__ mask, int words, int32_t* __restrict__ depth) {
    extern __shared__ int32_t up[];
    // whether the starts go down anywhere
    auto unordered = [&]() {
        int down = 0;
        for (int i = threadIdx.x; i < n_seq; i += kThreads) down |= q_start[i + 1] < q_start[i];
        return __syncthreads_or(down) != 0;
    };
    // rows [from, to), by this CTA of `many`
    auto clear = [&](int from, int to, int cta, int many, bool mixed) {
        from = max(from, 0), to = min(to, tokens);
        if (from >= to) return;
        const int64_t at = int64_t(cta) * kThreads + threadIdx.x, step = int64_t(many) * kThreads;
        if (mixed) {
            for (int64_t row = from + at; row < to; row += step) {
                bool free = true;
                for (int s = 0; s < n_seq && free; s++) {
                    int first, count;
                    free = !rows_of(q_start, s, tokens, max_new, first, count) || row < first || row >= first + count;
                }
                if (free && mask)
                    for (int w = 0; w < words; w++) mask[row * words + w] = 0;
                if (free && depth) depth[row] = 0;
            }
            return;
        }
        if (mask)
            for (int64_t i = int64_t(from) * words + at; i < int64_t(to) * words; i += step) mask[i] = 0;
        if (depth)
            for (int64_t i = from + at; i < to; i += step) depth[i] = 0;
    };
    if (blockIdx.x >= n_seq) {
        const int cta = blockIdx.x - n_seq, many = gridDim.x - n_seq;
        const bool mixed = unordered();
        clear(0, q_start[0], cta, many, mixed);
        clear(q_start[n_seq], tokens, cta, many, mixed);
        return;
    }
    int row0, n;
    if (!nodes_of(q_start, blockIdx.x, tokens, max_new, row0, n)) {
        if (n < 0) {
            const bool mixed = unordered();
            clear(row0, q_start[blockIdx.x + 1], 0, 1, mixed);
        }
        return;
    }
    for (int i = threadIdx.x; i < n; i += kThreads) up[i] = parent[row0 + i];
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads) {
        uint64_t* out = mask ? mask + int64_t(row0 + i) * words : nullptr;
        int w = words - 1, deep = -1;
        uint64_t bits = 0;
        for (int at = i;;) {
            if (out)
                for (; w > at >> 6; w--) out[w] = bits, bits = 0;
            bits |= uint64_t(1) << (at & 63);
            deep++;
            const int p = up[at];
            if (p < 0 || p >= at) break;
            at = p;
        }
        if (out)
            for (; w >= 0; w--) out[w] = bits, bits = 0;
        if (depth) depth[row0 + i] = deep;
    }
}

// Where each node leads is found for all nodes at once (the lowest child whose draft is the token chosen here); one thread walks.
__global__ void __launch_bounds__(kThreads) tree_accept_kernel(const int32_t* __restrict__ chosen, const int32_t* __restrict__ draft,
                                                              const int32_t* __restrict__ parent, const int32_t* __restrict__ q_start,
                                                              int tokens, int max_new, int32_t* __restrict__ path, int32_t* __restrict__ count,
                                                              int32_t* __restrict__ token) {
    extern __shared__ int32_t next[];  // [max_new], then the path
    int32_t* walk = next + max_new;
    __shared__ int steps;
    const int s = blockIdx.x;
    int row0, n;
    const bool any = nodes_of(q_start, s, tokens, max_new, row0, n);
    for (int i = threadIdx.x; i < n; i += kThreads) next[i] = 0x7fffffff;
    if (threadIdx.x == 0) steps = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const int p = parent[row0 + i];
        if (p >= 0 && p < i && draft[row0 + i] == chosen[row0 + p]) atomicMin(&next[p], i);
    }
    __syncthreads();
    if (threadIdx.x == 0 && any) {
        int k = 0;
        for (int at = 0; at < n; at = next[at]) walk[k++] = at;  // ascending: ends
        steps = k;
        token[s] = chosen[row0 + walk[k - 1]];
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        count[s] = steps;
        if (!any) token[s] = -1;
    }
    for (int k = threadIdx.x; k < max_new; k += kThreads) path[int64_t(s) * max_new + k] = k < steps ? walk[k] : 0;
}

}  // namespace

cudaError_t launch_tree_masks(const int32_t* parent, const int32_t* q_start, int n_seq, int tokens, int max_new, uint64_t* mask, int words,
                              int32_t* depth, cudaStream_t st) {
    const int64_t blank = std::min<int64_t>((int64_t(tokens) * (mask ? words : 1) + 4095) / 4096, num_sms());  // words counts with a mask only
    return launch_ex(tree_masks_kernel, dim3(unsigned(n_seq + blank)), dim3(kThreads), size_t(max_new) * 4, st, false, parent, q_start, n_seq, tokens,
                     max_new, mask, words, depth);
}

cudaError_t launch_tree_accept(const int32_t* chosen, const int32_t* draft, const int32_t* parent, const int32_t* q_start, int n_seq,
                               int tokens, int max_new, int32_t* path, int32_t* count, int32_t* token, cudaStream_t st) {
    return launch_ex(tree_accept_kernel, dim3(n_seq), dim3(kThreads), size_t(max_new) * 8, st, false, chosen, draft, parent, q_start, tokens, max_new,
                     path, count, token);
}

}  // namespace neko
