// C entries of the paged key/value cache (neko_op_paged_* in include/neko_cuda.h): the checks of the arguments.
#include "paged.cuh"

#include <algorithm>
#include <cmath>

using namespace neko;

namespace neko {
__device__ unsigned g_op_error = 0;
}

namespace {

int paged_fail(int code, const char* op, const char* why) {
    set_last_error(std::string(op) + ": " + why);
    return code;
}

bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// NULL when the cache's description is sound.
const char* bad_cache(const neko_paged_cache& c) {
    const bool q8 = c.type == NEKO_T_E4M3;
    if (!q8 && c.type != NEKO_T_F16) return "the cache is f16 or e4m3";
    if (!c.k_pages || !c.v_pages || !c.table) return "null cache pointer";
    if (q8 && (!c.k_scale || !c.v_scale)) return "an e4m3 cache needs its scales";
    if (c.n_seq < 0 || c.max_pages <= 0 || c.num_pages <= 0 || c.n_kv <= 0) return "cache sizes";
    if (c.page_size != 16 && c.page_size != 32 && c.page_size != 64 && c.page_size != 128)
        return "page size is 16, 32, 64 or 128";
    if (c.head_dim != 32 && c.head_dim != 64 && c.head_dim != 128) return "head dim is 32, 64 or 128";
    if (c.page_stride < int64_t(c.n_kv) * c.page_size * c.head_dim) return "pages overlap";
    if (!aligned(c.k_pages, 16) || !aligned(c.v_pages, 16) || (c.page_stride * (q8 ? 1 : 2)) % 16)
        return "pages must be 16-byte aligned";
    if (c.page_stride * (q8 ? 1 : 2) / 16 > 0xffffffffll) return "page stride of 64 GB or more";
    if (c.table_stride < c.max_pages) return "table stride below max_pages";
    if (q8 && c.scale_stride < c.n_kv) return "scale stride below n_kv";
    if (int64_t(c.max_pages) * c.page_size > (int64_t(1) << 30)) return "more than 2^30 positions per sequence";
    return nullptr;
}

bool real_type(int t) { return t == NEKO_T_F32 || t == NEKO_T_F16 || t == NEKO_T_BF16; }

int finish(const char* op, cudaError_t e) {
    if (e == cudaSuccess) return NEKO_OK;
    cudaGetLastError();
    set_last_error(cuda_msg(e, op));
    return NEKO_ERR_CUDA;
}

}  // namespace

static int append_call(const char* op, const neko_paged_append_args* a, const int32_t* depth, void* stream) {
    if (!a) return paged_fail(NEKO_ERR_ARG, op, "null arguments");
    if (const char* why = bad_cache(a->cache)) return paged_fail(NEKO_ERR_ARG, op, why);
    if (!real_type(a->type)) return paged_fail(NEKO_ERR_ARG, op, "q, k, v are f32, f16 or bf16");
    if (a->tokens < 0 || a->max_new < 0 || (a->q && a->n_head <= 0)) return paged_fail(NEKO_ERR_ARG, op, "sizes");
    if (a->tokens == 0 || a->max_new == 0 || a->cache.n_seq == 0) return NEKO_OK;
    if (!a->k || !a->v || !a->start || (a->q && !a->q_out)) return paged_fail(NEKO_ERR_ARG, op, "null pointer");
    if (!a->q_start && a->tokens != a->cache.n_seq)
        return paged_fail(NEKO_ERR_ARG, op, "without q_start there is one token per sequence");
    if (a->rot < 0 || a->rot > a->cache.head_dim || a->rot % 8)
        return paged_fail(NEKO_ERR_ARG, op, "rot is a multiple of 8 up to the head dim");
    if (a->rot && (!a->cs || a->cs_rows <= 0 || !aligned(a->cs, 16)))
        return paged_fail(NEKO_ERR_ARG, op, "a rotation needs its table (16-byte aligned)");
    // the rows of a page are addressed with 32 bits; the stride of a single row says nothing (a dimension of one may have any)
    for (const int64_t step : {a->q ? a->q_token : 0, a->k_token, a->v_token, a->q ? a->o_token : 0})
        if (a->tokens > 1 && (step >= (1 << 24) || step <= -(1 << 24)))
            return paged_fail(NEKO_ERR_UNSUPPORTED, op, "token strides of 2^24 elements or more");
    if (a->q && !a->q_gain != !a->k_gain) return paged_fail(NEKO_ERR_ARG, op, "both gains or neither");
    neko_paged_append_args own = *a;
    own.max_new = std::min(a->max_new, a->tokens);  // a sequence has no more than there are: a loose max_new costs nothing
    if (own.max_new / a->cache.page_size > 65530 || a->n_head > 65535 || a->cache.n_kv > 65535)  // the grid's second and third dimension
        return paged_fail(NEKO_ERR_UNSUPPORTED, op, "more than 65,530 pages of new tokens per sequence, or 65,535 heads");
    return finish(op, launch_paged_append(own, depth, static_cast<cudaStream_t>(stream)));
}

extern "C" int neko_op_paged_append(const neko_paged_append_args* a, void* stream) { return append_call("paged_append", a, nullptr, stream); }

extern "C" int neko_op_paged_tree_append(const neko_paged_append_args* a, const int32_t* depth, void* stream) {
    return append_call("paged_tree_append", a, depth, stream);
}

static int attention_call(const char* op, const neko_paged_attention_args* a, const neko_tree* tree, void* stream) {
    if (!a) return paged_fail(NEKO_ERR_ARG, op, "null arguments");
    if (const char* why = bad_cache(a->cache)) return paged_fail(NEKO_ERR_ARG, op, why);
    if (!real_type(a->type)) return paged_fail(NEKO_ERR_ARG, op, "q is f32, f16 or bf16");
    if (a->tokens < 0 || a->max_new < 0 || a->n_head <= 0 || a->n_head % a->cache.n_kv)
        return paged_fail(NEKO_ERR_ARG, op, "sizes (n_head is a multiple of n_kv)");
    if (a->tokens == 0 || a->max_new == 0 || a->cache.n_seq == 0) return NEKO_OK;
    if (!a->q || !a->out || !a->kv_len) return paged_fail(NEKO_ERR_ARG, op, "null pointer");
    if (!a->q_start && a->tokens != a->cache.n_seq)
        return paged_fail(NEKO_ERR_ARG, op, "without q_start there is one token per sequence");
    if (a->cache.n_seq > 16384) return paged_fail(NEKO_ERR_UNSUPPORTED, op, "more than 16384 sequences");
    // A sequence has no more rows than there are: a loose max_new costs nothing. The kernels count a KV head's rows (tokens x heads per KV
    // head) with 31 bits and divide them by the heads with a 32-bit reciprocal, exact below 2^32 / its excess over 1 / group.
    neko_paged_attention_args own = *a;
    own.max_new = std::min(a->max_new, a->tokens);
    const int64_t group = a->n_head / a->cache.n_kv, rows = own.max_new * group;
    const int64_t excess = ((int64_t(1) << 32) + group - 1) / group * group - (int64_t(1) << 32);
    if (rows > INT32_MAX - 1024 || rows * excess >= (int64_t(1) << 32))
        return paged_fail(NEKO_ERR_UNSUPPORTED, op, "2^31 rows (new tokens times heads per KV head) or more; fewer where those heads are no power of two");
    if (a->softcap == INFINITY) return paged_fail(NEKO_ERR_ARG, op, "softcap is finite (0: no cap)");
    if (a->window < 0 || !(a->softcap >= 0.0f) || !(a->scale == a->scale))
        return paged_fail(NEKO_ERR_ARG, op, "window and softcap are not negative");
    if (tree) {
        if (!tree->mask || !aligned(tree->mask, 8)) return paged_fail(NEKO_ERR_ARG, op, "a tree needs its masks (8-byte aligned)");
        if (int64_t(tree->words) * 64 < own.max_new) return paged_fail(NEKO_ERR_ARG, op, "fewer mask words than max_new nodes need");
        if (!tree->depth && (a->window || a->slopes)) return paged_fail(NEKO_ERR_ARG, op, "window and slopes need the nodes' depths");
        if (a->prefix) return paged_fail(NEKO_ERR_ARG, op, "no prefix with a tree");
    }
    return finish(op, launch_paged_attention(own, tree, static_cast<cudaStream_t>(stream)));
}

extern "C" int neko_op_paged_attention(const neko_paged_attention_args* a, void* stream) {
    return attention_call("paged_attention", a, nullptr, stream);
}

extern "C" int neko_op_paged_tree_attention(const neko_paged_attention_args* a, const neko_tree* tree, void* stream) {
    const char* op = "paged_tree_attention";
    if (!tree) return paged_fail(NEKO_ERR_ARG, op, "null tree");
    return attention_call(op, a, tree, stream);
}

extern "C" int neko_op_tree_masks(const int32_t* parent, const int32_t* q_start, int n_seq, int tokens, int max_new, uint64_t* mask, int words,
                                  int32_t* depth, void* stream) {
    const char* op = "tree_masks";
    if (n_seq < 0 || tokens < 0 || max_new < 0) return paged_fail(NEKO_ERR_ARG, op, "sizes");
    if (n_seq == 0 || tokens == 0 || max_new == 0 || (!mask && !depth)) return NEKO_OK;
    if (!parent || !q_start) return paged_fail(NEKO_ERR_ARG, op, "null pointer");
    max_new = std::min(max_new, tokens);
    if (max_new > NEKO_MAX_NODES) return paged_fail(NEKO_ERR_UNSUPPORTED, op, "more than 4096 nodes a sequence");
    if (n_seq > (1 << 30)) return paged_fail(NEKO_ERR_UNSUPPORTED, op, "more than 2^30 sequences");
    if (mask && (int64_t(words) * 64 < max_new || !aligned(mask, 8))) return paged_fail(NEKO_ERR_ARG, op, "mask words for max_new nodes, 8-byte aligned");
    return finish(op, launch_tree_masks(parent, q_start, n_seq, tokens, max_new, mask, words, depth, static_cast<cudaStream_t>(stream)));
}

extern "C" int neko_op_tree_accept(const int32_t* chosen, const int32_t* draft, const int32_t* parent, const int32_t* q_start, int n_seq,
                                   int tokens, int max_new, int32_t* path, int32_t* count, int32_t* token, void* stream) {
    const char* op = "tree_accept";
    if (n_seq < 0 || tokens < 0 || max_new < 0) return paged_fail(NEKO_ERR_ARG, op, "sizes");
    if (n_seq == 0) return NEKO_OK;
    if (!q_start || !path || !count || !token || (tokens && (!chosen || !draft || !parent))) return paged_fail(NEKO_ERR_ARG, op, "null pointer");
    if (max_new > NEKO_MAX_NODES) return paged_fail(NEKO_ERR_UNSUPPORTED, op, "more than 4096 nodes a sequence");
    return finish(op, launch_tree_accept(chosen, draft, parent, q_start, n_seq, tokens, max_new, path, count, token, static_cast<cudaStream_t>(stream)));
}

namespace {

const char* bad_planes(const neko_paged_planes& c) {
    const bool q8 = c.type == NEKO_T_E4M3;
    const int64_t size = q8 ? 1 : 2, page = int64_t(c.n_kv) * c.page_size * c.head_dim;
    if (!q8 && c.type != NEKO_T_F16) return "the cache is f16 or e4m3";
    if (!c.pages || (q8 && !c.scale)) return "null cache pointer";
    if (c.planes < 0 || c.n_seq < 0 || c.max_pages < 0 || c.num_pages <= 0 || c.n_kv <= 0) return "cache sizes";
    if (c.page_size != 16 && c.page_size != 32 && c.page_size != 64 && c.page_size != 128) return "page size is 16, 32, 64 or 128";
    if (c.head_dim != 32 && c.head_dim != 64 && c.head_dim != 128) return "head dim is 32, 64 or 128";
    if (c.page_stride < page || (c.planes > 1 && c.plane_stride < page)) return "pages overlap";
    if (!aligned(c.pages, 16) || c.page_stride * size % 16 || (c.planes > 1 && c.plane_stride * size % 16)) return "pages must be 16-byte aligned";
    if (q8 && (c.scale_stride < c.n_kv || (c.planes > 1 && c.scale_plane < c.n_kv))) return "scales overlap";
    if (c.planes > 65535) return "more than 65,535 planes";
    return nullptr;
}

}  // namespace

extern "C" int neko_op_paged_compact(const neko_paged_planes* c, const int32_t* start, const int32_t* path, int64_t path_stride,
                                     const int32_t* count, int max_count, void* stream) {
    const char* op = "paged_compact";
    if (!c) return paged_fail(NEKO_ERR_ARG, op, "null arguments");
    if (const char* why = bad_planes(*c)) return paged_fail(NEKO_ERR_ARG, op, why);
    if (max_count < 0 || (max_count && path_stride < max_count)) return paged_fail(NEKO_ERR_ARG, op, "rows of path overlap");
    if (c->planes == 0 || c->n_seq == 0 || max_count == 0 || c->max_pages == 0) return NEKO_OK;
    if (!c->table || !start || !path || !count) return paged_fail(NEKO_ERR_ARG, op, "null pointer");
    if (c->table_stride < c->max_pages) return paged_fail(NEKO_ERR_ARG, op, "table stride below max_pages");
    if (int64_t(c->max_pages) * c->page_size > (int64_t(1) << 30)) return paged_fail(NEKO_ERR_ARG, op, "more than 2^30 positions per sequence");
    if (c->n_kv > 65535) return paged_fail(NEKO_ERR_UNSUPPORTED, op, "more than 65,535 heads");
    return finish(op, launch_paged_compact(*c, start, path, path_stride, count, max_count, static_cast<cudaStream_t>(stream)));
}

extern "C" int neko_op_paged_copy(const neko_paged_planes* c, const int32_t* src, const int32_t* dst, int n, void* stream) {
    const char* op = "paged_copy";
    if (!c) return paged_fail(NEKO_ERR_ARG, op, "null arguments");
    if (const char* why = bad_planes(*c)) return paged_fail(NEKO_ERR_ARG, op, why);
    if (n < 0) return paged_fail(NEKO_ERR_ARG, op, "sizes");
    if (n == 0 || c->planes == 0) return NEKO_OK;
    if (!src || !dst) return paged_fail(NEKO_ERR_ARG, op, "null pointer");
    return finish(op, launch_paged_copy(*c, src, dst, n, static_cast<cudaStream_t>(stream)));
}

extern "C" int neko_op_sample_rows(const neko_sample_rows_args* a, void* stream) {
    const char* op = "sample_rows";
    if (!a) return paged_fail(NEKO_ERR_ARG, op, "null arguments");
    if (!real_type(a->type)) return paged_fail(NEKO_ERR_ARG, op, "logits are f32, f16 or bf16");
    if (a->rows < 0 || a->vocab <= 0) return paged_fail(NEKO_ERR_ARG, op, "sizes");
    if (a->rows == 0) return NEKO_OK;
    if (!a->logits || !a->token) return paged_fail(NEKO_ERR_ARG, op, "null pointer");
    if (!aligned(a->logits, a->type == NEKO_T_F32 ? 4 : 2)) return paged_fail(NEKO_ERR_ARG, op, "logits must be aligned to their type");
    if (a->vocab > NEKO_MAX_VOCAB) return paged_fail(NEKO_ERR_UNSUPPORTED, op, "a vocabulary of more than 262,144 tokens");
    if (a->rows > (1 << 24)) return paged_fail(NEKO_ERR_UNSUPPORTED, op, "more than 2^24 rows");
    if (!a->u && (a->temperatures || a->temperature > 0.0f)) return paged_fail(NEKO_ERR_ARG, op, "sampling needs its numbers");
    return finish(op, launch_sample_rows(*a, static_cast<cudaStream_t>(stream)));
}

extern "C" int neko_op_status(void* stream) {
    const char* op = "op_status";
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    unsigned code = 0;
    cudaError_t e = cudaMemcpyFromSymbolAsync(&code, g_op_error, sizeof code, 0, cudaMemcpyDeviceToHost, st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    if (e != cudaSuccess || code == kErrNone) return finish(op, e);
    const unsigned none = kErrNone;
    e = cudaMemcpyToSymbolAsync(g_op_error, &none, sizeof none, 0, cudaMemcpyHostToDevice, st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    if (e != cudaSuccess) return finish(op, e);
    return paged_fail(NEKO_ERR_DEVICE, op,
                      code == kErrBadIndex ? "a sequence of a paged call had more new tokens than max_new (or a path more than max_count), "
                                             "rows outside `tokens`, or positions past the rotation table; those rows were left out"
                      : code == kErrMbarTimeout ? "a bounded wait of a paged kernel gave up; its output is not valid"
                                                : "a paged kernel found its shared memory misaligned and did nothing");
}

extern "C" int neko_op_trim(size_t keep_bytes) { return finish("op_trim", scratch_trim(keep_bytes)); }
