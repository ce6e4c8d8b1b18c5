// Tokens from rows of logits with temperature, top-k, top-p and min-p (neko_op_sample_rows).
//
// A cluster of CTAs takes a row: each holds its slice in shared memory, so the logits are read from memory once whatever follows.
// Weights 2^(44 - y), y = (max - x) log2(e) / temperature, are rounded to integers and added as integers: sums do not depend on an
// order, and any split of a row gives the same token. They are computed in 64 bits (a table of 512 powers and a cubic): with V
// tokens of about equal weight a row's number falls within 2^-24 of a border once in 2^24 / V rows, so f32 sums would choose
// otherwise than the definition now and then.
//
// What is kept is a beginning of the row in descending order, found without sorting the row:
//  * the largest values of 64 groups of threads a CTA bound the r-th largest of the row from below (the r-th largest of them), and few
//    more than r tokens reach that bound: they are collected in one CTA, ranked by counting and cut there. Enough for top-k up to
//    three quarters of the groups, and for top-p where the collected tokens hold that much of the sum.
//  * else a histogram over equal steps of max - x, of counts or of weights in three pieces of 15 bits (32-bit additions in shared memory),
//    added up over the cluster, gives the step that the cut falls into; its tokens are collected and ranked, or where they are
//    too many the key's digits (11, 11 and 10 bits) lead to the cut's value, whose equals are cut by index.
// The draw goes through the slices in the order of the vocabulary: sums of CTAs, of warps' segments, of lanes.
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "paged.cuh"

namespace cg = cooperative_groups;

namespace neko {

namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kGroups = kThreads / 8;  // groups of threads whose largest values are known
constexpr int kCand = 1024;            // tokens that are ranked by counting
constexpr int kBins = 2048;
constexpr int kTable = 512;
constexpr int kMaxCluster = 8;
constexpr double kOne = 17592186044416.0;  // 2^44: the weight of the largest
constexpr int kSmemAux = 4 * kBins * 4;    // histograms, or the lists
static_assert(4 * kCand * 8 <= kSmemAux, "the lists take the histograms' place");

// The order of values as unsigned numbers; zeros are alike.
__device__ __forceinline__ uint32_t order_key(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k); }

template <typename T>
__device__ __forceinline__ float value_of(T v) {
    return float(v);
}

// What the threads of a row share. Lists are ordered by key (value, then lower index): (order_key << 32) | ~index.
struct Shared {
    double table[kTable];            // 2^(i / 512)
    float gmax[kMaxCluster * kGroups];
    unsigned long long sum[kMaxCluster];  // by CTA: of weights or counts
    unsigned long long warp_sum[kWarps];
    unsigned long long cut;          // tokens from here up (in the lists' order) are kept
    unsigned long long before, total;
    unsigned best, found;            // lowest index
    unsigned n_list, n_all, at_list; // tokens in this CTA's list, in the owner's, and where this CTA's begin there
    int bin, done;
    float pick;
    uint64_t bar;
};

struct Row {
    float m;        // largest value
    double c;       // log2(e) / temperature
    double lim;     // y up to this is kept (min-p)
};

// 2^(44 - y) to the nearest integer.
__device__ __forceinline__ double weight(const Row& r, const double* table, float x) {
    const double d = x == r.m ? 0.0 : double(r.m) - double(x);
    const double v = fma(-d, r.c, 44.0);
    if (!(v >= -1.0)) return 0.0;
    const double t = fma(v, double(kTable), 6755399441055744.0);  // + 1.5 * 2^52: the integer in the low word
    const int n = __double2loint(t);
    const double f = fma(t - 6755399441055744.0, -1.0 / kTable, v);
    double p = fma(f, 0.05550410866482158, 0.2402265069591007);  // ln2^3 / 6, ln2^2 / 2
    p = fma(p, f, 0.6931471805599453);
    const double w = table[n & (kTable - 1)];
    const double s = __hiloint2double(__double2hiint(w) + ((n >> 9) << 20), __double2loint(w));
    return (fma(p * f, s, s) + 4503599627370496.0) - 4503599627370496.0;  // 2^52
}
__device__ __forceinline__ bool within(const Row& r, float x) { return (x == r.m ? 0.0 : double(r.m) - double(x)) * r.c <= r.lim; }

__device__ __forceinline__ unsigned long long warp_total(unsigned long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ unsigned long long warp_upto(unsigned long long v, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long t = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += t;
    }
    return v;
}
// Sums up to and with each of `per` consecutive values a thread, in place.
template <int kPer>
__device__ __forceinline__ void cta_upto(Shared& sh, unsigned long long (&v)[kPer]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int i = 1; i < kPer; i++) v[i] += v[i - 1];
    const unsigned long long upto = warp_upto(v[kPer - 1], lane);
    __syncthreads();
    if (lane == 31) sh.warp_sum[warp] = upto;
    __syncthreads();
    unsigned long long before = upto - v[kPer - 1];
    for (int w = 0; w < warp; w++) before += sh.warp_sum[w];
#pragma unroll
    for (int i = 0; i < kPer; i++) v[i] += before;
}

template <typename T>
struct Sampler {
    static constexpr int kPer = 16 / sizeof(T);  // values of a 16-byte vector
    const neko_sample_rows_args& a;
    cg::cluster_group cluster;
    Shared& sh;
    uint8_t* aux;
    const uint4* data;
    int ctas, rank, nv, first;  // vectors of this CTA's slice; vocabulary index of the first vector's first place
    Row row;

    __device__ Sampler(const neko_sample_rows_args& a_, Shared& s, uint8_t* x) : a(a_), cluster(cg::this_cluster()), sh(s), aux(x) {}

    // f(value, index) of every value of the slice, by vectors of this thread. Places outside the row hold -infinity.
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        for (int v = threadIdx.x; v < nv; v += kThreads) {
            const uint4 w = data[v];
            const T* x = reinterpret_cast<const T*>(&w);
#pragma unroll
            for (int j = 0; j < kPer; j++) f(value_of(x[j]), first + v * kPer + j);
        }
    }
    __device__ __forceinline__ static unsigned long long entry(float x, int i) {
        return (static_cast<unsigned long long>(order_key(x)) << 32) | (0xFFFFFFFFu - unsigned(i));
    }
    // Values that can be taken at all: not NaN, not -infinity.
    __device__ __forceinline__ static bool real(float x) { return x > -INFINITY; }

    // The slices' sums meet: sum[i] of every CTA.
    __device__ void share_sum(unsigned long long v) {
        if (threadIdx.x < ctas) *cluster.map_shared_rank(&sh.sum[rank], threadIdx.x) = v;
        cluster.sync();
    }

    // The tokens for which take(value, index) holds come together in CTA 0's list (aux); n_all says how many there are, the
    // first kCand of them are in it.
    template <typename F, typename G>
    __device__ void collect(F take, G then) {
        unsigned long long* mine = reinterpret_cast<unsigned long long*>(aux) + kCand;
        unsigned long long* list = cluster.map_shared_rank(reinterpret_cast<unsigned long long*>(aux), 0);
        if (threadIdx.x == 0) sh.n_list = 0;
        __syncthreads();
        each([&](float x, int i) {
            if (take(x, i)) {
                const unsigned at = atomicAdd(&sh.n_list, 1u);
                if (at < kCand) mine[at] = entry(x, i);
            }
        });
        __syncthreads();
        const unsigned n = sh.n_list;
        if (threadIdx.x == 0) sh.at_list = atomicAdd(cluster.map_shared_rank(&sh.n_all, 0), n);
        __syncthreads();
        for (unsigned i = threadIdx.x; i < min(n, unsigned(kCand)); i += kThreads)
            if (sh.at_list + i < kCand) list[sh.at_list + i] = mine[i];
        then();
        cluster.sync();
    }

    // CTA 0's list in descending order (into the second list), and sums of measure(entry) up to and with each (the third).
    template <typename F>
    __device__ void rank_list(int n, F measure) {
        unsigned long long* list = reinterpret_cast<unsigned long long*>(aux);
        unsigned long long *sorted = list + kCand, *upto = list + 2 * kCand;
        for (int i = threadIdx.x; i < n; i += kThreads) {
            const unsigned long long e = list[i];
            int r = 0;
            for (int j = 0; j < n; j++) r += list[j] > e;
            sorted[r] = e;
        }
        __syncthreads();
        unsigned long long v[2];
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const int i = 2 * threadIdx.x + k;
            v[k] = i < n ? measure(sorted[i]) : 0ull;
        }
        cta_upto(sh, v);
#pragma unroll
        for (int k = 0; k < 2; k++)
            if (2 * threadIdx.x + k < n) upto[2 * threadIdx.x + k] = v[k];
        __syncthreads();
    }
    __device__ __forceinline__ unsigned long long weight_of(unsigned long long e) const {
        return static_cast<unsigned long long>(weight(row, sh.table, key_value(uint32_t(e >> 32))));
    }
    // How many of the n sums, each with what lies ahead, are below target.
    __device__ int below(const unsigned long long* upto, int n, double target, unsigned long long ahead) {
        int c = 0;
        for (int base = 0; base < n; base += kThreads)
            c += __syncthreads_count(base + threadIdx.x < n && double(ahead + upto[base + threadIdx.x]) < target);
        return c;
    }

    __device__ void answer(int r, int token, float x, unsigned long long total) {
        a.token[r] = token;
        if (a.prob) a.prob[r] = token < 0 ? 0.0f : float(exp2(-(x == row.m ? 0.0 : (double(row.m) - double(x)) * row.c)) * (kOne / double(total)));
    }
    // floor(u * total), below total.
    __device__ unsigned long long place(int r, unsigned long long total) {
        const double x = a.u[r] * double(total);
        const unsigned long long p = x > 0.0 ? static_cast<unsigned long long>(x) : 0ull;
        return min(p, total - 1);
    }

    // The first index, in the order of the vocabulary, at which the sum of measure(value, index) exceeds where(total): its CTA
    // gets found = index, pick = value; total to all. Sums of warps' segments of the slice, then of 32 vectors at a time.
    template <typename M, typename P>
    __device__ unsigned long long find(M measure, P where) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, seg = (nv + kWarps - 1) / kWarps;
        const int v0 = min(warp * seg, nv), v1 = min(v0 + seg, nv);
        double part = 0.0;  // of integers, exact
        for (int v = v0 + lane; v < v1; v += 32) {
            const uint4 w = data[v];
            const T* x = reinterpret_cast<const T*>(&w);
#pragma unroll
            for (int j = 0; j < kPer; j++) part += measure(value_of(x[j]), first + v * kPer + j);
        }
        const unsigned long long of_warp = warp_total(static_cast<unsigned long long>(part));
        if (threadIdx.x == 0) sh.found = 0xFFFFFFFFu;
        __syncthreads();
        if (lane == 0) sh.warp_sum[warp] = of_warp;
        __syncthreads();
        unsigned long long mine = 0, before = 0, total = 0;
        for (int w = 0; w < kWarps; w++) mine += sh.warp_sum[w];
        share_sum(mine);
        for (int i = 0; i < ctas; i++) {
            if (i < rank) before += sh.sum[i];
            total += sh.sum[i];
        }
        const unsigned long long at = where(total);
        for (int w = 0; w < warp; w++) before += sh.warp_sum[w];
        if (total && at >= before && at < before + of_warp) {  // one warp of the cluster
            for (int base = v0; base < v1; base += 32) {
                const int v = base + lane;
                unsigned long long s = 0;
                uint4 w = make_uint4(0, 0, 0, 0);
                const T* x = reinterpret_cast<const T*>(&w);
                if (v < v1) {
                    w = data[v];
#pragma unroll
                    for (int j = 0; j < kPer; j++) s += static_cast<unsigned long long>(measure(value_of(x[j]), first + v * kPer + j));
                }
                const unsigned long long upto = warp_upto(s, lane);
                if (before + upto > at && before + upto - s <= at) {  // one lane
                    unsigned long long sum = before + upto - s;
                    for (int j = 0; j < kPer; j++) {
                        sum += static_cast<unsigned long long>(measure(value_of(x[j]), first + v * kPer + j));
                        if (sum > at) {
                            sh.found = unsigned(first + v * kPer + j);
                            sh.pick = value_of(x[j]);
                            break;
                        }
                    }
                }
                before += __shfl_sync(0xffffffffu, upto, 31);
                if (before > at) break;
            }
        }
        __syncthreads();
        return total;
    }

    // Adds up a histogram over the cluster and finds the bin at which the sum reaches target(total of all bins, with what lies
    // before them): bin (-1: none does), before (without the bin), total to every CTA.
    template <bool MASS, typename F, typename G>
    __device__ void histogram(F bin_of, unsigned long long ahead, G target) {
        uint32_t* h = reinterpret_cast<uint32_t*>(aux);
        for (int i = threadIdx.x; i < (MASS ? 3 : 1) * kBins; i += kThreads) h[i] = 0;
        __syncthreads();
        each([&](float x, int i) {
            const int b = bin_of(x, i);
            if (b < 0) return;
            if constexpr (MASS) {
                const unsigned long long w = static_cast<unsigned long long>(weight(row, sh.table, x));
                const uint32_t p0 = uint32_t(w) & 0x7fffu, p1 = uint32_t(w >> 15) & 0x7fffu, p2 = uint32_t(w >> 30);
                if (p0) atomicAdd(&h[b], p0);
                if (p1) atomicAdd(&h[kBins + b], p1);
                if (p2) atomicAdd(&h[2 * kBins + b], p2);
            } else {
                atomicAdd(&h[b], 1u);
            }
        });
        cluster.sync();
        // this CTA's share of the bins, kBins / ctas of them: four at most a thread
        const int share = kBins / ctas, per = (share + kThreads - 1) / kThreads;
        unsigned long long v[4] = {0, 0, 0, 0};
        for (int c = 0; c < ctas; c++) {
            const uint32_t* o = cluster.map_shared_rank(h, c) + rank * share;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int b = threadIdx.x * per + k;
                if (k >= per || b >= share) continue;
                v[k] += o[b];
                if (MASS) v[k] += (static_cast<unsigned long long>(o[kBins + b]) << 15) + (static_cast<unsigned long long>(o[2 * kBins + b]) << 30);
            }
        }
        unsigned long long own[4];
#pragma unroll
        for (int k = 0; k < 4; k++) own[k] = v[k];
        cta_upto(sh, v);
        __syncthreads();
        unsigned long long all = 0;
        for (int w = 0; w < kWarps; w++) all += sh.warp_sum[w];
        if (threadIdx.x == 0) sh.bin = -1;
        share_sum(all);
        unsigned long long before = ahead, total = ahead;
        for (int i = 0; i < ctas; i++) {
            if (i < rank) before += sh.sum[i];
            total += sh.sum[i];
        }
        const double want = target(total);
        // one thread of the cluster has the bin that reaches it
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const unsigned long long upto = before + v[k], less = upto - own[k];
            if (own[k] && double(upto) >= want && double(less) < want) {
                for (int c = 0; c < ctas; c++) {
                    Shared* o = cluster.map_shared_rank(&sh, c);
                    o->bin = rank * share + int(threadIdx.x) * per + k;
                    o->before = less;
                }
            }
        }
        if (threadIdx.x == 0) sh.total = total;
        cluster.sync();
    }

    // Moves the cut (among what the present one keeps) to the first token, in descending order, at which the sum of the counts
    // (COUNT) or weights reaches want(total).
    template <bool MASS, typename G>
    __device__ void select(G want_of) {
        const unsigned long long cut = sh.cut;
        const float scale = fminf(64.0f * fmaxf(float(fmin(row.c, 1e30)), 1.0f), 1e30f);
        auto step_of = [&](float x, int i) {
            if (!real(x) || entry(x, i) < cut) return -1;
            return x == row.m ? 0 : int(fminf((row.m - x) * scale, float(kBins - 1)));
        };
        if (threadIdx.x == 0) sh.n_all = 0;
        histogram<MASS>(step_of, 0, want_of);
        const int step = sh.bin;
        if (step < 0) return;  // fewer than that many
        unsigned long long before = sh.before;
        const double want = want_of(sh.total);
        collect([&](float x, int i) { return step_of(x, i) == step; }, []() {});
        if (rank == 0) {
            const int n = int(min(sh.n_all, unsigned(kCand) + 1u));
            unsigned long long next = 0;
            if (n <= kCand) {
                unsigned long long* list = reinterpret_cast<unsigned long long*>(aux);
                rank_list(n, [&](unsigned long long e) { return MASS ? weight_of(e) : 1ull; });
                next = list[kCand + min(below(list + 2 * kCand, n, want, before), n - 1)];
            }
            if (threadIdx.x < ctas) {
                Shared* o = cluster.map_shared_rank(&sh, threadIdx.x);
                o->done = next != 0;
                if (next) o->cut = next;
            }
        }
        cluster.sync();
        if (sh.done) return;
        // too many tokens in one step: by the digits of their keys
        uint32_t key = 0, known = 0;
        for (int digit = 0; digit < 3; digit++) {
            const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0;
            const uint32_t most = digit == 2 ? 1023u : 2047u;
            histogram<MASS>([&](float x, int i) {
                const uint32_t k = order_key(x);
                return step_of(x, i) == step && (k & known) == key ? int(most - (k >> shift & most)) : -1;
            }, before, [&](unsigned long long) { return want; });
            before = sh.before;
            key |= (most - uint32_t(max(sh.bin, 0))) << shift;
            known |= most << shift;
        }
        const double each_one = MASS ? weight(row, sh.table, key_value(key)) : 1.0;
        const double more = ceil((want - double(before)) / each_one);
        find([&](float x, int i) { return step_of(x, i) == step && order_key(x) == key ? 1.0 : 0.0; },
             [&](unsigned long long total) { return more > 1.0 ? min(static_cast<unsigned long long>(more) - 1, total - 1) : 0ull; });
        if (threadIdx.x == 0 && sh.found != 0xFFFFFFFFu) {
            const unsigned long long next = (static_cast<unsigned long long>(key) << 32) | (0xFFFFFFFFu - sh.found);
            for (int c = 0; c < ctas; c++) cluster.map_shared_rank(&sh, c)->cut = next;
        }
        cluster.sync();
    }

    // The cut by the largest values alone (see above); true: the row is answered.
    __device__ bool few(int r, float t, int top_k, bool use_p, float top_p) {
        double part = 0.0;
        if (threadIdx.x == 0) sh.done = 0;
        collect([&](float x, int) {
            if (!top_k && real(x)) part += weight(row, sh.table, x);
            return x >= t && real(x);
        }, [&]() {
            if (top_k) return;
            const unsigned long long s = warp_total(static_cast<unsigned long long>(part));
            if ((threadIdx.x & 31) == 0) atomicAdd(cluster.map_shared_rank(&sh.total, 0), s);
        });
        if (rank == 0 && sh.n_all <= kCand) {
            unsigned long long *sorted = reinterpret_cast<unsigned long long*>(aux) + kCand, *upto = sorted + kCand, *w = upto + kCand;
            const int n = int(sh.n_all), n_k = top_k ? min(top_k, n) : n;
            rank_list(n, [&](unsigned long long e) { return weight_of(e); });
            int n_p = n_k;
            bool sure = top_k != 0;
            if (use_p) {
                const unsigned long long total = top_k ? upto[n_k - 1] : sh.total;
                const int less = below(upto, n_k, fmax(double(top_p) * double(total), 0.5), 0);
                if (less < n_k) n_p = less + 1, sure = true;
            }
            int n_m = 0;
            for (int base = 0; base < n_p; base += kThreads) {
                const int i = base + threadIdx.x;
                n_m += __syncthreads_count(i < n_p && within(row, key_value(uint32_t(sorted[i < n_p ? i : 0] >> 32))));
            }
            sure |= n_m < n_p;
            if (sure) {
                const unsigned long long total = upto[n_m - 1], at = place(r, total);
                for (int i = threadIdx.x; i < n_m; i += kThreads) w[i] = upto[i] - (i ? upto[i - 1] : 0ull);
                __syncthreads();
                for (int i = threadIdx.x; i < n_m; i += kThreads) {
                    const uint32_t low = uint32_t(sorted[i]);  // ~index
                    unsigned long long before = 0;
                    for (int j = 0; j < n_m; j++) before += uint32_t(sorted[j]) > low ? w[j] : 0ull;
                    if (at >= before && at < before + w[i]) answer(r, int(0xFFFFFFFFu - low), key_value(uint32_t(sorted[i] >> 32)), total);
                }
                if (threadIdx.x < ctas) cluster.map_shared_rank(&sh, threadIdx.x)->done = 1;
            }
        }
        cluster.sync();
        return sh.done != 0;
    }
};

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) sample_rows_kernel(const neko_sample_rows_args a, int slice) {
    using S = Sampler<T>;
    extern __shared__ __align__(128) uint8_t sm[];
    Shared& sh = *reinterpret_cast<Shared*>(sm);
    constexpr int kAuxOff = (sizeof(Shared) + 127) / 128 * 128;
    S s(a, sh, sm + kAuxOff);
    uint8_t* buf = sm + kAuxOff + kSmemAux;
    const int tid = threadIdx.x, lane = tid & 31;
    s.ctas = int(s.cluster.num_blocks()), s.rank = int(s.cluster.block_rank());
    const int r = blockIdx.x / s.ctas, ctas = s.ctas;
    const int b = min(s.rank * slice, a.vocab), n = min(slice, a.vocab - b);
    const T* src = static_cast<const T*>(a.logits) + r * a.row_stride + b;
    const int ph = int(reinterpret_cast<uintptr_t>(src) & 15) / int(sizeof(T));  // places before the slice in its first vector
    const int head = min(n, (S::kPer - ph) % S::kPer), body = (n - head) / S::kPer * S::kPer;
    s.nv = n ? (ph + n + S::kPer - 1) / S::kPer : 0;
    s.first = b - ph;
    s.data = reinterpret_cast<const uint4*>(buf);
    if (tid == 0) {
        mbar_init(&sh.bar, 1);
        fence_barrier_init();
        const uint32_t bytes = uint32_t(body) * sizeof(T);
        mbar_arrive_expect_tx(&sh.bar, bytes);
        for (uint32_t o = 0; o < bytes; o += 16384)
            bulk_g2s(buf + (ph + head) * sizeof(T) + o, reinterpret_cast<const uint8_t*>(src + head) + o, min(bytes - o, 16384u), &sh.bar);
        sh.best = 0xFFFFFFFFu, sh.n_all = 0, sh.total = 0, sh.cut = 0;
    }
    {
        T* x = reinterpret_cast<T*>(buf);
        const T none = T(-INFINITY);
        if (tid < ph) x[tid] = none;
        if (tid < head) x[ph + tid] = src[tid];
        const int at = head + body + tid;  // the last, partly filled vector
        if (tid < S::kPer && ph + at < s.nv * S::kPer) x[ph + at] = at < n ? src[at] : none;
    }
    sh.table[tid] = exp2(double(tid) / kTable);
    s.cluster.barrier_arrive();
    __syncthreads();
    bool ok = false;
    for (int tries = 0; tries < 2 && !ok; tries++) {
        for (uint32_t i = 0; i < kMbarMaxTries && !ok; i++) ok = mbar_try_wait(&sh.bar, 0);
        if (!ok) set_op_error(kErrMbarTimeout);
    }

    // ---- the largest values, by groups of eight threads, to every CTA
    float most = -INFINITY;
    s.each([&](float x, int) { most = fmaxf(most, x); });
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    s.cluster.barrier_wait();
    if ((tid & 7) < ctas) *s.cluster.map_shared_rank(&sh.gmax[s.rank * kGroups + tid / 8], tid & 7) = most;
    s.cluster.sync();
    const int groups = ctas * kGroups;
    const float g = tid < groups ? sh.gmax[tid] : -INFINITY;
    float m = warp_max(g);
    if (lane == 0) reinterpret_cast<float*>(sh.warp_sum)[tid >> 5] = m;
    __syncthreads();
    for (int w = 0; w < kWarps; w++) m = fmaxf(m, reinterpret_cast<float*>(sh.warp_sum)[w]);
    s.row.m = m;
    if (!(m > -INFINITY)) {  // nothing to take
        if (s.rank == 0 && tid == 0) s.answer(r, -1, 0.0f, 1);
        return;
    }

    // ---- greedy: the first maximum
    const float temperature = !a.u ? 0.0f : a.temperatures ? a.temperatures[r] : a.temperature;
    if (!(temperature > 0.0f)) {
        unsigned best = 0xFFFFFFFFu;
        s.each([&](float x, int i) { if (x == m) best = min(best, unsigned(i)); });
        best = __reduce_min_sync(0xffffffffu, best);
        if (lane == 0 && best != 0xFFFFFFFFu) atomicMin(s.cluster.map_shared_rank(&sh.best, 0), best);
        s.cluster.sync();
        if (s.rank == 0 && tid == 0) {
            a.token[r] = int(sh.best);
            if (a.prob) a.prob[r] = 1.0f;
        }
        return;
    }

    const float min_p = a.min_ps ? a.min_ps[r] : a.min_p, top_p = a.top_ps ? a.top_ps[r] : a.top_p;
    int top_k = a.top_ks ? a.top_ks[r] : a.top_k;
    if (top_k < 0 || top_k >= a.vocab) top_k = 0;
    const bool use_p = top_p < 1.0f;
    s.row.c = 1.4426950408889634 / double(temperature);
    s.row.lim = min_p > 0.0f ? fmax(-log2(double(min_p)), 0.0) : INFINITY;
    if (top_k || use_p) {
        const int want = top_k ? top_k : groups / 2;
        if (4 * want <= 3 * groups) {
            if (tid < groups) {
                int above = 0;
                for (int j = 0; j < groups; j++) above += sh.gmax[j] > g || (sh.gmax[j] == g && j < tid);
                if (above == want - 1) sh.pick = g;
            }
            __syncthreads();
            if (s.few(r, sh.pick, top_k, use_p, top_p)) return;
        }
        if (top_k) s.template select<false>([&](unsigned long long) { return double(top_k); });
        if (use_p) s.template select<true>([&](unsigned long long total) { return fmax(double(top_p) * double(total), 0.5); });
    }
    const unsigned long long cut = sh.cut;
    const unsigned long long total = s.find([&](float x, int i) { return S::real(x) && S::entry(x, i) >= cut && within(s.row, x) ? weight(s.row, sh.table, x) : 0.0; },
                                            [&](unsigned long long all) { return s.place(r, all); });
    if (tid == 0 && sh.found != 0xFFFFFFFFu) s.answer(r, int(sh.found), sh.pick, total);
}

template <typename T>
cudaError_t go(const neko_sample_rows_args& a, cudaStream_t st) {
    constexpr int kPer = 16 / sizeof(T);
    int ctas = 1;
    while (ctas < kMaxCluster && a.vocab > 4096 * ctas) ctas *= 2;
    const int slice = ((a.vocab + ctas - 1) / ctas + kPer - 1) / kPer * kPer;
    const size_t smem = (sizeof(Shared) + 127) / 128 * 128 + kSmemAux + size_t(slice + kPer) * sizeof(T);
    auto* fn = sample_rows_kernel<T>;
    if (cudaError_t e = ensure_dyn_smem(fn, smem); e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(a.rows) * unsigned(ctas));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = unsigned(ctas);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ctas > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, fn, a, slice);
}

}  // namespace

cudaError_t launch_sample_rows(const neko_sample_rows_args& a, cudaStream_t st) {
    return a.type == NEKO_T_F32 ? go<float>(a, st) : a.type == NEKO_T_F16 ? go<__half>(a, st) : go<__nv_bfloat16>(a, st);
}

}  // namespace neko
