// Tokens from rows of logits with temperature, top-k, top-p and min-p (neko_op_sample_rows).
//
// A cluster of one to eight CTAs takes a row, each a slice, which it reads again for each pass (two to four; all but the first from
// L2 unless the logits are far larger). Slices kept in shared memory would leave room for 33 rows of 151,936 at a time, and a row
// waits for its cluster's meetings as long as it computes (320 nuclei: 411 us that way).
// Weights 2^(44 - y), y = (max - x) log2(e) / temperature, are rounded to integers and added as integers: sums do not depend on an
// order, and any split of a row gives the same token. They are computed in 64 bits (a table of 32 powers, 16 copies of it so that no
// two lanes of a half warp meet in a bank, and a polynomial of degree 5): with V tokens of about equal weight a row's number falls
// within 2^-24 of a border once in 2^24 / V rows, so f32 sums would choose otherwise than the definition now and then.
//
// What is kept is a beginning of the row in descending order, found without sorting the row:
//  * top-k: the largest values of 64 groups of threads a CTA bound the k-th largest of the row from below (the k-th largest of them),
//    and few more than k tokens reach that bound: they are collected in one CTA, ranked by counting and cut there. Enough for k
//    up to three quarters of the groups.
//  * top-p alone: an eighth of the tokens is counted in 4,096 equal steps of max - x, which gives the step of the cut but for the
//    sample's error (the largest tokens, which would make it large, are summed as they are). One pass over the weights adds up
//    the row, what lies before that window, and puts the window's tokens aside; among those the cut is found by the exact sums,
//    which also tell a window that has missed it (then the next way is taken).
//  * else a histogram over equal steps, of counts or of weights in four pieces of 14 bits (32-bit additions in shared memory),
//    added up over the cluster, gives the step that the cut falls into; its tokens are collected and ranked, or where they are
//    too many the key's digits (11, 11 and 10 bits) lead to the cut's value, whose equals are cut by index.
// The draw goes through the slices in the order of the vocabulary: sums of CTAs, of warps' segments, of lanes.
//
// From a graph: 1 x 151,936 f32, k = 40, p = 0.95: 11.2 us (launch, two passes, the cluster's meetings); 64 x 50,257 bf16 with mixed
// parameters 59 us, the time of the slowest rows (k = 1000, some 40 us alone; nuclei 35; k = 40 10); 320 x 151,936 nuclei 261 us
// beside 30 for reading them once: 49 M weights in 64 bits, about 35 cycles a warp's 32, and the meetings. Rows whose tokens are all
// in one bin of a histogram wait for its additions, one after the other (200 flat rows of 262,144, a nucleus: 2.6 ms).
#include <cooperative_groups.h>

#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "paged.cuh"

namespace cg = cooperative_groups;

namespace neko {

namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kGroups = kThreads / 8;  // groups of threads whose largest values are known
constexpr int kCand = 1024;            // tokens that are ranked by counting
constexpr int kMine = 512;             // of them those of one CTA of several
constexpr int kBins = 2048;
constexpr int kPiece = 14, kPieces = 4;  // bits of a weight's pieces in the histograms, and how many: 2^44 takes 45
constexpr int kSteps = 4096;           // steps of max - x that a sample of the tokens is counted in
constexpr int kFine = 1024;            // steps of the window
constexpr int kRing = 4;
constexpr int kPowers = 32, kCopies = 16;
constexpr int kMaxCluster = 8;
constexpr double kOne = 17592186044416.0;  // 2^44: the weight of the largest
constexpr double kSquare = 4503599627370496.0;  // 2^52: a sample's squares are added up in units of it
static_assert(NEKO_MAX_VOCAB / 8 * (8 * kOne) * (8 * kOne) / kSquare < 0x1p63, "one token in 8, each for 8 of the largest weight");
// lists of CTA 0 (as collected, then the sums; in order), the CTA's own list, the counts; histograms take all of it
constexpr int kSortedOff = kCand * 8, kMineOff = 2 * kCand * 8;
__host__ __device__ constexpr int counts_off(int ctas) { return kMineOff + (ctas > 1 ? kMine : kCand) * 8; }
__host__ __device__ constexpr int window_off(int ctas) { return counts_off(ctas) + kSteps * 4; }
// tokens of the window in one CTA: with one CTA two of them fill an SM's shared memory
__host__ __device__ constexpr int window_room(int ctas) { return ctas == 1 ? 8192 : ctas == 2 ? 5120 : ctas == 4 ? 3584 : 2048; }
__host__ __device__ constexpr int aux_bytes(int ctas) { return window_off(ctas) + window_room(ctas) * 8; }
static_assert(window_off(kMaxCluster) >= kRing * kThreads * 16, "the ring");
static_assert(window_off(kMaxCluster) >= kPieces * kBins * 4, "the histograms");
// a CTA may hold a whole row, and all its tokens may be in one bin
static_assert((1ull << kPiece) * NEKO_MAX_VOCAB <= 1ull << 32 && kPiece * kPieces > 44, "a bin holds a row's pieces in 32 bits");

// The order of values as unsigned numbers; zeros are alike.
__device__ __forceinline__ uint32_t order_key(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k); }

// What the threads of a row share. Lists are ordered by key (value, then lower index): (order_key << 32) | ~index.
struct Shared {
    double table[kPowers * kCopies];      // 2^(i / 32) at [i][copy]
    float gmax[kMaxCluster * kGroups];
    unsigned long long sum[kMaxCluster];  // by CTA: of weights or counts
    unsigned long long warp_sum[kWarps];
    unsigned long long seg[kWarps];       // what is kept in each warp's segment
    unsigned long long cut;               // tokens from here up (in the lists' order) are kept
    unsigned long long before, total;
    unsigned long long others[kMaxCluster][2];  // by CTA: two more sums
    unsigned best, found;                 // lowest index
    unsigned n_list, n_all, at_list;      // tokens in this CTA's list, in CTA 0's, and where this CTA's begin there
    unsigned n_window;
    int bin, bin_end, done;
    float pick;
    uint4 ends[2];                        // the slice's first and last vector, -infinity in places outside it
};

// y = (m - x) c.
struct Row {
    float m;        // largest value
    float from;     // NaN, or: values are read as their differences from it, the largest one
    bool alone;     // the others then as -infinity: it is infinite, or the next value below weighs nothing
    float low;      // values count as no less than this, 46.5 to 303 powers of two below: they weigh nothing there
    float c32;
    double m64, c, c_powers;  // c = log2(e) / temperature, times the table's powers
    float least;    // of the values that min-p leaves in
    float cut;      // kept: larger values, and this one up to an index
    unsigned cut_at;
};

// 2^(44 - y) to the nearest integer, as the bits of 2^52 plus it. No branch, so that several values' chains run side by side.
constexpr unsigned long long kBits = 0x4330000000000000ull;  // of 2^52
__device__ __forceinline__ unsigned long long weight_bits(const Row& r, const double* table, float x) {
    const double d = double(fmaxf(x, r.low)) - r.m64;  // NaN: low
    constexpr double kMagic = 6755399441055744.0 + 44 * kPowers;  // 1.5 * 2^52: the integer in the low word
    const double t = fma(d, r.c_powers, kMagic);
    const int n = __double2loint(t);
    const double f = fma(d, r.c_powers, kMagic - t);
    // 2^(f / 32), |f| <= 1/2: (ln2 / 32)^k / k!
    double p = fma(f, 3.9737099845494154e-11, 9.172562701824643e-09);
    p = fma(p, f, 1.6938509724371819e-06);
    p = fma(p, f, 0.00023459619820224677);
    p = fma(p, f, 0.02166084939249829);
    const double w = table[(n & (kPowers - 1)) * kCopies + (threadIdx.x & (kCopies - 1))];
    const double s = __hiloint2double(__double2hiint(w) + ((n >> 5) << 20), __double2loint(w));
    return __double_as_longlong(fma(p * f, s, s) + 4503599627370496.0);
}
__device__ __forceinline__ unsigned long long weight(const Row& r, const double* table, float x) { return weight_bits(r, table, x) - kBits; }
// Four weights, all of them before any is asked for: moved under the conditions that they are used on, the chains run one after
// the other (a warp's 128 values 1,500 cycles instead of 230).
__device__ __forceinline__ void four_weights(const Row& r, const double* table, const float (&x)[4], unsigned long long (&y)[4]) {
#pragma unroll
    for (int j = 0; j < 4; j++) y[j] = weight(r, table, x[j]);
#pragma unroll
    for (int j = 0; j < 4; j++) asm volatile("" : "+l"(y[j]));
}
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
// Sums up to and with each of `per` consecutive values a thread, in place; the sum of all is returned.
template <int kPer>
__device__ __forceinline__ unsigned long long cta_upto(Shared& sh, unsigned long long (&v)[kPer]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int i = 1; i < kPer; i++) v[i] += v[i - 1];
    const unsigned long long upto = warp_upto(v[kPer - 1], lane);
    __syncthreads();
    if (lane == 31) sh.warp_sum[warp] = upto;
    __syncthreads();
    const unsigned long long x = lane < kWarps ? sh.warp_sum[lane] : 0ull, all = warp_total(x);
    const unsigned long long before = upto - v[kPer - 1] + warp_total(lane < warp ? x : 0ull);
#pragma unroll
    for (int i = 0; i < kPer; i++) v[i] += before;
    return all;
}

template <typename T>
struct Sampler {
    static constexpr int kPer = 16 / sizeof(T);  // values of a 16-byte vector
    using u64 = unsigned long long;
    const neko_sample_rows_args& a;
    cg::cluster_group cluster;
    Shared& sh;
    uint8_t* aux;
    const uint4* data;          // the slice's vectors; the first and the last are read from sh.ends
    int ctas, rank, nv, first;  // how many; vocabulary index of the first one's first place
    Row row;

    __device__ Sampler(const neko_sample_rows_args& a_, Shared& s, uint8_t* x) : a(a_), cluster(cg::this_cluster()), sh(s), aux(x) {}

    __device__ u64* list() const { return reinterpret_cast<u64*>(aux); }
    __device__ u64* sorted() const { return reinterpret_cast<u64*>(aux + kSortedOff); }
    __device__ u64* mine() const { return reinterpret_cast<u64*>(aux + kMineOff); }
    __device__ u64* window() const { return reinterpret_cast<u64*>(aux + window_off(ctas)); }
    __device__ uint32_t* counts() const { return reinterpret_cast<uint32_t*>(aux + counts_off(ctas)); }
    __device__ unsigned mine_room() const { return ctas > 1 ? kMine : kCand; }
    __device__ int segment() const { return (nv + kWarps - 1) / kWarps; }  // vectors of a warp's segment

    // A vector; past the end -infinities.
    __device__ __forceinline__ uint4 load(int v, int end) const {
        constexpr uint32_t none = std::is_same<T, float>::value ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
        if (v >= end) return make_uint4(none, none, none, none);
        return v == 0 || v == nv - 1 ? sh.ends[v != 0] : __ldg(data + v);
    }
    // What a value is read as: see Row::from.
    __device__ __forceinline__ float read(float x) const { return x == row.from ? 0.0f : row.alone ? -INFINITY : x - row.from; }
    // Values j0 .. j0 + 3 of a vector. Places outside the row hold -infinity.
    __device__ __forceinline__ void four(const uint4& w, int j0, float (&x)[4]) const {
        if constexpr (kPer == 4) {
            x[0] = __uint_as_float(w.x), x[1] = __uint_as_float(w.y), x[2] = __uint_as_float(w.z), x[3] = __uint_as_float(w.w);
        } else {
            const uint2 h = j0 ? make_uint2(w.z, w.w) : make_uint2(w.x, w.y);
            const T* y = reinterpret_cast<const T*>(&h);
#pragma unroll
            for (int j = 0; j < 4; j++) x[j] = float(y[j]);
        }
        if (row.from == row.from)
#pragma unroll
            for (int j = 0; j < 4; j++) x[j] = read(x[j]);
    }
    // f(four values, index of the first) of the vectors v0, v0 + step, .. before v1, kAhead of them on their way at a time.
    template <int kAhead, typename F>
    __device__ __forceinline__ void sweep(int v0, int step, int v1, F f) const {
        uint4 w[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; k++) w[k] = load(v0 + k * step, v1);
#pragma unroll 1
        for (int v = v0; v < v1; v += kAhead * step) {
            uint4 now[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; k++) now[k] = w[k], w[k] = load(v + (kAhead + k) * step, v1);
#pragma unroll
            for (int k = 0; k < kAhead; k++)
#pragma unroll
                for (int j0 = 0; j0 < kPer; j0 += 4) {
                    float x[4];
                    four(now[k], j0, x);
                    f(x, first + (v + k * step) * kPer + j0);
                }
        }
    }
    // The same, kRing vectors on their way to shared memory (aux, which holds nothing else then): the passes over the weights have no
    // registers for them (320 nuclei: 288 us with one ahead in registers).
    template <typename F>
    __device__ __forceinline__ void sweep_ring(int v0, int step, int v1, F f) const {
        uint4* ring = reinterpret_cast<uint4*>(aux) + threadIdx.x;
        auto fetch = [&](int v, int slot) {
            if (v < v1) {
                if (v == 0 || v == nv - 1) ring[slot * kThreads] = sh.ends[v != 0];
                else asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(ring + slot * kThreads)), "l"(data + v) : "memory");
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int k = 0; k < kRing; k++) fetch(v0 + k * step, k);
        int slot = 0;
#pragma unroll 1
        for (int v = v0; v < v1; v += step) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 1) : "memory");
            const uint4 now = ring[slot * kThreads];
            fetch(v + kRing * step, slot);
            slot = (slot + 1) & (kRing - 1);
#pragma unroll
            for (int j0 = 0; j0 < kPer; j0 += 4) {
                float x[4];
                four(now, j0, x);
                f(x, first + v * kPer + j0);
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    // Of all vectors, spread over the threads; of the warp's segment.
    template <int kAhead, typename F>
    __device__ __forceinline__ void each(F f) const {
        sweep<kAhead>(threadIdx.x, kThreads, nv, f);
    }
    template <typename F>
    __device__ __forceinline__ void each_of_segment(F f) const {
        const int v0 = int(threadIdx.x >> 5) * segment();
        sweep_ring(v0 + int(threadIdx.x & 31), 32, min(v0 + segment(), nv), f);
    }
    // What four tokens count of which take(value, index) holds: their weights, or 1 each.
    template <bool MASS, typename F>
    __device__ __forceinline__ u64 measured(const float (&x)[4], int i, F take) const {
        bool in[4];
#pragma unroll
        for (int j = 0; j < 4; j++) in[j] = take(x[j], i + j);
        if (!(in[0] || in[1] || in[2] || in[3])) return 0;
        u64 sum = 0, y[4] = {1, 1, 1, 1};
        if constexpr (MASS) four_weights(row, sh.table, x, y);
#pragma unroll
        for (int j = 0; j < 4; j++) sum += in[j] ? y[j] : 0ull;
        return sum;
    }
    __device__ __forceinline__ static u64 entry(float x, int i) { return (static_cast<u64>(order_key(x)) << 32) | (0xFFFFFFFFu - unsigned(i)); }
    __device__ __forceinline__ static float value(u64 e) { return key_value(uint32_t(e >> 32)); }
    // Values that can be taken at all: not NaN, not -infinity.
    __device__ __forceinline__ static bool real(float x) { return x > -INFINITY; }
    // Whether the cut leaves a token in.
    __device__ __forceinline__ bool kept(float x, int i) const { return x > row.cut || (x == row.cut && unsigned(i) <= row.cut_at); }
    __device__ void take_cut() {  // as sh.cut says it; 0: nothing is cut
        row.cut = sh.cut ? value(sh.cut) : -INFINITY;
        row.cut_at = sh.cut ? 0xFFFFFFFFu - uint32_t(sh.cut) : 0u;
    }
    __device__ void cut_least() {  // min-p's too
        if (row.least > row.cut) row.cut = row.least, row.cut_at = 0xFFFFFFFFu;
    }
    __device__ __forceinline__ u64 weight_of(float x) const { return weight(row, sh.table, x); }

    // The CTAs' sums meet: sum[i] of every CTA.
    __device__ void share_sum(u64 v) {
        if (threadIdx.x < ctas) *cluster.map_shared_rank(&sh.sum[rank], threadIdx.x) = v;
        cluster.sync();
    }

    // A token that take() has chosen goes to this CTA's list.
    __device__ __forceinline__ void put(float x, int i) {
        const unsigned at = atomicAdd(&sh.n_list, 1u);
        if (at < mine_room()) mine()[at] = entry(x, i);
    }
    // The CTAs' lists come together in CTA 0's: n_all says how many tokens there are, if more than kCand they are not all there.
    // then() before the CTAs meet.
    template <typename G>
    __device__ void gather(G then) {
        __syncthreads();
        const unsigned n = sh.n_list;
        u64* to = cluster.map_shared_rank(list(), 0);
        if (threadIdx.x == 0) sh.at_list = atomicAdd(cluster.map_shared_rank(&sh.n_all, 0), n > mine_room() ? kCand + 1 : n);
        __syncthreads();
        for (unsigned i = threadIdx.x; i < min(n, mine_room()); i += kThreads)
            if (sh.at_list + i < kCand) to[sh.at_list + i] = mine()[i];
        then();
        cluster.sync();
    }

    // CTA 0's list in descending order (sorted()), and in its place the sums of measure(entry) up to and with each.
    template <typename F>
    __device__ void rank_list(int n, F measure) {
        for (int i = threadIdx.x; i < n; i += kThreads) {
            const u64 e = list()[i];
            int r = 0, j = 0;
            for (; j + 4 <= n; j += 4) {
                const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(list() + j), y = *reinterpret_cast<const ulonglong2*>(list() + j + 2);
                r += (x.x > e) + (x.y > e) + (y.x > e) + (y.y > e);
            }
            for (; j < n; j++) r += list()[j] > e;
            sorted()[r] = e;
        }
        __syncthreads();
        u64 v[kCand / kThreads];
#pragma unroll
        for (int k = 0; k < kCand / kThreads; k++) {
            const int i = kCand / kThreads * threadIdx.x + k;
            v[k] = i < n ? measure(sorted()[i]) : 0ull;
        }
        cta_upto(sh, v);
#pragma unroll
        for (int k = 0; k < kCand / kThreads; k++)
            if (int(kCand / kThreads * threadIdx.x) + k < n) list()[kCand / kThreads * threadIdx.x + k] = v[k];
        __syncthreads();
    }
    // How many of CTA 0's n sums, each with what lies ahead, are below target.
    __device__ int below(int n, double target, u64 ahead) {
        int c = 0;
        for (int base = 0; base < n; base += kThreads)
            c += __syncthreads_count(base + threadIdx.x < n && double(ahead + list()[base + threadIdx.x]) < target);
        return c;
    }

    // The entry of CTA 0's n at which, in descending order, the sum of the weights (mass) or counts with what lies ahead reaches want:
    // by 512 bins of their keys, and the entries of one bin against each other. 0: none.
    __device__ u64 cut_in_list(int n, double want, u64 ahead, bool mass) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        if (n <= 32) {  // one warp's
            if (threadIdx.x == 0) sh.cut = 0;
            __syncthreads();
            if (warp == 0) {
                const u64 x = lane < n ? list()[lane] : 0ull, w = lane >= n ? 0ull : mass ? weight_of(value(x)) : 1ull;
                u64 sum = ahead;
                for (int j = 0; j < n; j++) {
                    const u64 y = __shfl_sync(0xffffffffu, x, j), v = __shfl_sync(0xffffffffu, w, j);
                    sum += y > x ? v : 0ull;
                }
                if (lane < n && double(sum) < want && double(sum + w) >= want) sh.cut = x;
            }
            __syncthreads();
            return sh.cut;
        }
        uint32_t* red = reinterpret_cast<uint32_t*>(sh.warp_sum);
        uint32_t most = 0, least = 0xFFFFFFFFu;
        for (int i = threadIdx.x; i < n; i += kThreads) {
            const uint32_t k = uint32_t(list()[i] >> 32);
            most = max(most, k), least = min(least, k);
        }
        most = __reduce_max_sync(0xffffffffu, most), least = __reduce_min_sync(0xffffffffu, least);
        if (lane == 0) red[warp] = most, red[kWarps + warp] = least;
        u64* bins = sorted();
        bins[threadIdx.x] = 0;
        if (threadIdx.x == 0) sh.n_list = 0, sh.cut = 0, sh.bin = -1;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWarps; w++) most = max(most, red[w]), least = min(least, red[kWarps + w]);
        const int shift = max(23 - __clz(most - least), 0);
        auto bin_of = [&](u64 e) { return int((most - uint32_t(e >> 32)) >> shift); };  // below 512
        for (int i = threadIdx.x; i < n; i += kThreads) {
            const u64 e = list()[i];
            atomicAdd(&bins[bin_of(e)], mass ? weight_of(value(e)) : 1ull);
        }
        __syncthreads();
        u64 v[1] = {bins[threadIdx.x]};
        const u64 own = v[0];
        cta_upto(sh, v);
        const u64 upto = ahead + v[0], less = upto - own;
        if (own && double(upto) >= want && double(less) < want) sh.bin = threadIdx.x, sh.before = less;
        __syncthreads();
        const int bin = sh.bin;
        ahead = sh.before;
        u64 e[kCand / kThreads];
#pragma unroll
        for (int k = 0; k < kCand / kThreads; k++) {
            const int i = threadIdx.x + k * kThreads;
            e[k] = i < n ? list()[i] : 0ull;
            if (i >= n || bin_of(e[k]) != bin) e[k] = 0;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kCand / kThreads; k++)
            if (e[k]) {
                const unsigned at = atomicAdd(&sh.n_list, 1u);
                sorted()[at] = e[k], list()[at] = mass ? weight_of(value(e[k])) : 1ull;
            }
        __syncthreads();
        const int few = int(sh.n_list);
        for (int i = threadIdx.x; i < few; i += kThreads) {
            const u64 x = sorted()[i];
            u64 sum = ahead;
            for (int j = 0; j < few; j++) sum += sorted()[j] > x ? list()[j] : 0ull;
            if (double(sum) < want && double(sum + list()[i]) >= want) sh.cut = x;
        }
        __syncthreads();
        return sh.cut;
    }

    __device__ void answer(int r, int token, float x, u64 total) {
        a.token[r] = token;
        if (a.prob) a.prob[r] = token < 0 ? 0.0f : float(exp2((double(x) - row.m64) * row.c) * (kOne / double(total)));
    }
    // floor(u * total), below total.
    __device__ u64 place(int r, u64 total) {
        const double x = a.u[r] * double(total);
        return min(x > 0.0 ? static_cast<u64>(x) : 0ull, total - 1);
    }

    // The first index, in the order of the vocabulary, at which the sum over the tokens taken exceeds where(sum of all): its CTA
    // gets found = index, pick = value. seg[] holds the segments' sums. The sum of all is returned.
    template <bool MASS, typename M, typename P>
    __device__ u64 locate(M take, P where) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        if (threadIdx.x == 0) sh.found = 0xFFFFFFFFu;
        __syncthreads();
        u64 of_cta = 0, before = 0, total = 0;
#pragma unroll
        for (int w = 0; w < kWarps; w++) of_cta += sh.seg[w];
        share_sum(of_cta);
        for (int i = 0; i < ctas; i++) {
            const u64 x = sh.sum[i];
            before += i < rank ? x : 0ull, total += x;
        }
        const u64 at = where(total);
        if (total && at >= before && at - before < of_cta) {  // one CTA of the cluster
            // its segment that has it, in as many parts as warps
            int w = 0;
            while (at - before >= sh.seg[w]) before += sh.seg[w++];
            const int s0 = w * segment(), s1 = min(s0 + segment(), nv), size = (s1 - s0 + kWarps - 1) / kWarps;
            const int v0 = min(s0 + warp * size, s1), v1 = min(v0 + size, s1);
            u64 part = 0;
            sweep<1>(v0 + lane, 32, v1, [&](const float (&x)[4], int i) { part += measured<MASS>(x, i, take); });
            part = warp_total(part);
            if (lane == 0) sh.warp_sum[warp] = part;
            __syncthreads();
            for (int i = 0; i < warp; i++) before += sh.warp_sum[i];
            if (at >= before && at - before < part)  // one warp
                for (int base = v0; base < v1; base += 32) {
                    const int v = base + lane;
                    u64 s = 0;
                    const uint4 w = load(v, v1);
                    float x[4];
#pragma unroll
                    for (int j0 = 0; j0 < kPer; j0 += 4) four(w, j0, x), s += measured<MASS>(x, first + v * kPer + j0, take);
                    const u64 upto = before + warp_upto(s, lane);
                    if (upto > at && upto - s <= at) {  // one lane
                        u64 sum = upto - s;
                        bool there = false;
#pragma unroll 1
                        for (int j = 0; j < kPer; j++) {
                            const int i = first + v * kPer + j;
                            four(w, j & ~3, x);
                            const float y = (j & 3) == 0 ? x[0] : (j & 3) == 1 ? x[1] : (j & 3) == 2 ? x[2] : x[3];
                            sum += !take(y, i) ? 0ull : MASS ? weight_of(y) : 1ull;
                            if (sum > at && !there) sh.found = unsigned(i), sh.pick = y, there = true;
                        }
                    }
                    before = __shfl_sync(0xffffffffu, upto, 31);
                    if (before > at) break;
                }
        }
        __syncthreads();
        return total;
    }
    template <bool MASS, typename M>
    __device__ void fill(M take) {
        u64 part = 0;
        __syncthreads();
        each_of_segment([&](const float (&x)[4], int i) { part += measured<MASS>(x, i, take); });
        part = warp_total(part);
        if ((threadIdx.x & 31) == 0) sh.seg[threadIdx.x >> 5] = part;
    }

    // Adds up a histogram of counts, or of weights (mass), over the cluster and finds the bin at which the sum, with what lies ahead
    // of it, reaches `part` of the sum of all (0: `want`): bin (-1: none does), before (the sum without the bin), total to every CTA.
    template <typename F>
    __device__ void histogram(bool mass, F bin_of, u64 ahead, double part, double want) {
        uint32_t* h = reinterpret_cast<uint32_t*>(aux);
        for (int i = threadIdx.x; i < (mass ? kPieces : 1) * kBins; i += kThreads) h[i] = 0;
        __syncthreads();
        each<1>([&](const float (&x)[4], int i) {
#pragma unroll 1
            for (int j = 0; j < 4; j++) {
                const float y = j == 0 ? x[0] : j == 1 ? x[1] : j == 2 ? x[2] : x[3];
                const int b = bin_of(y, i + j);
                if (b < 0) continue;
                if (!mass) {
                    atomicAdd(&h[b], 1u);
                    continue;
                }
                const u64 w = weight_of(y);
#pragma unroll
                for (int p = 0; p < kPieces; p++) {
                    const uint32_t piece = uint32_t(w >> kPiece * p) & ((1u << kPiece) - 1);
                    if (piece) atomicAdd(&h[p * kBins + b], piece);
                }
            }
        });
        cluster.sync();
        // this CTA's share of the bins, kBins / ctas of them: four at most a thread
        constexpr int kMost = kBins / kThreads;
        const int share = kBins / ctas, per = (share + kThreads - 1) / kThreads;
        u64 v[kMost] = {}, own[kMost];
#pragma unroll 1
        for (int c = 0; c < ctas; c++) {
            const uint32_t* o = cluster.map_shared_rank(h, c) + rank * share;
#pragma unroll
            for (int k = 0; k < kMost; k++) {
                const int b = threadIdx.x * per + k;
                if (k >= per || b >= share) continue;
                v[k] += o[b];
                if (mass)
#pragma unroll
                    for (int p = 1; p < kPieces; p++) v[k] += static_cast<u64>(o[p * kBins + b]) << kPiece * p;
            }
        }
#pragma unroll
        for (int k = 0; k < kMost; k++) own[k] = v[k];
        const u64 all = cta_upto(sh, v);
        if (threadIdx.x == 0) sh.bin = -1;
        share_sum(all);
        u64 before = ahead, total = ahead;
        for (int i = 0; i < ctas; i++) {
            if (i < rank) before += sh.sum[i];
            total += sh.sum[i];
        }
        if (part > 0.0) want = fmax(part * double(total), 0.5);
        // one thread of the cluster has the bin that reaches it
#pragma unroll
        for (int k = 0; k < kMost; k++) {
            const u64 upto = before + v[k], less = upto - own[k];
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

    // Moves the cut (among what the present one keeps) to the first token, in descending order, at which the count reaches top_k, or
    // (mass) the sum of the weights top_p times theirs. Equal steps of max - x first; where more tokens than can be ranked are in
    // the step of the cut, the three digits of their keys.
    __device__ void select(bool mass, int top_k, float top_p) {
        const float scale = fminf(64.0f * fmaxf(row.c32, 1.0f), 1e30f);
        auto step_of = [&](float x, int i) { return real(x) && kept(x, i) ? int(fminf((row.m - x) * scale, float(kBins - 1))) : -1; };
        if (threadIdx.x == 0) sh.n_all = sh.n_list = 0;
        uint32_t key = 0, known = 0;
        u64 before = 0;
        double want = mass ? 0.5 : double(top_k);
        int step = 0;
#pragma unroll 1
        for (int level = 0; level < 4; level++) {
            const int shift = level == 1 ? 21 : level == 2 ? 10 : 0;
            const uint32_t most = level == 3 ? 1023u : 2047u;
            histogram(mass, [&](float x, int i) {
                const int b = step_of(x, i);
                if (!level) return b;
                const uint32_t k = order_key(x);
                return b == step && (k & known) == key ? int(most - (k >> shift & most)) : -1;
            }, before, mass && !level ? fmax(double(top_p), 0x1p-80) : 0.0, want);
            if (sh.bin < 0) return;  // fewer than that many
            before = sh.before;
            if (level) {
                key |= (most - uint32_t(sh.bin)) << shift;
                known |= most << shift;
                continue;
            }
            step = sh.bin;
            if (mass) want = fmax(double(top_p) * double(sh.total), 0.5);
            each<1>([&](const float (&x)[4], int i) {
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (step_of(x[j], i + j) == step) put(x[j], i + j);
            });
            gather([]() {});
            if (rank == 0) {
                u64 next = 0;
                if (sh.n_all <= kCand) next = cut_in_list(int(sh.n_all), want, before, mass);
                if (threadIdx.x < ctas) {
                    Shared* o = cluster.map_shared_rank(&sh, threadIdx.x);
                    o->done = next != 0;
                    if (next) o->cut = next;
                }
            }
            cluster.sync();
            if (sh.done) return take_cut();
        }
        const double each_one = mass ? double(weight_of(key_value(key))) : 1.0;
        const double more = ceil((want - double(before)) / each_one);
        auto equal = [&](float x, int i) { return step_of(x, i) == step && order_key(x) == key; };
        fill<false>(equal);
        locate<false>(equal, [&](u64 total) { return more > 1.0 ? min(static_cast<u64>(more) - 1, total - 1) : 0ull; });
        if (threadIdx.x == 0 && sh.found != 0xFFFFFFFFu) {
            const u64 next = (static_cast<u64>(key) << 32) | (0xFFFFFFFFu - sh.found);
            for (int c = 0; c < ctas; c++) cluster.map_shared_rank(&sh, c)->cut = next;
        }
        cluster.sync();
        take_cut();
    }

    // Top-k by the largest values alone; true: the row is answered.
    __device__ bool few(int r, float t, int top_k, bool use_p, float top_p) {
        if (threadIdx.x == 0) sh.done = 0, sh.n_list = 0;
        __syncthreads();
        each<4>([&](const float (&x)[4], int i) {
            if (fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) >= t)
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (x[j] >= t && real(x[j])) put(x[j], i + j);
        });
        gather([]() {});
        if (rank == 0) {
            const unsigned n_all = sh.n_all;
            __syncthreads();  // read by all before it is set again below
            if (n_all <= kCand) {
                const int n = int(n_all), n_k = min(top_k, n);
                rank_list(n, [&](u64 e) { return weight_of(value(e)); });
                const u64* upto = list();
                int left = n_k;
                if (use_p) left = min(below(n_k, fmax(double(top_p) * double(upto[n_k - 1]), 0.5), 0) + 1, n_k);
                if (row.least > -INFINITY) {
                    int n_m = 0;
                    for (int base = 0; base < left; base += kThreads) {
                        const int i = base + threadIdx.x;
                        n_m += __syncthreads_count(i < left && value(sorted()[i < left ? i : 0]) >= row.least);
                    }
                    left = n_m;
                }
                const u64 total = upto[left - 1], at = place(r, total);
                for (int i = threadIdx.x; i < left; i += kThreads) {
                    const uint32_t low = uint32_t(sorted()[i]);  // ~index
                    u64 before = 0, last = 0;
                    for (int j = 0; j < left; j++) {
                        const u64 u = upto[j];
                        before += uint32_t(sorted()[j]) > low ? u - last : 0ull;
                        last = u;
                    }
                    if (at >= before && at - before < upto[i] - (i ? upto[i - 1] : 0ull))
                        answer(r, int(0xFFFFFFFFu - low), value(sorted()[i]), total);
                }
            }
            if (threadIdx.x < ctas) cluster.map_shared_rank(&sh, threadIdx.x)->done = n_all <= kCand;
            if (threadIdx.x == 0) sh.n_all = 0;
        }
        cluster.sync();
        return sh.done != 0;
    }

    // Steps of max - x: to nearest, NaN and what is far: the last; and what a step's tokens weigh by its middle.
    __device__ __forceinline__ int count_step(float x, float scale) const {
        return __float_as_int(fminf((row.m - x) * scale, float(kSteps - 1)) + 8388608.0f) & (kSteps - 1);
    }
    __device__ __forceinline__ float middle(int step, float scale) const {
        return step == kSteps - 1 ? 0.0f : exp2f(44.0f - (step ? float(step) : 0.25f) / scale * row.c32);
    }

    // Top-p alone; t: a value that some dozens of tokens reach. True: the cut is set, and seg[] holds what is kept.
    __device__ bool nucleus(float t, float top_p) {
        const float scale = fminf(128.0f * fmaxf(row.c32, 1.0f), 1e30f);
        // ---- a sample by steps: one in `rate` of each warp's turns, not the same ones for neighbours
        int rate = 1;
        while (rate < 8 && a.vocab > 16384 * rate) rate *= 2;
        for (int i = threadIdx.x; i < kSteps; i += kThreads) counts()[i] = 0;
        if (threadIdx.x == 0) sh.n_list = sh.n_window = 0;
        __syncthreads();
        u64 top = 0;
        int turn = threadIdx.x >> 5;
        each<4>([&](const float (&x)[4], int) {
            if (fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) >= t)
#pragma unroll 1
                for (int j = 0; j < 4; j++) {
                    const float y = j == 0 ? x[0] : j == 1 ? x[1] : j == 2 ? x[2] : x[3];
                    if (y >= t) top += weight_of(y);
                }
            if ((turn++ & (rate - 1)) == 0)
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (!(x[j] >= t)) {
                        const int step = count_step(x[j], scale);
                        if (step < kSteps - 1) atomicAdd(&counts()[step], 1u);
                    }
        });
        top = warp_total(top);
        __syncthreads();
        if ((threadIdx.x & 31) == 0) sh.warp_sum[threadIdx.x >> 5] = top;
        __syncthreads();
        if (threadIdx.x < ctas) {
            u64 s = 0;
            for (int w = 0; w < kWarps; w++) s += sh.warp_sum[w];
            cluster.map_shared_rank(&sh, threadIdx.x)->others[rank][0] = s;
        }
        cluster.sync();
        // ---- this CTA's share of the steps: what all their tokens weigh, by the middles, and the squares that the
        // sample's error goes by
        const int share = kSteps / ctas, per = share / kThreads, step0 = rank * share + int(threadIdx.x) * per;
        uint32_t* merged = reinterpret_cast<uint32_t*>(aux) + threadIdx.x * per;
        if (per == 1) {
            uint32_t n = 0;
#pragma unroll
            for (int c = 0; c < kMaxCluster; c++) n += cluster.map_shared_rank(counts(), c)[step0];  // side by side
            merged[0] = n;
        } else {
#pragma unroll 4
            for (int k = 0; k < per; k++) {
                uint32_t n = 0;
                for (int c = 0; c < ctas; c++) n += cluster.map_shared_rank(counts(), c)[step0 + k];
                merged[k] = n;
            }
        }
        auto weighed = [&](int k, u64& w, u64& q) {
            const uint32_t n = merged[k];
            const float one = middle(step0 + k, scale) * float(rate);
            w = static_cast<u64>(n) * static_cast<u64>(one), q = static_cast<u64>(float(n) * one * (one * float(1.0 / kSquare)));
        };
        u64 v[1] = {0}, q[1] = {0};
#pragma unroll 1
        for (int k = 0; k < per; k++) {
            u64 w, z;
            weighed(k, w, z);
            v[0] += w, q[0] += z;
        }
        u64 upto = 0 - v[0], upto_q = 0 - q[0];
        const u64 all = cta_upto(sh, v), all_q = cta_upto(sh, q);
        upto += v[0], upto_q += q[0];  // before this thread's steps
        if (threadIdx.x == 0) sh.bin = -1, sh.bin_end = kSteps - 1;
        if (threadIdx.x < ctas) cluster.map_shared_rank(&sh, threadIdx.x)->others[rank][1] = all_q;
        share_sum(all);
        u64 largest = 0, before = 0, sum = 0, before_q = 0, sum_q = 0;
        for (int i = 0; i < ctas; i++) {
            const u64 x = sh.sum[i], y = sh.others[i][1];
            largest += sh.others[i][0];
            before += i < rank ? x : 0ull, before_q += i < rank ? y : 0ull, sum += x, sum_q += y;
        }
        upto += before + largest, upto_q += before_q, sum += largest;
        // The first steps at which the sum may and must have reached its part. What the sample makes of a beginning less p times all
        // is off by (1 - p) of what is in it and p of what is not: three standard deviations, and a little for the middles.
        const long long want_near = static_cast<long long>(double(top_p) * double(sum));
        const float in = (1 - top_p) * (1 - top_p) * float(kSquare), out = top_p * top_p * float(kSquare), least = float(sum) * 0x1p-11f;
        auto margin = [&](u64 upto_q) {
            return rate > 1 ? static_cast<long long>(3.0f * sqrtf(in * float(upto_q) + out * float(sum_q - upto_q)) + least) : static_cast<long long>(least);
        };
        long long e_less = margin(upto_q);
#pragma unroll 1
        for (int k = 0; k < per; k++) {
            u64 w, z;
            weighed(k, w, z);
            if (!w) continue;
            const long long less = static_cast<long long>(upto) - want_near;
            upto += w, upto_q += z;
            const long long more = static_cast<long long>(upto) - want_near, e = margin(upto_q);
            const bool may = more + e >= 0 && less + e_less < 0, must = more - e >= 0 && less - e_less < 0;
            e_less = e;
            if (may || must)
                for (int c = 0; c < ctas; c++) {
                    Shared* o = cluster.map_shared_rank(&sh, c);
                    if (may) o->bin = step0 + k;
                    if (must) o->bin_end = step0 + k;
                }
        }
        cluster.sync();
        // none: the cut may be, or is, among the largest, which are not counted
        const int lo = max(sh.bin - 1, 0), hi = static_cast<long long>(largest) - want_near - margin(0) >= 0 ? min(count_step(t, scale) + 1, kSteps - 1) : sh.bin_end;
        // ---- one pass over the weights: the row's sum, the sum before the window, the window's tokens by finer steps
        u64* fine = reinterpret_cast<u64*>(counts());
        // the window: values from `bottom` to `top_value`; larger ones lie before it
        const float top_value = lo > 0 ? row.m - (float(lo) - 0.5f) / scale : INFINITY;
        const float bottom = hi < kSteps - 1 ? fmaxf(row.m - (float(hi) + 0.5f) / scale, -FLT_MAX) : -FLT_MAX;
        const float fine_scale = scale * (float(kFine) / float(hi - lo + 1)), fine_top = fminf(top_value, row.m);
        auto fine_step = [&](float x) { return int(fminf((fine_top - x) * fine_scale, float(kFine - 1))); };
        u64 part = 0, whole = 0;
        const unsigned room = window_room(ctas);
        each_of_segment([&](const float (&x)[4], int i) {
            u64 y[4];
            four_weights(row, sh.table, x, y);
            whole += (y[0] + y[1]) + (y[2] + y[3]);
            bool in[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (x[j] > top_value) part += y[j];
                in[j] = x[j] >= bottom && x[j] <= top_value;
            }
            const int n = in[0] + in[1] + in[2] + in[3];
            if (n) {
                unsigned at = atomicAdd(&sh.n_window, unsigned(n));
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    if (in[j] && at < room) window()[at] = entry(x[j], i + j);
                    at += in[j];
                }
            }
        });
        part = warp_total(part), whole = warp_total(whole);
        __syncthreads();
        for (int i = threadIdx.x; i < kFine; i += kThreads) fine[i] = 0;
        __syncthreads();
        const int n = int(min(sh.n_window, room));
        for (int i = threadIdx.x; i < n; i += kThreads) {
            const float x = value(window()[i]);
            atomicAdd(&fine[fine_step(x)], weight_of(x));
        }
        if ((threadIdx.x & 31) == 0) sh.seg[threadIdx.x >> 5] = part, sh.warp_sum[threadIdx.x >> 5] = whole;
        __syncthreads();
        if (threadIdx.x < ctas) {
            u64 p = 0, s = 0;
            for (int w = 0; w < kWarps; w++) p += sh.seg[w], s += sh.warp_sum[w];
            Shared* o = cluster.map_shared_rank(&sh, threadIdx.x);
            o->others[rank][0] = p, o->others[rank][1] = s + (sh.n_window > room ? 1ull << 63 : 0ull);  // no room: says so
        }
        cluster.sync();
        u64 ahead = 0, total = 0;
        bool fits = true;
        for (int i = 0; i < ctas; i++) {
            ahead += sh.others[i][0], total += sh.others[i][1] & ~(1ull << 63);
            fits &= !(sh.others[i][1] >> 63);
        }
        const double want = fmax(double(top_p) * double(total), 0.5);
        if (!fits || double(ahead) >= want) return false;
        // ---- the fine step of the cut, its tokens, the cut
        constexpr int kMostFine = kFine / kThreads;
        const int share_fine = kFine / ctas, per_fine = (share_fine + kThreads - 1) / kThreads;
        u64 f[kMostFine] = {}, own_fine[kMostFine];
        for (int c = 0; c < ctas; c++) {
            const u64* o = cluster.map_shared_rank(fine, c) + rank * share_fine;
#pragma unroll
            for (int k = 0; k < kMostFine; k++)
                if (k < per_fine && int(threadIdx.x) * per_fine + k < share_fine) f[k] += o[threadIdx.x * per_fine + k];
        }
#pragma unroll
        for (int k = 0; k < kMostFine; k++) own_fine[k] = f[k];
        const u64 of_cta = cta_upto(sh, f);
        if (threadIdx.x == 0) sh.bin = -1;
        share_sum(of_cta);
        for (int i = 0; i < rank; i++) ahead += sh.sum[i];
#pragma unroll
        for (int k = 0; k < kMostFine; k++) {
            const u64 upto = ahead + f[k], less = upto - own_fine[k];
            if (own_fine[k] && double(upto) >= want && double(less) < want)
                for (int c = 0; c < ctas; c++) {
                    Shared* o = cluster.map_shared_rank(&sh, c);
                    o->bin = rank * share_fine + int(threadIdx.x) * per_fine + k, o->before = less;
                }
        }
        cluster.sync();
        const int step = sh.bin;
        if (step < 0) return false;  // behind the window
        const u64 less = sh.before;
        for (int i = threadIdx.x; i < n; i += kThreads) {
            const u64 e = window()[i];
            const float x = value(e);
            if (fine_step(x) == step) put(x, int(0xFFFFFFFFu - uint32_t(e)));
        }
        gather([]() {});
        if (rank == 0) {
            u64 next = 0;
            const unsigned n_all = sh.n_all;
            if (n_all <= kCand) next = cut_in_list(int(n_all), want, less, true);
            if (threadIdx.x < ctas) {
                Shared* o = cluster.map_shared_rank(&sh, threadIdx.x);
                o->done = next != 0;
                if (next) o->cut = next;
            }
        }
        cluster.sync();
        if (!sh.done) return false;
        const int seg = segment();
        for (int i = threadIdx.x; i < n; i += kThreads) {
            const u64 e = window()[i];
            if (e >= sh.cut) atomicAdd(&sh.seg[(int(0xFFFFFFFFu - uint32_t(e)) - first) / kPer / seg], weight_of(value(e)));
        }
        __syncthreads();
        take_cut();
        return true;
    }
};

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) sample_rows_kernel(const neko_sample_rows_args a, int slice) {
    using S = Sampler<T>;
    extern __shared__ __align__(128) uint8_t sm[];
    Shared& sh = *reinterpret_cast<Shared*>(sm);
    constexpr int kAuxOff = (sizeof(Shared) + 127) / 128 * 128;
    S s(a, sh, sm + kAuxOff);
    s.ctas = int(s.cluster.num_blocks()), s.rank = int(s.cluster.block_rank());
    const int tid = threadIdx.x, lane = tid & 31, r = blockIdx.x / s.ctas, ctas = s.ctas;
    const int b = min(s.rank * slice, a.vocab), n = min(slice, a.vocab - b);
    const T* src = static_cast<const T*>(a.logits) + r * a.row_stride + b;
    const int ph = int(reinterpret_cast<uintptr_t>(src) & 15) / int(sizeof(T));  // places before the slice in its first vector
    s.nv = n ? (ph + n + S::kPer - 1) / S::kPer : 0;
    s.first = b - ph;
    s.data = reinterpret_cast<const uint4*>(src - ph);
    s.row.from = NAN;
    if (tid == 0) sh.best = 0xFFFFFFFFu, sh.n_all = 0, sh.total = 0, sh.cut = 0;
    const float asked = !a.u ? 0.0f : a.temperatures ? a.temperatures[r] : a.temperature;
    const float temperature = asked > 0.0f ? fminf(asked, 1e36f) : 0.0f;  // above, all weigh the same; NaN: greedy
    const float min_p = a.min_ps ? a.min_ps[r] : a.min_p, top_p = a.top_ps ? a.top_ps[r] : a.top_p;
    int top_k = a.top_ks ? a.top_ks[r] : a.top_k;
    if (top_k < 0 || top_k >= a.vocab) top_k = 0;
    if (tid < 2 * S::kPer && s.nv > (tid < S::kPer ? 0 : 1)) {
        const int at = (tid < S::kPer ? tid : (s.nv - 1) * S::kPer + tid - S::kPer) - ph;
        reinterpret_cast<T*>(sh.ends)[tid] = at >= 0 && at < n ? src[at] : T(-INFINITY);
    }
    if (temperature > 0.0f) {
        for (int i = tid; i < kPowers * kCopies; i += kThreads) sh.table[i] = exp2(double(i / kCopies) / kPowers);
        s.row.c = 1.4426950408889634 / double(temperature);
        s.row.c_powers = s.row.c * kPowers;
        s.row.c32 = fminf(float(s.row.c), 1e30f);
    }
    s.cluster.barrier_arrive();
    __syncthreads();
    // ---- the largest values, by groups of eight threads, to every CTA
    float most = -INFINITY;
    s.template each<4>([&](const float (&x)[4], int) { most = fmaxf(most, fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]))); });
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    s.cluster.barrier_wait();
    if ((tid & 7) < ctas) *s.cluster.map_shared_rank(&sh.gmax[s.rank * kGroups + tid / 8], tid & 7) = most;
    s.cluster.sync();
    const int groups = ctas * kGroups;
    float g = tid < groups ? sh.gmax[tid] : -INFINITY;
    float m = warp_max(g);
    if (lane == 0) reinterpret_cast<float*>(sh.warp_sum)[tid >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; w++) m = fmaxf(m, reinterpret_cast<float*>(sh.warp_sum)[w]);
    s.row.m = m;
    if (!(m > -INFINITY)) {  // nothing to take
        if (s.rank == 0 && tid == 0) s.answer(r, -1, 0.0f, 1);
        return;
    }

    // ---- greedy: the first maximum
    if (!(temperature > 0.0f)) {
        unsigned best = 0xFFFFFFFFu;
        s.template each<4>([&](const float (&x)[4], int i) {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (x[j] == m) best = min(best, unsigned(i + j));
        });
        best = __reduce_min_sync(0xffffffffu, best);
        if (lane == 0 && best != 0xFFFFFFFFu) atomicMin(s.cluster.map_shared_rank(&sh.best, 0), best);
        s.cluster.sync();
        if (s.rank == 0 && tid == 0) {
            a.token[r] = int(sh.best);
            if (a.prob) a.prob[r] = 1.0f;
        }
        return;
    }

    // Where the next value below m weighs 2^-128 of it or less, m is alone; else steps of the values near m are 256 powers of two at most,
    // which bounds what low adds to 46.5. Where low would lie below the lowest finite value, all finite values are within a factor of
    // 2 of m, so that differences from it are exact, and -infinity and places outside the row still weigh nothing.
    s.row.alone = !(double(fabsf(m)) * 0x1p-25 * s.row.c < 64.0);
    const double far = double(temperature) * (46.5 / 1.4426950408889634);
    if (s.row.alone || double(m) - far < -double(FLT_MAX)) {
        s.row.from = m;
        g = s.read(g), m = 0.0f, s.row.m = 0.0f;
    }
    s.row.m64 = double(m);
    s.row.low = __double2float_rd(s.row.m64 - far);
    s.row.cut = s.row.least = -INFINITY, s.row.cut_at = 0;
    if (min_p > 0.0f) {  // the least float with (m - x) c <= -log2(min_p): near the quotient, then one by one
        const double lim = fmax(-log2(double(min_p)), 0.0);
        auto in = [&](float x) { return (s.row.m64 - double(x)) * s.row.c <= lim; };
        float x = fminf(float(s.row.m64 - lim / s.row.c), m);
        for (int i = 0; i < 64 && !in(x); i++) x = fminf(nextafterf(x, INFINITY), m);
        for (int i = 0; i < 64 && in(nextafterf(x, -INFINITY)); i++) x = nextafterf(x, -INFINITY);
        s.row.least = x;
    }

    const bool use_p = top_p < 1.0f;
    bool ready = false;  // seg[] holds what is kept
    if (top_k || use_p) {
        const int want = top_k ? top_k : min(3 * groups / 4, 96);
        if (4 * want <= 3 * groups) {
            // the bound: a key that `want` groups reach, by halving below the bits that the largest has in common with the smallest group
            const uint32_t key = tid < groups ? order_key(g) : 0xFFFFFFFFu, top = order_key(m);
            uint32_t least = __reduce_min_sync(0xffffffffu, key);
            uint32_t* by_warp = reinterpret_cast<uint32_t*>(sh.warp_sum) + kWarps;  // behind the warps' largest, which others may still read
            if (lane == 0) by_warp[tid >> 5] = least;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < kWarps; w++) least = min(least, by_warp[w]);
            const int same = __clz(top ^ least);  // 32: all alike
            uint32_t bound = same ? top & ~(0xFFFFFFFFu >> (same - 1) >> 1) : 0u;
            const int last = max(min(31 - same - 8, 16), 0);
            for (int bit = 31 - same; bit >= last; bit--) {
                const uint32_t next = bound | 1u << bit;
                if (__syncthreads_count(tid < groups && key >= next) >= want) bound = next;
            }
            const float t = bound >= 0x00800000u ? key_value(bound) : -INFINITY;  // below: no finite value
            if (top_k) {
                if (s.few(r, t, top_k, use_p, top_p)) return;
            } else {
                ready = s.nucleus(t, top_p);
            }
        }
        if (!ready) {
#pragma unroll 1
            for (int mass = top_k ? 0 : 1; mass < (use_p ? 2 : 1); mass++) s.select(mass, top_k, top_p);
        }
    }
    if (s.row.least > s.row.cut) ready = false;
    s.cut_least();
    auto kept = [&](float x, int i) { return s.kept(x, i); };
    if (!ready) s.template fill<true>(kept);
    const unsigned long long total = s.template locate<true>(kept, [&](unsigned long long all) { return s.place(r, all); });
    if (tid == 0 && sh.found != 0xFFFFFFFFu) s.answer(r, int(sh.found), sh.pick, total);
}

template <typename T>
cudaError_t go(const neko_sample_rows_args& a, cudaStream_t st) {
    constexpr int kPer = 16 / sizeof(T);
    // As many CTAs a row as run at once (two an SM), slices of 4,096 tokens at least: 24 rows of 151,936, k = 40: 8 CTAs 15.1 us, 4 14.5,
    // nuclei 47 and 48; 64 rows 8 CTAs 28.2, 4 18.1, 2 19.3, nuclei 99, 68, 75. More rows than that: one each (320 x 50,257: 31.5 us,
    // two 40.8), but two where one would leave a wave of large slices nearly empty (320 x 151,936: 83 us, one 107).
    const int64_t room = 2 * num_sms();
    int ctas = 1;
    while (ctas < kMaxCluster && a.vocab > 4096 * ctas && a.rows * ctas * 2 <= room) ctas *= 2;
    if (a.rows > room && a.vocab > 100000) {
        auto waste = [&](int64_t n) { return double((a.rows * n + room - 1) / room) / double(a.rows * n); };
        if (waste(1) > 1.25 * waste(2)) ctas = 2;
    }
    const int slice = ((a.vocab + ctas - 1) / ctas + kPer - 1) / kPer * kPer;
    const size_t smem = (sizeof(Shared) + 127) / 128 * 128 + aux_bytes(ctas);
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
