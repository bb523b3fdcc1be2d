// Sampling a token per row of logits from a given uniform number.
//
//   d_i = (x_i - max x) / T,  w_i = exp(d_i)  (0 where d_i < -30),
//   rows ordered by (x descending, index ascending): keep the first k (top-k), then the
//   shortest prefix that holds a share p of what is kept (top-p), then w_i >= min_p,
//   token = first index, in index order, whose cumulative kept weight exceeds u * total.
//
// The token is a whole number that has to come out the same whatever the split, so weights are
// computed in 64 bits and summed as fixed-point integers of 44 fractional bits (the longest row
// has fewer than 2^20 tokens, so a sum stays below 2^64): sums do not depend on their order,
// borders move by 2^-45 per token.
//
// A thread-block cluster holds one row in the shared memory of its CTAs (the row is read from
// HBM once) and agrees on maxima, counts and sums through distributed shared memory.  Nothing
// is sorted as a whole: a histogram over 1023 bins of d (monotone in x) bounds the part of the
// row that can be kept, from counts alone (a bin's weights differ by 3%, so the nucleus is
// bounded from above).  Where at most kList tokens are left, one CTA settles those exactly;
// otherwise the cut is found bin by bin, from exact weights per bin, and inside its bin by finer
// buckets or, if ties make it large, by halving the range of values.
// Bound by the latency of those exchanges (barriers are the top stall; the 64-bit pipe is 7% busy).
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdlib>
#include <cstring>
#include <utility>

#include "common.cuh"
#include "decode_ops.h"
#include "kernels.h"

namespace cg = cooperative_groups;

namespace escha {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCtas = 8;                 // of a row's cluster
constexpr int kBins = 1024;                 // the last one is not counted: weight 0
constexpr int kList = 2048;
constexpr int kCounted = 256;               // tokens that are compared all with all
constexpr int kEach = kList / kThreads;     // listed tokens per thread
constexpr int kByMaxima = 1024;             // largest top-k that is bounded by the threads' maxima
constexpr int kNear = 5;                    // bins around where a top-p cut is expected
constexpr int kSparse = 2048;               // listed tokens of a slice (16-bit places over the counts)
constexpr float kCut = -30.0f;
constexpr int kFraction = 44;
constexpr double k512 = 738.65986093514925;  // 512 log2(e)
static_assert(kThreads == 512 && kBins == 2 * kThreads,
              "one thread per entry of the table of powers, and per two bins");
constexpr float kBinsPerNat = (kBins - 1) / 30.25f;
typedef unsigned long long u64;

template <typename T> __device__ __forceinline__ float to_float(T x);
template <> __device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float to_float(float x) { return x; }
template <typename T> __device__ __forceinline__ T lowest();      // -inf
template <> __device__ __forceinline__ __half lowest() { return __ushort_as_half(0xfc00); }
template <> __device__ __forceinline__ __nv_bfloat16 lowest() { return __ushort_as_bfloat16(0xff80); }
template <> __device__ __forceinline__ float lowest() { return __int_as_float(0xff800000); }

// Order-preserving key of a value, the same for both zeros.  (A NaN's key is of no
// consequence: it has no bin and no weight.)
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

struct Shared {
    double pow2[512];                       // 2^(j / 512)
    u64 best;                               // this CTA's largest (key, ~index)
    u64 sum;                                // this CTA's sum of weights
    u64 warp_sum[kWarps];
    u64 scan[kWarps];
    uint32_t scan32[kWarps];
    float scanf[kWarps];
    uint32_t ties;                          // this CTA's tokens at the cut
    uint32_t count;                         // a count exchanged between CTAs
    uint32_t found, found2;                 // a thread's find, for its CTA
    uint32_t list_n;                        // (leader) tokens in the list
    uint32_t cut_key;                       // (leader) the cut, for all CTAs
    uint32_t cut_ties;
    u64 bin_above;
    u64 near[kNear + 2];                    // weights of the bins around a cut, before them, of all
    u64 near_all[kNear + 2];                // the same of the row
    uint32_t warp_ties[kWarps];
    __align__(16) uint32_t hist[kBins];     // counts of this CTA
    __align__(16) uint32_t cum[kBins];      // counts of the row, inclusive prefix
    __align__(16) uint32_t work[2 * kList]; // sums by bucket; weights of listed tokens
    __align__(16) u64 list[kList];          // (leader) tokens as ~(key, ~index)
};

// Weight of a token in units of 2^-44.  2^(y / 512) = 2^(n / 512) * exp(r): a table for the
// 512ths, a Taylor series of degree 3 for |r| <= ln 2 / 1024 (remainder below 9e-15).
struct Weights {
    double top, inv512;                     // 512 log2(e) / T
    const double* pow2;
    __device__ __forceinline__ u64 operator()(float x) const {
        // no branches: the chains of several tokens overlap
        const double y = (static_cast<double>(x) - top) * inv512;
        const bool counts = y >= static_cast<double>(kCut) * k512;
        const double magic = 6755399441055744.0;                     // 1.5 * 2^52: rounds to integer
        const double shifted = y + magic;
        const int n = static_cast<int>(__double_as_longlong(shifted));
        const double r = y - (shifted - magic);
        constexpr double c = 0.0013538030870311433;                  // ln 2 / 512
        double e = fma(c * c * c / 6.0, r, c * c / 2.0);
        e = fma(e, r, c);
        e = fma(e, r, 1.0);
        const long long scale = static_cast<long long>((n >> 9) + kFraction) << 52;
        const double t = __longlong_as_double(__double_as_longlong(pow2[n & 511]) + scale);
        // t * e <= 2^44: adding 2^52 leaves the nearest integer in the low mantissa bits
        const u64 w = static_cast<u64>(__double_as_longlong(fma(t, e, 4503599627370496.0))) & 0xfffffffffffffull;
        return counts ? w : 0ull;
    }
};

// One word of each CTA of the cluster (0 past the last): the loads are in flight together.
template <typename V>
__device__ __forceinline__ void read_ranks(const cg::cluster_group& cluster, V* word, int ctas,
                                           V (&out)[kMaxCtas]) {
#pragma unroll
    for (int r = 0; r < kMaxCtas; ++r) out[r] = r < ctas ? *cluster.map_shared_rank(word, r) : V(0);
}

template <typename V>
__device__ __forceinline__ V warp_sum(V v) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}

// Inclusive prefix of a value per thread over the CTA; `scratch` one word per warp.
template <typename V>
__device__ __forceinline__ V block_inclusive(V v, V* scratch, V* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const V o = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) v += o;
    }
    __syncthreads();
    if (lane == 31) scratch[warp] = v;
    __syncthreads();
    V base = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        const V s = scratch[w];
        if (w < warp) base += s;
        all += s;
    }
    *total = all;
    return v + base;
}

__device__ __forceinline__ int power_of_two(int n) { return n <= 2 ? 2 : 1 << (32 - __clz(n - 1)); }

// What a row asks of its list.
struct ListRow {
    int64_t* token;
    int k;                                  // 0: no top-k
    bool p_on;
    float share;
    u64 least_w;
    int V;
};

// 64-bit sums by bucket, as low and high words (the low one's carry is seen by whoever causes
// it), and the first bucket at which their running sum exceeds `want`.
struct Buckets {
    uint32_t* lo;                           // [kBins]
    uint32_t* hi;
    __device__ __forceinline__ void clear() {
        for (int i = threadIdx.x; i < kBins / 2; i += kThreads)
            reinterpret_cast<uint4*>(lo)[i] = make_uint4(0, 0, 0, 0);      // lo and hi are neighbours
        __syncthreads();
    }
    __device__ __forceinline__ void add(int b, u64 w) {
        const uint32_t wl = static_cast<uint32_t>(w);
        const uint32_t old = atomicAdd(&lo[b], wl);
        const uint32_t up = static_cast<uint32_t>(w >> 32) + (old + wl < old);
        if (up) atomicAdd(&hi[b], up);
    }
    // found, above: one shared word each, the bucket and the sum before it
    __device__ __forceinline__ void find(u64 want, u64* scratch, uint32_t* found, u64* above) {
        __syncthreads();
        const uint2 l = reinterpret_cast<const uint2*>(lo)[threadIdx.x];
        const uint2 h = reinterpret_cast<const uint2*>(hi)[threadIdx.x];
        const u64 w[2] = {(static_cast<u64>(h.x) << 32) + l.x, (static_cast<u64>(h.y) << 32) + l.y};
        u64 total;
        const u64 mine = w[0] + w[1];
        u64 before = block_inclusive(mine, scratch, &total) - mine;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            if (before <= want && want < before + w[e]) {
                *found = 2 * threadIdx.x + e;
                *above = before;
            }
            before += w[e];
        }
        __syncthreads();
    }
};

// Threads that share a token when `count` tokens are compared all with all: within a warp, at
// most a warp, and a divisor of the block.
__device__ __forceinline__ int threads_per(int count) {
    return count <= kThreads / 32 ? 32 : count <= kThreads ? kThreads / power_of_two(count) : 1;
}

// Of tokens ordered by (bucket, key), both ascending, the key at which the running sum of w
// exceeds `want`.  Up to kEach tokens per thread; those with w == 0 are not there.  Sums by
// bucket first, then all with all inside the one bucket.  Writes s.work and s.list.
__device__ u64 locate(Shared& s, const int (&bucket)[kEach], const u64 (&key)[kEach], const u64 (&w)[kEach],
                      u64 want) {
    const int tid = threadIdx.x, lane = tid & 31;
    Buckets b{s.work, s.work + kBins};
    __syncthreads();
    b.clear();
#pragma unroll
    for (int e = 0; e < kEach; ++e)
        if (w[e] != 0) b.add(bucket[e], w[e]);
    if (tid == 0) s.count = 0;
    b.find(want, s.scan, &s.found, &s.bin_above);
    const int at = s.found;
    want -= s.bin_above;
    u64* ws = reinterpret_cast<u64*>(s.work);             // the buckets are read
#pragma unroll
    for (int e = 0; e < kEach; ++e)
        if (w[e] != 0 && bucket[e] == at) {
            const uint32_t i = atomicAdd(&s.count, 1u);
            s.list[i] = key[e];
            ws[i] = w[e];
        }
    __syncthreads();
    const int n = s.count, per = threads_per(n);
    const unsigned group = per == 32 ? 0xffffffffu : ((1u << per) - 1) << (lane / per * per);
    for (int i = tid / per; i < n; i += kThreads / per) {
        const u64 k = s.list[i];
        u64 before = 0;
        for (int j = tid % per; j < n; j += per)
            if (s.list[j] < k) before += ws[j];
        for (int d = 1; d < per; d <<= 1) before += __shfl_xor_sync(group, before, d);
        if (before <= want && want < before + ws[i]) s.best = k;
    }
    __syncthreads();
    return s.best;
}

__device__ __forceinline__ u64 sum_of(Shared& s, const u64 (&w)[kEach]) {
    u64 mine = 0, total;
#pragma unroll
    for (int e = 0; e < kEach; ++e) mine += w[e];
    block_inclusive(mine, s.scan, &total);
    return total;
}

// Settles a row whose kept tokens are all among the `count` of s.list (any order), by one CTA.
// `all`: weight of the whole row, 0: that of the list (its first k).
template <class W, class B, class G>
__device__ void settle_list(Shared& s, int count, const ListRow& r, const W& weight, const B& bin_of,
                            const G& target_of, u64 all) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (count <= kCounted) {
        const int per = threads_per(count), i = tid / per, part = tid % per;
        u64* ws = reinterpret_cast<u64*>(s.work);         // weights by rank, then the kept ones
        int* at = reinterpret_cast<int*>(s.work + 2 * kCounted);
        const u64 x = i < count ? s.list[i] : 0;
        int ahead = 0;
        if (i < count)
            for (int j = part; j < count; j += per) ahead += s.list[j] < x;
        for (int d = 1; d < per; d <<= 1) ahead += __shfl_xor_sync(0xffffffffu, ahead, d);
        const int index = static_cast<int>(0xffffffffu - static_cast<uint32_t>(~x));
        if (i < count && part == 0) {
            ws[ahead] = weight(value_of(static_cast<uint32_t>(~x >> 32)));
            at[ahead] = index;
        }
        __syncthreads();
        if (warp == 0) {
            constexpr int kMine = kCounted / 32;
            u64 w[kMine], mine = 0;
#pragma unroll
            for (int e = 0; e < kMine; ++e) {
                const int j = lane * kMine + e;
                w[e] = j < count && (r.k == 0 || j < r.k) ? ws[j] : 0;
                mine += w[e];
            }
            u64 inc = mine;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const u64 o = __shfl_up_sync(0xffffffffu, inc, d);
                if (lane >= d) inc += o;
            }
            u64 before = inc - mine;
            const u64 total = __shfl_sync(0xffffffffu, inc, 31);
            const double want = static_cast<double>(r.share) * static_cast<double>(all ? all : total);
            mine = 0;
#pragma unroll
            for (int e = 0; e < kMine; ++e) {
                const int j = lane * kMine + e;
                const bool keep = w[e] >= r.least_w && (!r.p_on || j == 0 || static_cast<double>(before) < want);
                before += w[e];
                if (!keep) w[e] = 0;
                if (j < count) ws[j] = w[e];
                mine += w[e];
            }
            mine = warp_sum(mine);
            if (lane == 0) s.bin_above = target_of(mine);
        }
        __syncthreads();
        const u64 want = s.bin_above;
        u64 upto = 0;
        if (i < count)
            for (int j = part; j < count; j += per) upto += at[j] <= index ? ws[j] : 0;
        for (int d = 1; d < per; d <<= 1) upto += __shfl_xor_sync(0xffffffffu, upto, d);
        if (i < count && part == 0 && upto - ws[ahead] <= want && want < upto) *r.token = index;
        return;
    }

    u64 x[kEach], w[kEach];
    int bucket[kEach];
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        const int i = tid + e * kThreads;
        x[e] = i < count ? s.list[i] : ~0ull;
        const float v = value_of(static_cast<uint32_t>(~x[e] >> 32));
        bucket[e] = i < count ? bin_of(v) : 0;
        w[e] = i < count ? weight(v) : 0;
    }
    if (r.k > 0) {
        u64 one[kEach];                                   // tokens that weigh something
#pragma unroll
        for (int e = 0; e < kEach; ++e) one[e] = w[e] != 0;
        if (static_cast<u64>(r.k) < sum_of(s, one)) {
            const u64 cut = locate(s, bucket, x, one, r.k - 1);
#pragma unroll
            for (int e = 0; e < kEach; ++e)
                if (x[e] > cut) w[e] = 0;
        }
    }
    if (r.p_on) {
        const u64 total = sum_of(s, w);
        // kept while the sum before a token is below share * total: up to the first token at
        // which the running sum exceeds the last whole number below that
        const double want_d = ceil(static_cast<double>(r.share) * static_cast<double>(all ? all : total)) - 1.0;
        u64 want = want_d > 0.0 ? static_cast<u64>(want_d) : 0ull;
        if (want > total - 1) want = total - 1;
        const u64 cut = locate(s, bucket, x, w, want);
#pragma unroll
        for (int e = 0; e < kEach; ++e)
            if (x[e] > cut) w[e] = 0;
    }
    const int shift = max(0, 32 - __clz(r.V - 1) - 10);   // 1024 ranges of indices
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        if (w[e] < r.least_w) w[e] = 0;
        x[e] = 0xffffffffu - static_cast<uint32_t>(~x[e]);
        bucket[e] = static_cast<int>(x[e] >> shift) & (kBins - 1);
    }
    const u64 want = target_of(sum_of(s, w));
    const u64 token = locate(s, bucket, x, w, want);
    if (tid == 0) *r.token = static_cast<int64_t>(token);
}

// RESIDENT: CTAs that share an SM, 2 at 64 registers a thread, 1 at what it likes (100).  One where
// the launch has no more CTAs than the GPU has SMs: 16 rows of 50257 binary32 30.0 us against
// 35.4, one row of 151936 binary16 9.1 against 9.9; 64 rows 59 us against 54.
template <typename T, int RESIDENT>
__global__ void __launch_bounds__(kThreads, RESIDENT) sample_kernel(const SampleParams p) {
    extern __shared__ __align__(16) uint8_t smem[];
    Shared& s = *reinterpret_cast<Shared*>(smem);
    T* xs = reinterpret_cast<T*>(smem + sizeof(Shared));
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = cluster.block_rank(), ctas = cluster.num_blocks();
    int row = blockIdx.x / ctas;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    grid_launch_dependents();
    s.pow2[tid] = exp2(tid / 512.0);
    if (tid == 0) s.list_n = 0;
    grid_dependency_wait();
    if (p.by_length) {
        // Rows that may keep most of the vocabulary take two to three times as long as those with
        // a small top-k or none to draw: where rows wait for a place, the long ones go first.
        int k = 0;
        float t = 0.0f;
        if (tid < p.B) {
            t = p.temperature ? p.temperature[tid] : p.temperature1;
            k = p.top_k ? p.top_k[tid] : p.top_k1;
        }
        const uint32_t is_long = tid < p.B && t > 0.0f && !(k > 0 && k <= kByMaxima);
        uint32_t all;
        const uint32_t upto = block_inclusive(is_long, s.scan32, &all);
        const int place = is_long ? upto - 1 : all + (tid - upto);
        if (tid < p.B && place == row) s.found = tid;
        __syncthreads();
        row = s.found;
    }

    // settings of the row, on their way while the logits are read
    const float temperature = p.temperature ? p.temperature[row] : p.temperature1;
    const int k = p.top_k ? p.top_k[row] : p.top_k1;
    const float share0 = p.top_p ? p.top_p[row] : p.top_p1;
    const float least0 = p.min_p ? p.min_p[row] : p.min_p1;
    const float u = p.uniforms[row];

    // ---- the CTA's slice (filled up with -inf), and the row's maximum with its lowest index
    const int base = rank * p.slice;
    const int n = min(max(p.V - base, 0), p.slice);
    const T* src = static_cast<const T*>(p.logits) + static_cast<long>(row) * p.stride + base;
    constexpr int kVec = 16 / sizeof(T);
    const int vecs = p.slice / kVec;
    uint4* const xv = reinterpret_cast<uint4*>(xs);
    float most = __int_as_float(0xff800000);
    int most_at = 0;
    auto take = [&](int i, T raw) {
        // a thread's indices ascend, so the first of equals stays
        const float x = to_float(raw);
        if (x > most) { most = x; most_at = i; }
    };
    const bool aligned = (reinterpret_cast<uintptr_t>(src) & 15) == 0;
    const int whole = aligned ? n / kVec : 0;             // vectors read as such
    constexpr int kBatch = 4;                             // loads in flight per thread
    for (int v0 = tid; v0 < whole; v0 += kBatch * kThreads) {
        uint4 q[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j)
            if (v0 + j * kThreads < whole) q[j] = reinterpret_cast<const uint4*>(src)[v0 + j * kThreads];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const int v = v0 + j * kThreads;
            if (v >= whole) break;
            xv[v] = q[j];
            const T* e = reinterpret_cast<const T*>(&q[j]);
#pragma unroll
            for (int k = 0; k < kVec; ++k) take(v * kVec + k, e[k]);
        }
    }
    const int head_of_rest = whole * kVec;                // the rest, token by token
    for (int i0 = head_of_rest + tid; i0 < p.slice; i0 += 2 * kBatch * kThreads) {
        T q[2 * kBatch];
#pragma unroll
        for (int j = 0; j < 2 * kBatch; ++j)
            q[j] = i0 + j * kThreads < n ? src[i0 + j * kThreads] : lowest<T>();
#pragma unroll
        for (int j = 0; j < 2 * kBatch; ++j)
            if (i0 + j * kThreads < p.slice) xs[i0 + j * kThreads] = q[j];
    }
    __syncthreads();
    // a thread's maximum is over the vectors that it owns in every later pass too
    for (int v = whole + (tid + kThreads - whole % kThreads) % kThreads; v < vecs; v += kThreads) {
        const uint4 q = xv[v];
        const T* e = reinterpret_cast<const T*>(&q);
#pragma unroll
        for (int k = 0; k < kVec; ++k) take(v * kVec + k, e[k]);
    }
    u64 best = static_cast<u64>(key_of(most)) << 32 | (0xffffffffu - (base + most_at));
#pragma unroll
    for (int d = 16; d; d >>= 1) {
        const u64 o = __shfl_xor_sync(0xffffffffu, best, d);
        best = o > best ? o : best;
    }
    if (lane == 0) s.scan[warp] = best;
    __syncthreads();
    if (tid == 0) {
#pragma unroll
        for (int w = 1; w < kWarps; ++w) best = s.scan[w] > best ? s.scan[w] : best;
        s.best = best;
    }
    for (int i = tid; i < kBins; i += kThreads) s.hist[i] = 0;
    cluster.sync();
    best = 0;
    {
        u64 o[kMaxCtas];
        read_ranks(cluster, &s.best, ctas, o);
#pragma unroll
        for (int r = 0; r < kMaxCtas; ++r) best = o[r] > best ? o[r] : best;
    }
    float top = value_of(static_cast<uint32_t>(best >> 32));
    const int top_index = static_cast<int>(0xffffffffu - static_cast<uint32_t>(best));
    const bool empty = top == __int_as_float(0xff800000);
    if (empty || !(temperature > 0.0f)) {
        if (rank == 0 && tid == 0) p.tokens[row] = empty ? -1 : top_index;
        cluster.sync();                     // no CTA leaves while its memory is read
        return;
    }
    const float share = fmaxf(share0, 0.0f), least = fminf(least0, 1.0f);
    bool k_on = k > 0 && k < p.V;
    const bool p_on = share0 < 1.0f, m_on = least > 0.0f;
    const u64 least_w = m_on ? static_cast<u64>(ceil(static_cast<double>(least) * (1ull << kFraction))) : 0;

    auto value = [&](int i) { return to_float(xs[i]); };
    if (top == __int_as_float(0x7f800000)) {
        // infinite logits take everything: 0 where x is infinite, -inf elsewhere
        __syncthreads();
        for (int i = tid; i < p.slice; i += kThreads) xs[i] = value(i) == top ? T(0.0f) : lowest<T>();
        if (most == top) most = 0.0f;
        else most = __int_as_float(0xff800000);
        top = 0.0f;
        __syncthreads();
    }
    Weights weight;
    weight.top = top;
    weight.inv512 = k512 / static_cast<double>(temperature);
    weight.pow2 = s.pow2;
    // bins of (top - x) / T; a finite factor, so that the top itself has bin 0 at any
    // temperature, and half the difference, which does not overflow
    const float bins = fminf(2.0f * kBinsPerNat / temperature, 3e38f), half_top = 0.5f * top;
    auto place_of = [&](float x) { return fmaf(-0.5f, x, half_top) * bins; };
    auto bin_of = [&](float x) {
        const float z = place_of(x);
        return z < static_cast<float>(kBins - 1) ? static_cast<int>(z) : kBins - 1;
    };
    // token to take from a total, as a cumulative weight that has to be exceeded
    auto target_of = [&](u64 total) {
        const double t = floor(static_cast<double>(u) * static_cast<double>(total));
        const u64 most = total - 1;
        return t >= static_cast<double>(most) ? most : t > 0.0 ? static_cast<u64>(t) : 0ull;
    };

    // In index order a warp has a contiguous part of the slice, 32 vectors at a time.
    const int part_vecs = (vecs + kWarps - 1) / kWarps;
    const int first_vec = min(warp * part_vecs, vecs), last_vec = min(first_vec + part_vecs, vecs);
    // tokens of the slice that can be kept, by index (over the counts); -1: not listed
    uint16_t* const left = reinterpret_cast<uint16_t*>(s.hist);
    int sparse = -1;
    // bins around a top-p cut, and this part's kept weight in those before them
    int near_lo = -1, near_hi = -2;
    u64 kept_ahead = 0;

    // ---- the cut: kept are keys above cut_key and the first cut_ties (by index) at it
    uint32_t cut_key = 0, cut_ties = 0xffffffffu;
    if (k_on || p_on || m_on) {
        Shared* leader = cluster.map_shared_rank(&s, 0);
        const int my_bin = bin_of(most);                  // the first bin among this thread's tokens
        // tokens of bins [from, to] to the leader's list (as far as it has room)
        auto gather = [&](int from, int to) {
            if (__ballot_sync(0xffffffffu, my_bin <= to) == 0) return;
            const float lowest_z = from, highest_z = min(to + 1, kBins - 1);
            // 64 tokens per thread and round: their hits as a mask, one reservation per warp
            constexpr int kRound = 64 / kVec;
            for (int v0 = 0; v0 < vecs; v0 += kRound * kThreads) {
                u64 hits = 0;
                if (my_bin <= to) {
#pragma unroll
                    for (int j = 0; j < kRound; ++j) {
                        const int v = v0 + j * kThreads + tid;
                        if (v >= vecs) break;
                        const uint4 q = xv[v];
                        const T* e = reinterpret_cast<const T*>(&q);
                        unsigned some = 0;
#pragma unroll
                        for (int k = 0; k < kVec; ++k) {
                            const float z = place_of(to_float(e[k]));
                            if (z >= lowest_z && z < highest_z) some |= 1u << k;
                        }
                        hits |= static_cast<u64>(some) << (j * kVec);
                    }
                }
                if (__ballot_sync(0xffffffffu, hits != 0) == 0) continue;
                int inc = __popcll(hits);
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const int o = __shfl_up_sync(0xffffffffu, inc, d);
                    if (lane >= d) inc += o;
                }
                uint32_t at = 0;
                if (lane == 31) at = atomicAdd(&leader->list_n, static_cast<uint32_t>(inc));
                at = __shfl_sync(0xffffffffu, at, 31) + inc - __popcll(hits);
                for (; hits; hits &= hits - 1, ++at) {
                    const int k = __ffsll(hits) - 1;
                    const int i = (v0 + k / kVec * kThreads + tid) * kVec + k % kVec;
                    // ascending: the largest value, then the lowest index, first
                    if (at < kList)
                        leader->list[at] = ~(static_cast<u64>(key_of(value(i))) << 32 | (0xffffffffu - (base + i)));
                }
            }
        };
        // counts of the row by bin, from those of the CTAs: an inclusive prefix in s.cum, the
        // thread's four bins in c, its prefix before them returned
        uint2 c;
        uint32_t counted;
        auto merge = [&]() {
            uint2 o[kMaxCtas];
#pragma unroll
            for (int r = 0; r < kMaxCtas; ++r)
                o[r] = r < ctas ? reinterpret_cast<const uint2*>(cluster.map_shared_rank(s.hist, r))[tid]
                                : make_uint2(0, 0);
            c = o[0];
#pragma unroll
            for (int r = 1; r < kMaxCtas; ++r) {
                c.x += o[r].x;
                c.y += o[r].y;
            }
            if (tid == 0) s.found = s.found2 = kBins - 1;
            const uint32_t mine = c.x + c.y;
            const uint32_t before = block_inclusive(mine, s.scan32, &counted) - mine;
            reinterpret_cast<uint2*>(s.cum)[tid] = make_uint2(before + c.x, before + mine);
            return before;
        };
        // the bin in which the count-th token lies (the last: not among the counted); a barrier
        auto bin_of_count = [&](uint32_t before, uint32_t count) {
            if (before < count && count <= before + c.x + c.y)
                s.found = 2 * tid + (count <= before + c.x ? 0 : 1);
            __syncthreads();
            return static_cast<int>(s.found);
        };
        int m_bin = kBins - 1;
        if (m_on) m_bin = min(kBins - 1, static_cast<int>((-logf(least) + 1e-3f) * kBinsPerNat));
        const ListRow row_of{p.tokens + row, k_on ? k : 0, p_on, share, least_w, p.V};

        if (k_on && k <= kByMaxima) {
            // ---- a small top-k: the count-th largest of the threads' maxima is a lower bound
            // of the count-th largest token, and nearly as large where k is far fewer than the
            // threads; only the maxima are counted (all tokens: 5 us of shared-memory atomics)
            if (my_bin < kBins - 1) atomicAdd(&s.hist[my_bin], 1u);
            cluster.sync();
            const uint32_t before = merge();
            if (static_cast<uint32_t>(k) <= counted) {
                const int k_bin = bin_of_count(before, k);
                gather(0, p_on ? k_bin : min(k_bin, m_bin));
                cluster.sync();
                const uint32_t got = leader->list_n;
                if (got <= kList) {
                    cluster.sync();                       // the others leave, for another row
                    if (rank == 0) settle_list(s, static_cast<int>(got), row_of, weight, bin_of, target_of, 0);
                    return;
                }
            }
            cluster.sync();                               // all have read the counts and list_n
            if (rank == 0 && tid == 0) s.list_n = 0;
            for (int i = tid; i < kBins; i += kThreads) s.hist[i] = 0;
            __syncthreads();
        }

        // ---- counts of all tokens by bin, as far as they can matter: without top-k, those that
        // weigh less than (1 - p) / V of the largest together weigh less than top-p leaves out
        int last = kBins - 1;
        if (p_on && !k_on)
            last = min(last, static_cast<int>((logf(static_cast<float>(p.V) / (1.0f - share)) + 1e-2f) * kBinsPerNat) + 1);
        else if (!k_on) last = min(last, m_bin + 1);
        for (int v = tid; v < vecs; v += kThreads) {
            const uint4 q = xv[v];
            const T* e = reinterpret_cast<const T*>(&q);
#pragma unroll
            for (int k = 0; k < kVec; ++k) {
                const float z = place_of(to_float(e[k]));
                if (z < static_cast<float>(last)) atomicAdd(&s.hist[static_cast<int>(z)], 1u);
            }
        }
        cluster.sync();
        const uint32_t before_bins = merge();
        // tokens past the counted bins weigh nothing, so a top-k that reaches them cuts nothing
        k_on = k_on && static_cast<uint32_t>(k) <= counted;
        const int k_bin = k_on ? bin_of_count(before_bins, k) : kBins - 1;
        // Top-p without top-k: the bins' weights lie within 3% (a thousandth for rounding), so
        // the cut is surely not past p_bin, and probably within two bins of p_near.
        int p_bin = last - 1, p_near = 0;
        if (p_on && !k_on) {
            auto low = [](int b) { return exp2f((b + 1) * (-1.44269504f / kBinsPerNat)) * 0.999f; };
            constexpr float kHigh = 1.033f;               // top of a bin over its low
            const float w0 = c.x * low(2 * tid), w1 = w0 + c.y * low(2 * tid + 1);
            float total;
            const float before = block_inclusive(w1, s.scanf, &total) - w1;
            // the first bins at which the running sum reaches what is surely, and what is probably
            // enough (tokens that were not counted weigh 1 - share at most)
            auto first = [&](float want, uint32_t* found) {
                const bool reached = before + w1 >= want;
                const unsigned m = __ballot_sync(0xffffffffu, reached);
                if (reached && lane == __ffs(m) - 1) atomicMin(found, 2u * tid + (before + w0 >= want ? 0 : 1));
            };
            first(share * (total * kHigh + (1.0f - share)) * 1.0001f, &s.found);
            first(share * total, &s.found2);
            __syncthreads();
            p_bin = min(static_cast<int>(s.found), last - 1);
            p_near = min(static_cast<int>(s.found2), last - 1);
        }
        __syncthreads();                                  // s.cum
        const int bound = k_on ? (p_on ? k_bin : min(k_bin, m_bin)) : min(p_bin, m_bin);
        const uint32_t kept = s.cum[bound];
        if (kept <= kList) {
            // ---- everything that can be kept fits the list: one CTA settles the row
            gather(0, bound);
            u64 sum = 0;
            if (p_on && !k_on) {                          // top-p asks for the weight of the row
                for (int v = tid; v < vecs; v += kThreads) {
                    const uint4 q = xv[v];
                    const T* e = reinterpret_cast<const T*>(&q);
#pragma unroll
                    for (int k = 0; k < kVec; ++k) sum += weight(to_float(e[k]));
                }
                u64 mine;
                block_inclusive(sum, s.scan, &mine);
                if (tid == 0) s.sum = mine;
            }
            cluster.sync();
            u64 all = 0;
            if (rank == 0 && p_on && !k_on) {
                u64 o[kMaxCtas];
                read_ranks(cluster, &s.sum, ctas, o);
#pragma unroll
                for (int r = 0; r < kMaxCtas; ++r) all += o[r];
            }
            cluster.sync();                               // the others leave, for another row
            if (rank == 0) {
                ListRow r = row_of;
                if (!k_on) r.k = 0;
                settle_list(s, static_cast<int>(kept), r, weight, bin_of, target_of, all);
            }
            return;
        }

        // ---- more than that is left: list this CTA's share by index, if it is few
        if (k_on || !p_on) {
            cluster.sync();                               // every CTA has read the counts
            auto hits_of = [&](int v) {                   // tokens of a vector that are left
                unsigned hits = 0;
                if (v < last_vec) {
                    const uint4 q = xv[v];
                    const T* e = reinterpret_cast<const T*>(&q);
#pragma unroll
                    for (int k = 0; k < kVec; ++k) {
                        const int b = bin_of(to_float(e[k]));
                        if (b <= bound && b < kBins - 1) hits |= 1u << k;
                    }
                }
                return hits;
            };
            uint32_t mine_n = 0;
            for (int v = first_vec + lane; v < last_vec; v += 32) mine_n += __popc(hits_of(v));
            mine_n = warp_sum(mine_n);
            if (lane == 0) s.scan32[warp] = mine_n;
            __syncthreads();
            uint32_t at = 0, all_n = 0;
            for (int w = 0; w < kWarps; ++w) {
                if (w < warp) at += s.scan32[w];
                all_n += s.scan32[w];
            }
            if (all_n <= kSparse && p.slice <= 65536) {
                sparse = all_n;
                for (int v0 = first_vec; v0 < last_vec; v0 += 32) {
                    unsigned hits = hits_of(v0 + lane);
                    uint32_t inc = __popc(hits);
#pragma unroll
                    for (int d = 1; d < 32; d <<= 1) {
                        const uint32_t o = __shfl_up_sync(0xffffffffu, inc, d);
                        if (lane >= d) inc += o;
                    }
                    uint32_t to = at + inc - __popc(hits);
                    for (; hits; hits &= hits - 1) left[to++] = (v0 + lane) * kVec + __ffs(hits) - 1;
                    at += __shfl_sync(0xffffffffu, inc, 31);
                }
            }
            __syncthreads();
        }

        // ---- the cut bin by bin.  Sum of a count and a weight over the cluster.
        auto agree = [&](uint32_t cnt, u64 w, uint32_t* all_cnt, u64* all_w) {
            cnt = warp_sum(cnt);
            w = warp_sum(w);
            if (lane == 0) { s.scan32[warp] = cnt; s.warp_sum[warp] = w; }
            __syncthreads();
            if (tid == 0) {
                cnt = 0; w = 0;
                for (int i = 0; i < kWarps; ++i) { cnt += s.scan32[i]; w += s.warp_sum[i]; }
                s.count = cnt; s.sum = w;
            }
            cluster.sync();
            *all_cnt = 0; *all_w = 0;
            for (int r = 0; r < ctas; ++r) {
                *all_cnt += *cluster.map_shared_rank(&s.count, r);
                *all_w += *cluster.map_shared_rank(&s.sum, r);
            }
            cluster.sync();
        };
        // Inside bin `bin`: the value and its ties at which the first `count` tokens, or the
        // shortest prefix with a weight of at least `need`, end.
        auto cut_in_bin = [&](int bin, uint32_t size, bool by_count, uint32_t count, u64 need) {
            if (size <= kList) {
                gather(bin, bin);
                cluster.sync();
                if (rank == 0) {
                    // buckets: a 1024th of the bin each
                    u64 x[kEach], w[kEach];
                    int sub[kEach];
                    const u64 goal = by_count ? count : need;
#pragma unroll
                    for (int e = 0; e < kEach; ++e) {
                        const int i = tid + e * kThreads;
                        x[e] = i < size ? s.list[i] : ~0ull;
                        const uint32_t key = static_cast<uint32_t>(~x[e] >> 32);
                        const float v = value_of(key);
                        w[e] = i >= size ? 0 : by_count ? 1 : key >= cut_key ? weight(v) : 0;
                        const float z = place_of(v) - static_cast<float>(bin);
                        sub[e] = min(max(static_cast<int>(z * kBins), 0), kBins - 1);
                    }
                    const u64 last_kept = locate(s, sub, x, w, goal - 1);
                    u64 same[kEach];
#pragma unroll
                    for (int e = 0; e < kEach; ++e) same[e] = x[e] <= last_kept && (x[e] ^ last_kept) >> 32 == 0;
                    const u64 ties = sum_of(s, same);
                    if (tid == 0) {
                        s.cut_key = static_cast<uint32_t>(~last_kept >> 32);
                        s.cut_ties = static_cast<uint32_t>(ties);
                    }
                    if (tid == 0) s.list_n = 0;
                }
                cluster.sync();
                cut_key = leader->cut_key;
                cut_ties = leader->cut_ties;
                return;
            }
            // largest key t with enough tokens (weight) at or above it, bit by bit
            uint32_t t = 0, above = 0;
            u64 above_w = 0;
            for (int bit = 31; bit >= 0; --bit) {
                const uint32_t trial = t | 1u << bit;
                uint32_t cnt = 0;
                u64 w = 0;
                for (int i = tid; i < n; i += kThreads) {
                    const float x = value(i);
                    if (bin_of(x) == bin && key_of(x) >= trial && key_of(x) >= cut_key) {
                        ++cnt;
                        if (!by_count) w += weight(x);
                    }
                }
                uint32_t all_cnt;
                u64 all_w;
                agree(cnt, w, &all_cnt, &all_w);
                if (by_count ? all_cnt >= count : all_w >= need) t = trial;
                else { above = all_cnt; above_w = all_w; }
            }
            // `above` counts the tokens above t: the last trial that failed was the next key up
            uint32_t ties = count - above;
            if (!by_count) {
                const u64 w = weight(value_of(t));
                ties = w ? static_cast<uint32_t>((need - above_w + w - 1) / w) : 0xffffffffu;
            }
            cut_ties = t == cut_key ? min(ties, cut_ties) : ties;
            cut_key = t;
        };
        if (k_on) {
            const uint32_t above = k_bin ? s.cum[k_bin - 1] : 0;
            cut_in_bin(k_bin, s.cum[k_bin] - above, true, k - above, 0);
        }
        bool settled = !p_on;
        if (p_on && !k_on) {
            // One pass over the tokens (each thread its part in index order): the exact weights
            // of the bins before the cut's neighbourhood, of each bin in it and of those behind.
            near_lo = max(p_near - 2, 0);
            near_hi = min(p_near + 2, last - 1);
            uint32_t* lo = s.work;
            if (tid < 2 * kNear) lo[tid] = 0;
            __syncthreads();
            u64 ahead = 0, whole = 0;
            const float from = static_cast<float>(near_lo), upto = static_cast<float>(near_hi + 1);
            for (int v = first_vec + lane; v < last_vec; v += 32) {
                const uint4 q = xv[v];
                const T* e = reinterpret_cast<const T*>(&q);
#pragma unroll
                for (int k = 0; k < kVec; ++k) {
                    const float x = to_float(e[k]), z = place_of(x);
                    const u64 w = weight(x);
                    whole += w;
                    if (z < from) ahead += w;
                    if (m_on) kept_ahead += z < from && w >= least_w ? w : 0;
                    if (z >= from && z < upto) Buckets{lo, lo + kNear}.add(static_cast<int>(z) - near_lo, w);
                }
            }
            if (!m_on) kept_ahead = ahead;
            ahead = warp_sum(ahead);
            whole = warp_sum(whole);
            if (lane == 0) {
                s.warp_sum[warp] = ahead;
                s.scan[warp] = whole;
            }
            __syncthreads();
            if (tid < kNear) s.near[tid] = (static_cast<u64>(lo[kNear + tid]) << 32) + lo[tid];
            else if (tid < kNear + 2) {
                u64 t = 0;
                for (int w = 0; w < kWarps; ++w) t += tid == kNear ? s.warp_sum[w] : s.scan[w];
                s.near[tid] = t;
            }
            cluster.sync();
            u64* sums = s.near_all;
            if (tid < kNear + 2) {
                u64 o[kMaxCtas], t = 0;
                read_ranks(cluster, s.near + tid, ctas, o);
#pragma unroll
                for (int r = 0; r < kMaxCtas; ++r) t += o[r];
                sums[tid] = t;
            }
            __syncthreads();
            u64 before = sums[kNear];
            const u64 total = sums[kNear + 1];
            const double want_d = ceil(static_cast<double>(share) * static_cast<double>(total));
            u64 want = want_d > 1.0 ? static_cast<u64>(want_d) : 1ull;
            if (want > total) want = total;
            int bin = -1;
            u64 need = 0;
            if (want > before)
                for (int b = 0; b < kNear && bin < 0; ++b) {
                    if (want <= before + sums[b]) {
                        bin = near_lo + b;
                        need = want - before;
                    }
                    before += sums[b];
                }
            if (bin >= 0) {
                cut_in_bin(bin, s.cum[bin] - (bin ? s.cum[bin - 1] : 0), false, 0, need);
                settled = true;
            } else {
                near_lo = -1, near_hi = -2;                // somewhere else: all bins, below
                kept_ahead = 0;
                cluster.sync();
            }
        }
        if (!settled) {
            // exact weights of every bin of what is kept so far
            Buckets b{s.work, s.work + kBins};
            b.clear();
            const int walk = sparse >= 0 ? sparse : p.slice;
            for (int j = tid; j < walk; j += kThreads) {
                const float x = value(sparse >= 0 ? left[j] : j);
                // ties at a top-k cut: only cut_ties of them count, all of one weight and bin
                if (k_on && key_of(x) <= cut_key) continue;
                const int bin = bin_of(x);
                const u64 w = bin < kBins - 1 ? weight(x) : 0;
                if (w != 0) b.add(bin, w);
            }
            cluster.sync();
            u64 wb[2] = {0, 0};
#pragma unroll 4
            for (int r = 0; r < ctas; ++r) {
                const uint32_t* rl = cluster.map_shared_rank(b.lo, r);
                const uint2 l = reinterpret_cast<const uint2*>(rl)[tid];
                const uint2 h = reinterpret_cast<const uint2*>(rl + kBins)[tid];
                wb[0] += (static_cast<u64>(h.x) << 32) + l.x;
                wb[1] += (static_cast<u64>(h.y) << 32) + l.y;
            }
            if (k_on) {
                const u64 tie_w = weight(value_of(cut_key));
                const int bin = bin_of(value_of(cut_key));
                if (bin >> 1 == tid && bin < kBins - 1) (bin & 1 ? wb[1] : wb[0]) += tie_w * cut_ties;
            }
            u64 total;
            u64 before = block_inclusive(wb[0] + wb[1], s.scan, &total) - wb[0] - wb[1];
            const double want_d = ceil(static_cast<double>(share) * static_cast<double>(total));
            u64 want = want_d > 1.0 ? static_cast<u64>(want_d) : 1ull;
            if (want > total) want = total;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                if (before < want && before + wb[e] >= want) {
                    s.found = 2 * tid + e;
                    s.bin_above = before;
                }
                before += wb[e];
            }
            __syncthreads();
            const int bin = s.found;
            const u64 need = want - s.bin_above;
            cluster.sync();                               // the per-bin weights are read
            cut_in_bin(bin, s.cum[bin] - (bin ? s.cum[bin - 1] : 0), false, 0, need);
        }
    }

    // ---- cumulative weights in index order.  Tokens at the cut (of one weight) are counted
    // apart, so that one exchange tells both how many of them a CTA keeps and what it holds.
    const bool cut = cut_ties != 0xffffffffu;
    u64 tie_w = cut ? weight(value_of(cut_key)) : 0;
    if (tie_w < least_w) tie_w = 0;
    auto kept = [&](float x, u64 w, int& ties) {
        const uint32_t key = key_of(x);
        const bool tie = cut && key == cut_key;
        ties += tie;
        return key >= cut_key && w >= least_w && !tie ? w : 0ull;
    };
    // a warp's part: vectors of the slice, or listed tokens
    const int part = (sparse + kWarps - 1) / kWarps;
    const int from = sparse >= 0 ? min(warp * part, sparse) : first_vec;
    const int to = sparse >= 0 ? min(from + part, sparse) : last_vec;
    u64 sum = kept_ahead;
    int ties = 0;
    auto weigh = [&](int v, u64& sum, int& ties) {        // a vector, or a listed token
        if (sparse >= 0) {
            const float x = value(left[v]);
            sum += kept(x, weight(x), ties);
        } else {
            const uint4 q = xv[v];
            const T* e = reinterpret_cast<const T*>(&q);
#pragma unroll
            for (int k = 0; k < kVec; ++k) sum += kept(to_float(e[k]), weight(to_float(e[k])), ties);
        }
    };
    for (int v = from + lane; v < to; v += 32) {
        if (near_lo < 0) {
            weigh(v, sum, ties);
        } else {                                          // few are left to weigh
            const uint4 q = xv[v];
            const T* e = reinterpret_cast<const T*>(&q);
#pragma unroll
            for (int k = 0; k < kVec; ++k) {
                const float x = to_float(e[k]);
                const float z = place_of(x);
                if (z >= static_cast<float>(near_lo) && z < static_cast<float>(near_hi + 1))
                    sum += kept(x, weight(x), ties);
            }
        }
    }
    sum = warp_sum(sum);
    ties = warp_sum(ties);
    if (lane == 0) {
        s.warp_sum[warp] = sum;
        s.warp_ties[warp] = ties;
    }
    __syncthreads();
    if (tid == 0) {
        sum = 0;
        ties = 0;
        for (int w = 0; w < kWarps; ++w) {
            sum += s.warp_sum[w];
            ties += s.warp_ties[w];
        }
        s.sum = sum;
        s.ties = ties;
    }
    cluster.sync();
    // kept weight of what comes before a place with `sum` of weights and `ties` at the cut
    auto with_ties = [&](u64 sum, u64 ties) { return sum + (ties < cut_ties ? ties : cut_ties) * tie_w; };
    u64 before = 0, ties_before = 0, total;
    {
        u64 o[kMaxCtas], all_sum = 0, all_ties = 0;
        uint32_t o_ties[kMaxCtas];
        read_ranks(cluster, &s.sum, ctas, o);
        read_ranks(cluster, &s.ties, ctas, o_ties);
#pragma unroll
        for (int r = 0; r < kMaxCtas; ++r) {
            if (r < rank) {
                before += o[r];
                ties_before += o_ties[r];
            }
            all_sum += o[r];
            all_ties += o_ties[r];
        }
        total = with_ties(all_sum, all_ties);
    }
    const u64 want = target_of(total);
    for (int w = 0; w < warp; ++w) {
        before += s.warp_sum[w];
        ties_before += s.warp_ties[w];
    }
    if (with_ties(before, ties_before) <= want &&
        want < with_ties(before + s.warp_sum[warp], ties_before + s.warp_ties[warp])) {
        // the token is in this warp's part: 32 vectors (listed tokens) at a time
        for (int v0 = from; v0 < to; v0 += 32) {
            const int v = v0 + lane;
            u64 mine = 0;
            int mine_ties = 0;
            if (v < to) weigh(v, mine, mine_ties);
            u64 inc = mine;
            int inc_ties = mine_ties;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const u64 o = __shfl_up_sync(0xffffffffu, inc, d);
                const int t = __shfl_up_sync(0xffffffffu, inc_ties, d);
                if (lane >= d) {
                    inc += o;
                    inc_ties += t;
                }
            }
            u64 at = before + inc - mine, at_ties = ties_before + inc_ties - mine_ties;
            if (with_ties(at, at_ties) <= want && want < with_ties(before + inc, ties_before + inc_ties)) {
                int i = sparse >= 0 ? static_cast<int>(left[v]) : v * kVec;
                if (sparse < 0)
                    for (;; ++i) {                        // one of the vector's tokens
                        int tie = 0;
                        const float x = value(i);
                        at += kept(x, weight(x), tie);
                        at_ties += tie;
                        if (want < with_ties(at, at_ties) || i + 1 == (v + 1) * kVec) break;
                    }
                p.tokens[row] = base + i;
            }
            before += __shfl_sync(0xffffffffu, inc, 31);
            ties_before += __shfl_sync(0xffffffffu, inc_ties, 31);
            if (with_ties(before, ties_before) > want) break;
        }
    }
    cluster.sync();
}

template <typename T, int RESIDENT>
cudaError_t launch(const SampleParams& p, int ctas, cudaStream_t st) {
    static SmemLimit limit;
    const size_t smem = sizeof(Shared) + (static_cast<size_t>(p.slice) * sizeof(T) + 15) / 16 * 16;
    cudaError_t e = limit.ensure(sample_kernel<T, RESIDENT>, smem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(p.B) * ctas);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_allowed() ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, sample_kernel<T, RESIDENT>, p);
}

template <typename T>
cudaError_t launch(SampleParams p, int ctas, cudaStream_t st) {
    const long all = static_cast<long>(p.B) * ctas;
    if (all <= sm_count()) return launch<T, 1>(p, ctas, st);
    // with settings that differ, more CTAs than places, and a thread for each row to sort them
    // (64 rows of 151936, mixed: 50 us against 54)
    p.by_length = (p.temperature != nullptr || p.top_k != nullptr) && all > 2 * sm_count() && p.B <= kThreads;
    return launch<T, 2>(p, ctas, st);
}

}  // namespace

int sample_max_vocab(int type) {
    const int bytes = 227 * 1024 - static_cast<int>(sizeof(Shared)) - 16;
    return 8 * (bytes / (type == kF32 ? 4 : 2) / 8 * 8);
}

cudaError_t launch_sample(const SampleParams& p0, int type, cudaStream_t st) {
    SampleParams p = p0;
    const int size = type == kF32 ? 4 : 2;
    // CTAs per row: eight share a long row's latency; a slice below a few thousand tokens is
    // not worth another CTA
    int ctas = 1;
    while (ctas < 8 && (p.V + ctas - 1) / ctas > 4096) ctas *= 2;
    p.slice = ((p.V + ctas - 1) / ctas + 16 / size - 1) / (16 / size) * (16 / size);
    if (type == kF16) return launch<__half>(p, ctas, st);
    if (type == kBF16) return launch<__nv_bfloat16>(p, ctas, st);
    return launch<float>(p, ctas, st);
}

}  // namespace escha
