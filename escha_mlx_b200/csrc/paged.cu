// Page plans and stores of the paged key-value cache.
//
// Plan.  With page size P, request b holds have_b = ceil(len_b / P) pages and needs
// then_b = ceil((len_b + new_b) / P) after the step.  Rows of the step are packed by request
// (first_b = exclusive prefix of new), missing pages are taken from the free list in request
// order (before_b = exclusive prefix of then - have).  Everything follows from two prefix
// sums over the batch, so every CTA computes both for itself (a batch is a few KB, read from
// L2) and then writes its share of the rows and table entries: one launch, no wait between
// CTAs, no counters.  Bound by launch and load latency, not by its bytes.
//
// Store.  One thread per 8 elements of a row; a copy for 16-bit caches.  The 8-bit cache
// keeps, per token and head, scale = max|x| / 127 in 32 bits and the code nearest to
// x / scale: the D/8 threads of a row find the maximum by shuffles.  Bound by HBM.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <cstdlib>
#include <cstring>
#include <utility>

#include "common.cuh"
#include "decode_ops.h"

namespace escha {
namespace {

constexpr int kPlanThreads = 256;

// Exclusive prefix of one value per thread over the block, and the block's sum.
__device__ __forceinline__ long long block_exclusive(long long v, long long* total) {
    __shared__ long long sums[kPlanThreads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long inc = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const long long o = __shfl_up_sync(0xffffffffu, inc, d);
        if (lane >= d) inc += o;
    }
    __syncthreads();          // the previous use of sums is over
    if (lane == 31) sums[warp] = inc;
    __syncthreads();
    long long base = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kPlanThreads / 32; ++w) {
        if (w < warp) base += sums[w];
        all += sums[w];
    }
    *total = all;
    return base + inc - v;
}

// Last index b in [0, n) with prefix[b] <= x (prefix[0] == 0 <= x).
__device__ __forceinline__ int owner_of(const int* prefix, int n, int x) {
    int lo = 0, hi = n;       // prefix[lo] <= x, prefix[hi] > x or hi == n
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (prefix[mid] <= x) lo = mid; else hi = mid;
    }
    return lo;
}

struct Request {
    long long len, add;
    int have, need;
    bool valid;
};
__device__ __forceinline__ Request request(const PlanParams& p, int b, long long first) {
    Request r;
    r.len = p.lengths[b];
    r.add = p.added[b];
    const long long most = static_cast<long long>(p.W) << p.log_page;
    r.valid = r.len >= 0 && r.add >= 0 && r.len + r.add <= most && first + r.add <= p.rows;
    const long long up = (1ll << p.log_page) - 1;
    r.have = r.valid ? static_cast<int>((r.len + up) >> p.log_page) : 0;
    r.need = r.valid ? static_cast<int>((r.len + r.add + up) >> p.log_page) - r.have : 0;
    return r;
}

__global__ void __launch_bounds__(kPlanThreads) page_plan_kernel(const PlanParams p) {
    __shared__ int s_first[kPlanMaxBatch];    // first row of a request
    __shared__ int s_before[kPlanMaxBatch];   // pages taken before it
    grid_launch_dependents();
    grid_dependency_wait();
    const int tid = threadIdx.x;
    const int each = (p.B + kPlanThreads - 1) / kPlanThreads;
    const int lo = min(tid * each, p.B), hi = min(lo + each, p.B);
    const bool writes = blockIdx.x == 0;

    long long sum = 0, rows_in;
    for (int b = lo; b < hi; ++b) sum += max(p.added[b], 0);
    long long at = block_exclusive(sum, &rows_in);
    const long long first0 = at;
    long long need = 0, pages_in;
    for (int b = lo; b < hi; ++b) {
        s_first[b] = static_cast<int>(min(at, 0x7fffffffll));
        if (writes) p.starts[b] = s_first[b];
        need += request(p, b, at).need;
        at += max(p.added[b], 0);
    }
    long long before = block_exclusive(need, &pages_in);
    // the list from head on; a head outside the list leaves nothing to take
    const int head = *p.head;
    const long long avail = head >= 0 && head <= p.F ? p.F - head : 0;
    long long took = 0, refused = 0;
    at = first0;
    for (int b = lo; b < hi; ++b) {
        const Request r = request(p, b, at);
        s_before[b] = static_cast<int>(before);
        const bool fine = r.valid && (r.need == 0 || before + r.need <= avail);
        took += fine ? r.need : 0;
        refused += !fine;
        if (writes) {
            const long long most = static_cast<long long>(p.W) << p.log_page;
            p.ends[b] = static_cast<int>(fine ? r.len + r.add : min(max(r.len, 0ll), most));
        }
        before += r.need;
        at += max(p.added[b], 0);
    }
    long long all_took, all_refused;
    block_exclusive(took, &all_took);
    block_exclusive(refused, &all_refused);      // its barriers also publish s_first, s_before
    if (writes && tid == 0) {
        p.starts[p.B] = static_cast<int>(min(rows_in, 0x7fffffffll));
        *p.head_out = head + static_cast<int>(all_took);
        *p.refused = static_cast<int>(all_refused);
    }
    const int step = gridDim.x * kPlanThreads, me = blockIdx.x * kPlanThreads + tid;
    // Requests are served in order until the list ends, so the pages taken are the first
    // all_took of the prefix: page i belongs to the request whose range holds it.
    for (int i = me; i < all_took; i += step) {
        const int b = owner_of(s_before, p.B, i);
        const Request r = request(p, b, s_first[b]);
        p.table[static_cast<size_t>(b) * p.W + r.have + (i - s_before[b])] = p.free_pages[head + i];
    }
    for (int row = me; row < p.rows; row += step) {
        int slot = -1, pos = 0;
        if (row < rows_in) {
            const int b = owner_of(s_first, p.B, row);
            const Request r = request(p, b, s_first[b]);
            if (r.valid && (r.need == 0 || s_before[b] + static_cast<long long>(r.need) <= avail)) {
                pos = static_cast<int>(r.len) + row - s_first[b];
                const int idx = pos >> p.log_page;
                // pages that the request already held are in its table; the others are read
                // from the list, since another CTA may be writing their entries now
                const int page = idx < r.have ? p.table[static_cast<size_t>(b) * p.W + idx]
                                              : p.free_pages[head + s_before[b] + idx - r.have];
                if (page >= 0 && page < p.n_pages)
                    slot = (page << p.log_page) + (pos & ((1 << p.log_page) - 1));
            }
        }
        p.slots[row] = slot;
        p.positions[row] = pos;
    }
}

template <typename T> struct Pair;
template <> struct Pair<__half> {
    static __device__ float2 f32(uint32_t w) {
        return __half22float2(*reinterpret_cast<const __half2*>(&w));
    }
};
template <> struct Pair<__nv_bfloat16> {
    static __device__ float2 f32(uint32_t w) {
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    }
};

// The code nearest to x / scale, ties to even, from a guess that is off by one at most.  Whether
// x lies above the middle between two codes is the sign of x - (c +- 1/2) scale, which one fused
// multiply-add gives exactly (a rounded quotient can land on the wrong side); `times` 2 keeps
// the half of a denormal scale.  Adding 1.5 * 2^23 rounds to an integer and leaves it in the low
// bits.
__device__ __forceinline__ uint32_t code_of(float x, float scale, float guess, float times) {
    const float shifted = guess + 12582912.0f, c = shifted - 12582912.0f;
    const int bits = __float_as_int(shifted);
    const bool odd = bits & 1;
    const float above = __fmaf_rn(-times * (c + 0.5f), scale, times * x);
    const float below = __fmaf_rn(-times * (c - 0.5f), scale, times * x);
    const int up = above > 0.0f || (odd && above == 0.0f), down = below < 0.0f || (odd && below == 0.0f);
    return static_cast<uint32_t>(min(max(((bits << 8) >> 8) - 0x400000 + up - down, -127), 127)) & 0xffu;
}

constexpr int kAppendThreads = 256;
// Items of a thread in flight: slots, then rows, then stores.  One at a time: 25.0 us for 131 MB
// (16001 rows of 8 heads of 128, scattered slots), two 22.9 (5.7 TB/s), four 23.9.
constexpr int kAppendBatch = 2;

// T: type of the rows; Q: 8-bit cache.  Item = 8 elements of one row of one head of k or v;
// fewer than 2^31 of them.
template <typename T, bool Q>
__global__ void __launch_bounds__(kAppendThreads)
paged_append_kernel(const AppendParams p, int log_d8) {
    grid_launch_dependents();
    grid_dependency_wait();
    const unsigned d8 = 1u << log_d8;                     // items per row of a head: 8, 16 or 32
    const unsigned items = 2u * p.T * p.H * d8;           // [T][k, v][H][D / 8]
    const unsigned step = gridDim.x * kAppendThreads;
    const unsigned lane = threadIdx.x & 31;
    // every thread of a warp runs the same rounds (items are whole rows of 8..32 threads and
    // a warp's first item is a multiple of 32), so the shuffles below always meet
    for (unsigned i0 = blockIdx.x * kAppendThreads + (threadIdx.x & ~31u); i0 < items;
         i0 += kAppendBatch * step) {
        int slot[kAppendBatch];
        unsigned row[kAppendBatch], head[kAppendBatch];
        bool is_v[kAppendBatch];
#pragma unroll
        for (int j = 0; j < kAppendBatch; ++j) {
            const unsigned i = i0 + j * step + lane;
            const unsigned hh = i >> log_d8, tv = hh / p.H;   // [T][k, v][H], [T][k, v]
            head[j] = hh - tv * p.H;
            is_v[j] = tv & 1;
            row[j] = tv >> 1;
            slot[j] = i < items ? p.slots[row[j]] : -1;
            if (slot[j] < 0 || (slot[j] >> p.log_page) >= p.n_pages) slot[j] = -1;
        }
        const unsigned d = lane & (d8 - 1);               // steps are multiples of 32
        uint4 x[kAppendBatch];
#pragma unroll
        for (int j = 0; j < kAppendBatch; ++j) {
            x[j] = make_uint4(0, 0, 0, 0);
            if (slot[j] >= 0) {
                const T* src = is_v[j] ? static_cast<const T*>(p.v) + row[j] * p.v_row + head[j] * p.v_head
                                       : static_cast<const T*>(p.k) + row[j] * p.k_row + head[j] * p.k_head;
                x[j] = *reinterpret_cast<const uint4*>(src + d * 8);
            }
        }
#pragma unroll
        for (int j = 0; j < kAppendBatch; ++j) {
            if (i0 + j * step >= items) break;            // the same for the whole warp
            const long page = slot[j] >> p.log_page;
            const long at = ((page * p.H + head[j]) << p.log_page) + (slot[j] & ((1 << p.log_page) - 1));
            if constexpr (!Q) {
                if (slot[j] >= 0) {
                    T* dst = static_cast<T*>(is_v[j] ? p.v_cache : p.k_cache) + at * p.D + d * 8;
                    *reinterpret_cast<uint4*>(dst) = x[j];
                }
            } else {
                const uint32_t w[4] = {x[j].x, x[j].y, x[j].z, x[j].w};
                float f[8];
                float top = 0.0f, nothing = 0.0f;         // NaN if a value is not finite
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float2 y = Pair<T>::f32(w[k]);
                    f[2 * k] = y.x;
                    f[2 * k + 1] = y.y;
                }
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    top = fmaxf(top, fabsf(f[k]));
                    nothing = fmaf(f[k], 0.0f, nothing);
                }
                if (!(nothing == 0.0f)) top = __int_as_float(0x7f800000);
                for (unsigned o = d8 >> 1; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                // a row that is not finite is stored as NaN: its values have no scale
                const bool finite = top <= 3.4e38f;
                const float scale = finite ? __fdiv_rn(top, 127.0f) : __int_as_float(0x7fc00000);
                if (slot[j] >= 0) {
                    uint32_t c[2] = {0, 0};
                    if (finite && scale > 1e-36f) {
                        const float by = __frcp_rn(scale);
                        float edge = 0.0f;                // how near to a middle the quotients come
                        uint32_t b[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const float t = f[k] * by, shifted = t + 12582912.0f;
                            edge = fmaxf(edge, fabsf(t - (shifted - 12582912.0f)));
                            b[k] = __float_as_uint(shifted);
                        }
                        // t is good to 2e-5: nearer than that, the exact comparison
                        if (edge > 0.4999f)
#pragma unroll
                            for (int k = 0; k < 8; ++k) b[k] = code_of(f[k], scale, f[k] * by, 1.0f);
#pragma unroll
                        for (int k = 0; k < 2; ++k)
                            c[k] = __byte_perm(__byte_perm(b[4 * k], b[4 * k + 1], 0x0040),
                                               __byte_perm(b[4 * k + 2], b[4 * k + 3], 0x0040), 0x5410);
                    } else if (finite && scale > 0.0f) {          // its reciprocal may not exist
                        for (int k = 0; k < 8; ++k)
                            c[k >> 2] |= code_of(f[k], scale, __fdiv_rn(f[k], scale), 2.0f) << (8 * (k & 3));
                    }
                    int8_t* dst = static_cast<int8_t*>(is_v[j] ? p.v_cache : p.k_cache) + at * p.D + d * 8;
                    *reinterpret_cast<uint2*>(dst) = make_uint2(c[0], c[1]);
                    if (d == 0) (is_v[j] ? p.v_scale : p.k_scale)[at] = scale;
                }
            }
        }
    }
}

}  // namespace

int sm_count() {
    static std::atomic<int> known[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    int sms = known[dev].load(std::memory_order_relaxed);
    if (sms == 0) {
        if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
        known[dev].store(sms, std::memory_order_relaxed);
    }
    return sms;
}

cudaError_t launch_page_plan(const PlanParams& p, cudaStream_t st) {
    const int most = (p.rows + kPlanThreads - 1) / kPlanThreads;
    const int grid = most < 1 ? 1 : most > sm_count() ? sm_count() : most;
    return launch_chained(page_plan_kernel, dim3(grid), dim3(kPlanThreads), 0, st, p);
}

cudaError_t launch_paged_append(const AppendParams& all, int in_type, int cache_type, cudaStream_t st) {
    AppendParams p = all;
    const int log_d8 = p.D == 64 ? 3 : p.D == 128 ? 4 : 5;
    // a launch numbers its items in 32 bits: more rows take several
    const long per_row = 2l * p.H << log_d8;
    const long most_rows = 0x7f000000l / per_row;
    for (long r = 0; r < all.T; r += most_rows) {
        p.T = static_cast<int>(all.T - r < most_rows ? all.T - r : most_rows);
        p.k = static_cast<const char*>(all.k) + 2 * r * p.k_row;
        p.v = static_cast<const char*>(all.v) + 2 * r * p.v_row;
        p.slots = all.slots + r;
        const long most = (per_row * p.T + kAppendThreads - 1) / kAppendThreads;
        const long cap = 8l * sm_count();
        const dim3 grid(static_cast<unsigned>(most < cap ? most : cap));
        // the type of a 16-bit copy does not matter
        const auto kernel = cache_type != kI8 ? paged_append_kernel<__half, false>
                            : in_type == kF16 ? paged_append_kernel<__half, true>
                                              : paged_append_kernel<__nv_bfloat16, true>;
        const cudaError_t e = launch_chained(kernel, grid, dim3(kAppendThreads), 0, st, p, log_d8);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

}  // namespace escha
