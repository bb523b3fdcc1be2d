// Attention of one new token per request over the paged key-value cache.
//
//   S = scale * q K^T over the request's tokens,  P = softmax(S),  O = P V
//
// per query head; the `group` query heads of a key/value head read the same K and V, so they
// are the columns of one product and the cache is read once.  Bound by reading the cache from
// HBM: at 8 query heads a byte of it meets 8 multiply-adds, far below what even mma.sync
// offers, and a token block of 16 x 8 heads is no tile for tcgen05 (128 rows at least).
//
// Layout.  Both products are computed transposed, S^T = K q^T and O^T = V^T P^T, so that the
// cache is the A operand (16 tokens, resp. 16 channels, per mma.m16n8k16) and the heads are
// the 8 columns.  The order of the summed index is free, so lane (g, t) = (lane / 4, lane % 4)
// takes 16 contiguous bytes of token rows g and g + 8 for the first product, and contiguous
// bytes of token rows 2t, 2t + 1, 2t + 8, 2t + 9 for the second, whose pairs along the tokens
// are put together by byte permutes.  Each warp has a ring of its own (keys, values,
// keys, ... of 16 to 64 tokens) that it fills with cp.async, 512 contiguous bytes of the cache
// per instruction: fetching each lane's own operand bytes instead (64-byte runs) needed no
// exchange between lanes but ran at 4.9 TB/s against 6.8.  The 16-byte pieces of a tile are
// stored with an exclusive-or swizzle under which the fill and both operand reads are free of
// bank conflicts.  Rows past a request's end are zero-filled, never read.
//
// Softmax.  Scores are held in 32 bits, times log2(e); a running maximum per head, sums in
// 32 bits per lane until the end.  P is rounded to 16 bits for the product, as a pair hi + lo
// of them, so that this rounding stays below that of the output; with binary16 P is scaled by
// 2^13 against underflow of the many small weights of a long context.  The 8-bit cache holds
// codes, exact in binary16; K's scale multiplies the score, V's the weight (the running
// maximum then includes V's exponent, so that the weights stay in range).
//
// Split.  The work is a line of blocks of 64 tokens, over all requests and key/value heads;
// each CTA takes an equal share of it, whatever the lengths are, and cuts rows where its share
// ends.  Every row counts for some blocks more than it has (the exchange between its warps and
// its first loads), so that a CTA with many short rows is not the last.  A CTA leaves at most two unfinished rows (its first and its last); a second, chained
// kernel joins the pieces of each row in order.  No counters, nothing to clear.  Where all rows
// fit the GPU at once and none can be long, a row is cut between the CTAs of a cluster instead,
// which join through distributed shared memory: one launch and no scratch.
#pragma once

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdlib>
#include <cstring>
#include <utility>

#include "common.cuh"
#include "decode_ops.h"
#include "kernels.h"

namespace escha {
namespace attend {

namespace cg = cooperative_groups;

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;

// A lane's copy of N bytes, completed by cp.async.wait_group; bytes past `have` are zeros.
template <int N>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, int have) {
    if constexpr (N == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(have) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(dst), "l"(src), "r"(have), "n"(N) : "memory");
}
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
template <bool BF>
__device__ __forceinline__ void mma(float d[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                    uint32_t b0, uint32_t b1) {
    if constexpr (!BF) {
        mma16816(d, a0, a1, a2, a3, b0, b1);
    } else {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
            "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
}
template <bool BF>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (!BF) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}
template <bool BF>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
    if constexpr (!BF) return __half22float2(*reinterpret_cast<const __half2*>(&w));
    else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
// Codes of an 8-bit word, offset to 0..255: byte pairs (0, 1) or (2, 3) as binary16.  0x6400 | u
// is 1024 + u; minus 1152 is the code, exactly.
template <int SEL>
__device__ __forceinline__ uint32_t codes_f16(uint32_t offset_word) {
    const uint32_t x = __byte_perm(offset_word, 0x64646464u, SEL);
    const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&x), __float2half2_rn(1152.0f));
    return *reinterpret_cast<const uint32_t*>(&y);
}
// Place in a tile of byte `byte` of token row r.  Reads of 128 bits run in groups of eight
// lanes: two rows 2i, 2i + 1 of 64 bytes (keys), or rows 2t + c, t = 0..3, of 32 bytes
// (values); the bits exclusive-ored in tell those rows apart.  Rows of 64 bytes share a line.
template <int ROW>
__device__ __forceinline__ int place(int r, int byte) {
    if constexpr (ROW >= 128) {
        return r * ROW + (byte ^ (((r >> 1 & 3) ^ (r & 1) << 1) << 5));
    } else {
        return (r >> 1) * 128 + (((r & 1) * 64 + byte) ^ ((r >> 1 & 3) << 5));
    }
}
template <int BYTES> struct Words;
template <> struct Words<16> { uint4 v; __device__ uint32_t operator[](int i) const { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; } };
template <> struct Words<8> { uint2 v; __device__ uint32_t operator[](int i) const { return i == 0 ? v.x : v.y; } };
template <> struct Words<4> { uint32_t v; __device__ uint32_t operator[](int) const { return v; } };

// QBF: queries and output are bfloat16.  I8: 8-bit cache.  D: channels of a head.
// NT: groups of 8 query heads.
template <bool QBF, bool I8, int D, int NT>
struct Shape {
    static constexpr bool kBF = QBF && !I8;               // type of the products
    static constexpr int kResident = 2;                   // CTAs that share an SM
    static constexpr int kElem = I8 ? 1 : 2;
    static constexpr int kRow = D * kElem;                // bytes of a token's row
    static constexpr int kChunks = kRow / 64;             // 64-byte pieces of a row
    // A warp's step takes kSubs tiles of 16 tokens: with short rows the softmax around a single
    // one (exchanges, votes) would take longer than its bytes.
    static constexpr int kSubs = NT == 2 ? (kRow <= 128 ? 2 : 1) : kRow >= 512 ? 1 : kRow == 256 ? 2 : 4;
    static constexpr int kTile = 16 * kSubs;
    static constexpr int kHalf = kTile * kRow;            // bytes of a step's keys or values
    static constexpr int kSets = kRow == 512 ? 2 : 1;     // value rows as 16 pieces per set
    static constexpr int kPiece = kRow / kSets / 16;      // bytes of a piece: 16, 8 or 4
    static constexpr int kPerPiece = kPiece / kElem;      // channels of a piece
    static constexpr int kMma = kSets * kPerPiece;        // O^T tiles of 16 channels
    static constexpr int kScales = I8 ? 2 * kTile * 4 : 0;   // bytes of a step's scales in the ring
    static constexpr int kQWords = I8 ? 8 : 4;            // query words per lane and chunk
    static constexpr int kQBytes = NT * kChunks * kQWords * 4 * 32;
    static constexpr int kRingStage = kHalf + kScales;
    static constexpr int kHeads = 8 * NT;
    static constexpr int kFixed = (kAttendMaxBatch + 4) * 4 + 2 * kWarps * kHeads * 4 + kHeads * 4 + 64;
    // depth of a warp's ring: what the CTAs that share an SM leave
    static constexpr int kJoin = kWarps * kHeads * (D + 4) * 4;   // the warps' sums
    static constexpr bool kAhead = kJoin - kWarps * kRingStage <= 2048;
    static constexpr int kMost = (226 * 1024 / kResident - 1024 - kFixed - kQBytes - (kAhead ? 2048 : 0)) /
                                 (kWarps * kRingStage);
    static constexpr int kStages = kMost > 8 ? 8 : kMost;
    static_assert(kStages >= 3, "a step's keys and values in flight beside what is in use");
    // The warps' sums lie over the ring's stage 0 (with a little room behind it), so that a
    // segment's first tiles can be fetched into the other stages before the one before it is
    // joined; over the whole ring where they are much larger.
    static constexpr int kAll = kWarps * kRingStage;      // a stage of all warps
    static constexpr int kGap = kJoin > kAll ? kJoin - kAll : 0;
    static constexpr int kRing = kStages * kAll;
    static constexpr int kBody = kAhead ? kRing + kGap : kRing > kJoin ? kRing : kJoin;
    static constexpr int kFirst = kAhead ? 1 : 0;
    static __device__ constexpr int stage_at(int stage) { return stage * kAll + (kAhead && stage ? kGap : 0); }
    static constexpr int kShared = kBody + kQBytes + kFixed;
};

// Exclusive prefix of the requests' blocks and row costs in s_prefix[0 .. B], by the whole CTA.
__device__ __forceinline__ void block_counts(const AttendParams& p, int* s_prefix, int* s_sums) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int kEach = kAttendMaxBatch / kThreads;
    const int most = p.W << p.log_page;
    int n[kEach], sum = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int b = tid * kEach + i;
        const int len = b < p.B ? min(max(p.lengths[b], 0), most) : 0;
        n[i] = len > 0 ? (len + kAttendBlock - 1) / kAttendBlock + p.row_cost : 0;
        sum += n[i];
    }
    int inc = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, inc, d);
        if (lane >= d) inc += o;
    }
    if (lane == 31) s_sums[warp] = inc;
    __syncthreads();
    int at = inc - sum;
    for (int w = 0; w < warp; ++w) at += s_sums[w];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int b = tid * kEach + i;
        if (b <= p.B) s_prefix[b] = at;
        at += n[i];
    }
    if (tid == kThreads - 1 && p.B == kAttendMaxBatch) s_prefix[p.B] = at;
    __syncthreads();
}

// CL: a row per cluster of p.ctas CTAs; otherwise equal shares of all blocks, p.ctas of them.
template <bool QBF, bool I8, int D, int NT, bool CL>
__global__ void __launch_bounds__(kThreads, Shape<QBF, I8, D, NT>::kResident) attend_kernel(const AttendParams p) {
    using S = Shape<QBF, I8, D, NT>;
    constexpr bool BF = S::kBF;
    // power of two on the weights (binary16 products only)
    constexpr float kLift = BF ? 0.0f : 13.0f;
    extern __shared__ __align__(16) uint8_t smem[];
    uint8_t* s_body = smem;
    uint32_t* s_q = reinterpret_cast<uint32_t*>(smem + S::kBody);
    int* s_prefix = reinterpret_cast<int*>(smem + S::kBody + S::kQBytes);
    float* s_m = reinterpret_cast<float*>(s_prefix + kAttendMaxBatch + 4);
    float* s_l = s_m + kWarps * S::kHeads;
    float* s_qscale = s_l + kWarps * S::kHeads;
    int* s_sums = reinterpret_cast<int*>(s_qscale + S::kHeads);
    float* s_part = reinterpret_cast<float*>(s_prefix);   // CL: maximum and sum by head

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t = lane & 3;
    grid_launch_dependents();
    grid_dependency_wait();
    if constexpr (!CL) block_counts(p, s_prefix, s_sums);

    const int per_request = p.H * p.chunks;               // rows of a request
    const int c = blockIdx.x;
    using QT = typename std::conditional<QBF, __nv_bfloat16, __half>::type;
    const QT* q = static_cast<const QT*>(p.q);
    QT* out = static_cast<QT*>(p.out);
    const int heads_total = p.H * p.group;
    long long total = 0, shares = 0, u = 0, u_end = 1;
    if constexpr (!CL) {
        total = static_cast<long long>(s_prefix[p.B]) * per_request;
        // As many CTAs as there are blocks at most, so that no share is empty, and no more than
        // the largest share asks for: fewer pieces to join (one request of 9000 tokens, 2 heads of
        // 256: 15.5 us against 19.0; no difference with many blocks per CTA).
        shares = min(static_cast<long long>(p.ctas), total);
        if (shares > 0) {
            const long long most = (total + shares - 1) / shares;
            shares = (total + most - 1) / most;
        }
        u = c < shares ? total * c / shares : 0;
        u_end = c < shares ? total * (c + 1) / shares : 0;
        // requests without a token: zeros
        for (int b = c; b < p.B; b += p.ctas)
            if (s_prefix[b + 1] == s_prefix[b])
                for (int i = tid; i < heads_total * D / 8; i += kThreads)
                    reinterpret_cast<uint4*>(out + static_cast<size_t>(b) * heads_total * D)[i] =
                        make_uint4(0, 0, 0, 0);
    }
    int unfinished_row = -1, unfinished_last = -1;

    const uint32_t ring = smem_u32(s_body) + warp * S::kRingStage;
    const uint8_t* ring_ptr = s_body + warp * S::kRingStage;
    const uint8_t* kc = static_cast<const uint8_t*>(p.k_cache);
    const uint8_t* vc = static_cast<const uint8_t*>(p.v_cache);

    // A segment: blocks [k0, k1) of a row (rr: its head and chunk) of request b.
    // used: what of the line it takes up.
    struct Segment { int b, rr, k0, k1, blocks, used; };
    auto segment_at = [&](long long u) {
        Segment x;
        if constexpr (CL) {
            const int row = c / p.ctas, part = c - row * p.ctas;
            x.b = row / per_request;
            x.rr = row - x.b * per_request;
            x.blocks = (min(max(p.lengths[x.b], 0), p.W << p.log_page) + kAttendBlock - 1) / kAttendBlock;
            x.k0 = x.blocks * part / p.ctas;
            x.k1 = x.blocks * (part + 1) / p.ctas;
            x.used = 1;
        } else {
            // the row that holds block u
            int hi = p.B;
            x.b = 0;
            while (hi - x.b > 1) {
                const int mid = (x.b + hi) >> 1;
                if (static_cast<long long>(s_prefix[mid]) * per_request <= u) x.b = mid; else hi = mid;
            }
            const int units = s_prefix[x.b + 1] - s_prefix[x.b];      // the row's cost, then its blocks
            const int in_request = static_cast<int>(u - static_cast<long long>(s_prefix[x.b]) * per_request);
            x.rr = in_request / units;
            const int at = in_request - x.rr * units;
            x.used = static_cast<int>(min(static_cast<long long>(units - at), u_end - u));
            x.blocks = units - p.row_cost;
            x.k0 = max(at - p.row_cost, 0);
            x.k1 = max(at + x.used - p.row_cost, 0);
        }
        return x;
    };
    constexpr int kSubs = S::kSubs, kTile = S::kTile;
    Segment seg;
    int h, head0, nheads, t0, t1;                         // of the segment: heads and tokens
    int mine, halves;                                     // this warp's steps warp, warp + kWarps, ...
    const int32_t* pages;
    int ids;                                              // lane j: page of the 16 tokens j (mod 32)
    uint32_t bad;                                         // those (mod 32) without a usable page
    size_t rows[kSubs];                                   // cache rows of the step being fetched
    int have[kSubs];                                      // and its tokens, by 16
    bool full = false;                                    // whether all of them are there
    auto open = [&](const Segment& x) {
        seg = x;
        const int len = min(max(p.lengths[x.b], 0), p.W << p.log_page);
        h = x.rr / p.chunks;
        const int chunk = x.rr - h * p.chunks;
        head0 = h * p.group + chunk * S::kHeads;
        nheads = min(S::kHeads, p.group - chunk * S::kHeads);
        t0 = x.k0 * kAttendBlock;
        t1 = min(len, x.k1 * kAttendBlock);
        const int steps = (t1 - t0 + kTile - 1) / kTile;
        mine = steps > warp ? (steps - warp + kWarps - 1) / kWarps : 0;
        halves = 2 * mine;                                // K0, V0, K1, V1, ...
        pages = p.table + static_cast<size_t>(x.b) * p.W;
        ids = -1;
        bad = 0;
    };
    auto fetch_rows = [&](uint32_t dst, const uint8_t* cache) {
        if (full) {
#pragma unroll
            for (int x = 0; x < S::kHalf / 512; ++x) {
                constexpr int kRows = 512 / S::kRow;
                const int m = x * kRows / 16;
                copy_async(dst + place<S::kRow>(x * kRows + lane / (S::kRow / 16), lane % (S::kRow / 16) * 16),
                           cache + rows[m] * S::kRow + (x * 512 - m * 16 * S::kRow) + lane * 16);
            }
            return;
        }
#pragma unroll
        for (int x = 0; x < S::kHalf / 512; ++x) {
            constexpr int kRows = 512 / S::kRow;      // rows per instruction, of one 16
            const int m = x * kRows / 16;
            const int r = x * kRows % 16 + lane / (S::kRow / 16);
            const int byte = lane % (S::kRow / 16) * 16;
            const bool in = r < have[m];
            copy_async<16>(dst + place<S::kRow>(m * 16 + r, byte),
                           cache + rows[m] * S::kRow + (in ? r * S::kRow + byte : 0), in ? 16 : 0);
        }
    };
    auto fetch = [&](int i, int stage) {
        if (i < halves) {
            const int j = i >> 1;
            const uint32_t dst = ring + S::stage_at(stage);
            if ((i & 1) == 0) {
                if ((j * kSubs & 31) == 0) {
                    const int tok = t0 + kTile * (warp + kWarps * (j + lane / kSubs)) + lane % kSubs * 16;
                    ids = tok < t1 ? pages[tok >> p.log_page] : -1;
                }
                full = t1 - t0 - kTile * (warp + kWarps * j) >= kTile;
#pragma unroll
                for (int m = 0; m < kSubs; ++m) {
                    const int at = (j * kSubs + m) & 31;
                    const int page = __shfl_sync(0xffffffffu, ids, at);
                    const int tok = t0 + kTile * (warp + kWarps * j) + 16 * m;
                    const bool ok = page >= 0 && page < p.n_pages;
                    bad = (bad & ~(1u << at)) | (ok ? 0u : 1u << at);
                    full = full && ok;
                    have[m] = ok ? min(16, t1 - tok) : 0;
                    rows[m] = (((ok ? static_cast<size_t>(page) : 0) * p.H + h) << p.log_page) +
                              (tok & ((1 << p.log_page) - 1));
                    if constexpr (I8) {
                        // scales: lanes 0..15 K's, the others V's
                        const float* src = (lane < 16 ? p.k_scale : p.v_scale) + rows[m];
                        const bool in = (lane & 15) < have[m];
                        copy_async<4>(dst + S::kHalf + (m * 32 + lane) * 4, src + (in ? lane & 15 : 0),
                                      in ? 4 : 0);
                    }
                }
                fetch_rows(dst, kc);
            } else {
                fetch_rows(dst, vc);
            }
        }
        cp_async_commit();
    };
    // the first kStages - 1 tiles of a segment, from stage kFirst on
    auto prologue = [&]() {
        __syncwarp();                                 // the other lanes' last reads
#pragma unroll
        for (int i = 0; i < S::kStages - 1; ++i) fetch(i, (S::kFirst + i) % S::kStages);
    };
    // queries of the segment: lane (g, t) of chunk x holds head g's channels that meet the
    // lane's bytes of the key rows
    auto load_queries = [&]() {
        if (warp >= NT) return;
        const int nt = warp, b = seg.b;
        const bool in = nt * 8 + g < nheads;
        const QT* src = q + static_cast<long>(b) * p.q_row +
                        static_cast<long>(head0 + (in ? nt * 8 + g : 0)) * p.q_head;
        uint4 w[S::kChunks * S::kQWords / 4];
#pragma unroll
        for (int x = 0; x < S::kChunks * S::kQWords / 4; ++x) {
            // 16 channels (8-bit cache) are two loads of 8
            const int off = I8 ? (x >> 1) * 64 + t * 16 + (x & 1) * 8 : x * 32 + t * 8;
            w[x] = in ? *reinterpret_cast<const uint4*>(src + off) : make_uint4(0, 0, 0, 0);
        }
        float by = p.scale_log2;
        if constexpr (I8 && QBF) {
            // bfloat16 queries against codes in binary16: bring the row's largest value
            // to [2^14, 2^15) by a power of two, so that small ones beside it keep their bits
            float top = 0.0f;
#pragma unroll
            for (int x = 0; x < S::kChunks * S::kQWords / 4; ++x)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float2 f = unpack2<true>(k == 0 ? w[x].x : k == 1 ? w[x].y : k == 2 ? w[x].z : w[x].w);
                    top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
                }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int e = min(max((__float_as_int(top) >> 23) - 127, -100), 120);
            const float down = __int_as_float((127 + 14 - e) << 23);
            by *= __int_as_float((127 - 14 + e) << 23);
#pragma unroll
            for (int x = 0; x < S::kChunks * S::kQWords / 4; ++x) {
                uint32_t* v = &w[x].x;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float2 f = unpack2<true>(v[k]);
                    v[k] = pack2<false>(f.x * down, f.y * down);
                }
            }
        }
        if (t == 0) s_qscale[nt * 8 + g] = by;
#pragma unroll
        for (int x = 0; x < S::kChunks * S::kQWords / 4; ++x)
            reinterpret_cast<uint4*>(s_q)[(nt * (S::kChunks * S::kQWords / 4) + x) * 32 + lane] = w[x];
    };

    // the next segment with a block in it (a share may end within the cost of a row)
    auto next = [&]() {
        while (u < u_end) {
            const Segment x = segment_at(u);
            u += x.used;
            if (CL || x.k1 > x.k0) {
                open(x);
                return true;
            }
        }
        return false;
    };
    bool more = next();
    if (more) {
        prologue();
        load_queries();
        __syncthreads();
    }
    while (more) {
        float qs[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            qs[nt][0] = s_qscale[nt * 8 + 2 * t];
            qs[nt][1] = s_qscale[nt * 8 + 2 * t + 1];
        }

        float acc[NT][S::kMma][4];
        float m_run[NT][2], l[NT][2];                     // running maxima; sums by lane
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int k = 0; k < S::kMma; ++k)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[nt][k][e] = 0.0f;
            m_run[nt][0] = m_run[nt][1] = __int_as_float(0xff800000);
            l[nt][0] = l[nt][1] = 0.0f;
        }

        int rd = S::kFirst, wr = (S::kFirst + S::kStages - 1) % S::kStages;   // stages to read and to fill next
        for (int j = 0; j < mine; ++j) {
            // ---- scores of the step's tokens
            cp_async_wait<S::kStages - 2>();
            __syncwarp();         // the other lanes' copies; their reads of the stage to fill next
            const uint8_t* tile = ring_ptr + S::stage_at(rd);
            // two chains of products where the step has one tile only
            constexpr int kChains = kSubs == 1 ? 2 : 1;
            float s[NT][kSubs][kChains][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int m = 0; m < kSubs; ++m)
#pragma unroll
                    for (int e = 0; e < 4 * kChains; ++e) s[nt][m][e >> 2][e & 3] = 0.0f;
#pragma unroll
            for (int x = 0; x < S::kChunks; ++x) {
                constexpr int kPer = S::kQWords / 4;
                Words<16> qa[NT], qb[NT];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    qa[nt].v = reinterpret_cast<const uint4*>(s_q)[((nt * S::kChunks + x) * kPer) * 32 + lane];
                    if constexpr (I8)
                        qb[nt].v = reinterpret_cast<const uint4*>(s_q)[((nt * S::kChunks + x) * kPer + 1) * 32 + lane];
                }
#pragma unroll
                for (int m = 0; m < kSubs; ++m) {
                    Words<16> r0, r1;
                    r0.v = *reinterpret_cast<const uint4*>(tile + place<S::kRow>(m * 16 + g, x * 64 + t * 16));
                    r1.v = *reinterpret_cast<const uint4*>(tile + place<S::kRow>(m * 16 + g + 8, x * 64 + t * 16));
                    if constexpr (!I8) {
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            mma<BF>(s[nt][m][0], r0[0], r1[0], r0[1], r1[1], qa[nt][0], qa[nt][1]);
                            mma<BF>(s[nt][m][kChains - 1], r0[2], r1[2], r0[3], r1[3], qa[nt][2], qa[nt][3]);
                        }
                    } else {
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint32_t a = r0[k] ^ 0x80808080u, e = r1[k] ^ 0x80808080u;
                            const uint32_t a0 = codes_f16<0x4140>(a), a1 = codes_f16<0x4140>(e);
                            const uint32_t a2 = codes_f16<0x4342>(a), a3 = codes_f16<0x4342>(e);
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
                                mma<false>(s[nt][m][k & (kChains - 1)], a0, a1, a2, a3,
                                           k < 2 ? qa[nt][2 * k] : qb[nt][2 * k - 4],
                                           k < 2 ? qa[nt][2 * k + 1] : qb[nt][2 * k - 3]);
                        }
                    }
                }
            }
            // K's, then V's scales of tokens g, g + 8
            float4 sc[I8 ? kSubs : 1];
            if constexpr (I8) {
                const float* scales = reinterpret_cast<const float*>(tile + S::kHalf);
#pragma unroll
                for (int m = 0; m < kSubs; ++m)
                    sc[m] = make_float4(scales[m * 32 + g], scales[m * 32 + g + 8], scales[m * 32 + 16 + g],
                                        scales[m * 32 + 24 + g]);
            }
            fetch(2 * j + S::kStages - 1, wr);
            rd = rd + 1 == S::kStages ? 0 : rd + 1;
            wr = wr + 1 == S::kStages ? 0 : wr + 1;

            // ---- weights
            const int left = t1 - (t0 + kTile * (warp + kWarps * j));
            uint32_t hi0[NT][kSubs], hi1[NT][kSubs], lo0[NT][kSubs], lo1[NT][kSubs];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float x[kSubs][4], up[2];
                up[0] = up[1] = __int_as_float(0xff800000);
#pragma unroll
                for (int m = 0; m < kSubs; ++m) {
                    const int usable = (bad >> ((j * kSubs + m) & 31)) & 1 ? 0 : left - 16 * m;
                    float above[2] = {0.0f, 0.0f};
                    if constexpr (I8) {
                        // exponents of V's scales, so that weight times scale stays at most 2
                        above[0] = static_cast<float>(max((__float_as_int(sc[m].z) >> 23) - 127, -90));
                        above[1] = static_cast<float>(max((__float_as_int(sc[m].w) >> 23) - 127, -90));
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float y = s[nt][m][0][e];
                        if constexpr (kChains == 2) y += s[nt][m][1][e];
                        if constexpr (I8) y *= e < 2 ? sc[m].x : sc[m].y;
                        y *= qs[nt][e & 1];
                        x[m][e] = g + (e < 2 ? 0 : 8) < usable ? y : __int_as_float(0xff800000);
                        up[e & 1] = fmaxf(up[e & 1], I8 ? x[m][e] + above[e >> 1] : x[m][e]);
                    }
                }
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) {
                    up[0] = fmaxf(up[0], __shfl_xor_sync(0xffffffffu, up[0], d));
                    up[1] = fmaxf(up[1], __shfl_xor_sync(0xffffffffu, up[1], d));
                }
                const bool raise = up[0] > m_run[nt][0] || up[1] > m_run[nt][1];
                if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float to = fmaxf(m_run[nt][e], up[e]);
                        const float a = to == __int_as_float(0xff800000) ? 1.0f : exp2_approx(m_run[nt][e] - to);
                        m_run[nt][e] = to;
                        l[nt][e] *= a;
#pragma unroll
                        for (int k = 0; k < S::kMma; ++k) {
                            acc[nt][k][e] *= a;
                            acc[nt][k][e + 2] *= a;
                        }
                    }
                }
                // no finite score yet: every weight is zero
                const float ref0 = m_run[nt][0] == __int_as_float(0xff800000) ? 0.0f : m_run[nt][0] - kLift;
                const float ref1 = m_run[nt][1] == __int_as_float(0xff800000) ? 0.0f : m_run[nt][1] - kLift;
#pragma unroll
                for (int m = 0; m < kSubs; ++m) {
                    float w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        w[e] = exp2_approx(x[m][e] - (e & 1 ? ref1 : ref0));
                        l[nt][e & 1] += w[e];
                        if constexpr (I8) {
                            // a masked token's scale is zero-filled: 0 * 0
                            w[e] *= e < 2 ? sc[m].z : sc[m].w;
                        }
                    }
                    const uint32_t h0 = pack2<BF>(w[0], w[1]), h1 = pack2<BF>(w[2], w[3]);
                    const float2 f0 = unpack2<BF>(h0), f1 = unpack2<BF>(h1);
                    hi0[nt][m] = transpose8(h0);
                    hi1[nt][m] = transpose8(h1);
                    lo0[nt][m] = transpose8(pack2<BF>(w[0] - f0.x, w[1] - f0.y));
                    lo1[nt][m] = transpose8(pack2<BF>(w[2] - f1.x, w[3] - f1.y));
                }
            }

            // ---- weighted values
            cp_async_wait<S::kStages - 2>();
            __syncwarp();
            tile = ring_ptr + S::stage_at(rd);
#pragma unroll
            for (int m = 0; m < kSubs; ++m)
#pragma unroll
                for (int z = 0; z < S::kSets; ++z) {
                    Words<S::kPiece> v[2][4];             // piece g, g + 8; tokens 2t, 2t+1, 2t+8, 2t+9
#pragma unroll
                    for (int y = 0; y < 8; ++y)
                        v[y >> 2][y & 3].v = *reinterpret_cast<const decltype(v[0][0].v)*>(
                            tile + place<S::kRow>(m * 16 + 2 * t + (y & 1) + (y & 2) * 4,
                                                  (z * 16 + (y >> 2) * 8 + g) * S::kPiece));
#pragma unroll
                    for (int w = 0; w < S::kPiece / 4; ++w) {
                        uint32_t a[4][I8 ? 4 : 2];        // operand registers of the word's channels
#pragma unroll
                        for (int r = 0; r < 4; ++r) {     // r: (piece, token pair) in A's order
                            uint32_t v0 = v[r & 1][(r >> 1) * 2][w], v1 = v[r & 1][(r >> 1) * 2 + 1][w];
                            if constexpr (!I8) {
                                a[r][0] = __byte_perm(v0, v1, 0x5410);
                                a[r][1] = __byte_perm(v0, v1, 0x7632);
                            } else {
                                v0 ^= 0x80808080u;
                                v1 ^= 0x80808080u;
                                const uint32_t p01 = __byte_perm(v0, v1, 0x5140), p23 = __byte_perm(v0, v1, 0x7362);
                                a[r][0] = codes_f16<0x4140>(p01);
                                a[r][1] = codes_f16<0x4342>(p01);
                                a[r][2] = codes_f16<0x4140>(p23);
                                a[r][3] = codes_f16<0x4342>(p23);
                            }
                        }
#pragma unroll
                        for (int i = 0; i < (I8 ? 4 : 2); ++i) {
                            const int k = z * S::kPerPiece + w * (I8 ? 4 : 2) + i;
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                mma<BF>(acc[nt][k], a[0][i], a[1][i], a[2][i], a[3][i], hi0[nt][m], hi1[nt][m]);
                                mma<BF>(acc[nt][k], a[0][i], a[1][i], a[2][i], a[3][i], lo0[nt][m], lo1[nt][m]);
                            }
                        }
                    }
                }
            fetch(2 * j + S::kStages, wr);
            rd = rd + 1 == S::kStages ? 0 : rd + 1;
            wr = wr + 1 == S::kStages ? 0 : wr + 1;
        }

        // ---- join the warps through shared memory
        const Segment was = seg;
        const int was_head0 = head0, was_nheads = nheads;
        const bool starts = was.k0 == 0, ends = was.k1 == was.blocks;
        more = next();
        if constexpr (S::kAhead) {
            // the next segment's first tiles are on their way meanwhile: the sums take the place
            // of stage 0 only, which it uses last
            if (more) prologue();
        }
        __syncthreads();                                  // every warp is through with its stages
        float* s_acc = reinterpret_cast<float*>(s_body);  // [warp][head][D + 4]
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int head = nt * 8 + 2 * t + e;
                float sum = l[nt][e];
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
                if (g == 0) {
                    s_m[warp * S::kHeads + head] = m_run[nt][e];
                    s_l[warp * S::kHeads + head] = sum;
                }
                float* dst = s_acc + (warp * S::kHeads + head) * (D + 4);
#pragma unroll
                for (int z = 0; z < S::kSets; ++z)
#pragma unroll
                    for (int half = 0; half < 2; ++half)
#pragma unroll
                        for (int k = 0; k < S::kPerPiece; k += 4)
                            *reinterpret_cast<float4*>(dst + (z * 16 + half * 8 + g) * S::kPerPiece + k) =
                                make_float4(acc[nt][z * S::kPerPiece + k][2 * half + e],
                                            acc[nt][z * S::kPerPiece + k + 1][2 * half + e],
                                            acc[nt][z * S::kPerPiece + k + 2][2 * half + e],
                                            acc[nt][z * S::kPerPiece + k + 3][2 * half + e]);
            }
        if (more) load_queries();
        __syncthreads();
        const int slot = starts ? 2 * c + 1 : 2 * c;      // piece of an unfinished row
        for (int i = tid; i < was_nheads * (D / 4); i += kThreads) {
            const int head = i / (D / 4), d = (i % (D / 4)) * 4;
            float top = s_m[head];
#pragma unroll
            for (int w = 1; w < kWarps; ++w) top = fmaxf(top, s_m[w * S::kHeads + head]);
            const float ref = top == __int_as_float(0xff800000) ? 0.0f : top;
            float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float a = exp2_approx(s_m[w * S::kHeads + head] - ref);
                const float4 x = *reinterpret_cast<const float4*>(s_acc + (w * S::kHeads + head) * (D + 4) + d);
                sum += a * s_l[w * S::kHeads + head];
                o.x += a * x.x;
                o.y += a * x.y;
                o.z += a * x.z;
                o.w += a * x.w;
            }
            if (CL && p.ctas > 1) {
                // the CTA's sums in place of the first warp's
                *reinterpret_cast<float4*>(s_acc + head * (D + 4) + d) = o;
                if (d == 0) {
                    s_part[2 * head] = top;
                    s_part[2 * head + 1] = sum;
                }
            } else if (CL || (starts && ends)) {
                // nothing to attend to (no usable page): zeros
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                QT* dst = out + (static_cast<size_t>(was.b) * heads_total + was_head0 + head) * D + d;
                *reinterpret_cast<uint2*>(dst) =
                    make_uint2(pack2<QBF>(o.x * inv, o.y * inv), pack2<QBF>(o.z * inv, o.w * inv));
            } else {
                const size_t at = static_cast<size_t>(slot) * S::kHeads + head;
                *reinterpret_cast<float4*>(p.part + at * D + d) = o;
                if (d == 0) *reinterpret_cast<float2*>(p.part_ml + 2 * at) = make_float2(top, sum);
            }
        }
        if constexpr (CL) {
            if (p.ctas > 1) {
                cg::cluster_group cluster = cg::this_cluster();
                cluster.sync();
                const int items = was_nheads * (D / 4);
                for (int i = cluster.block_rank() * kThreads + tid; i < items; i += p.ctas * kThreads) {
                    const int head = i / (D / 4), d = (i % (D / 4)) * 4;
                    float top = __int_as_float(0xff800000), sum = 0.0f;
                    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    for (int r0 = 0; r0 < p.ctas; r0 += 8) {          // eight CTAs at a time
                        float2 ml[8];
                        float4 x[8];
#pragma unroll
                        for (int r = 0; r < 8; ++r)
                            if (r0 + r < p.ctas) {
                                ml[r] = *reinterpret_cast<const float2*>(cluster.map_shared_rank(s_part, r0 + r) + 2 * head);
                                x[r] = *reinterpret_cast<const float4*>(cluster.map_shared_rank(s_acc, r0 + r) +
                                                                        head * (D + 4) + d);
                            }
                        float to = top;
#pragma unroll
                        for (int r = 0; r < 8; ++r)
                            if (r0 + r < p.ctas) to = fmaxf(to, ml[r].x);
                        const float ref = to == __int_as_float(0xff800000) ? 0.0f : to;
                        const float down = exp2_approx(top - ref);
                        top = to;
                        sum *= down;
                        o.x *= down;
                        o.y *= down;
                        o.z *= down;
                        o.w *= down;
#pragma unroll
                        for (int r = 0; r < 8; ++r)
                            if (r0 + r < p.ctas) {
                                const float a = exp2_approx(ml[r].x - ref);
                                sum += a * ml[r].y;
                                o.x += a * x[r].x;
                                o.y += a * x[r].y;
                                o.z += a * x[r].z;
                                o.w += a * x[r].w;
                            }
                    }
                    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                    QT* dst = out + (static_cast<size_t>(was.b) * heads_total + was_head0 + head) * D + d;
                    *reinterpret_cast<uint2*>(dst) =
                        make_uint2(pack2<QBF>(o.x * inv, o.y * inv), pack2<QBF>(o.z * inv, o.w * inv));
                }
                cluster.sync();                           // no CTA leaves while its sums are read
            }
            return;
        }
        if (starts && !ends) {
            unfinished_row = was.b * per_request + was.rr;
            // last CTA of the row: the one whose share holds the row's last block
            const long long last = static_cast<long long>(s_prefix[was.b]) * per_request +
                                   static_cast<long long>(was.rr + 1) * (was.blocks + p.row_cost) - 1;
            long long cl = last * shares / total;         // near; settled by the shares themselves
            while (cl + 1 < shares && total * (cl + 1) / shares <= last) ++cl;
            while (cl > 0 && total * cl / shares > last) --cl;
            unfinished_last = static_cast<int>(cl);
        }
        if (more) {
            __syncthreads();                              // the sums are read
            if constexpr (!S::kAhead) prologue();
        }
    }
    if (tid == 0 && p.meta != nullptr) {
        p.meta[2 * c] = unfinished_row;
        p.meta[2 * c + 1] = unfinished_last;
    }
}

constexpr int kJoinThreads = 256;

// Joins the pieces of the row that CTA blockIdx.x of the attention started and did not
// finish: its own last piece, then the first pieces of the following CTAs, in order.  Four
// channels per thread.  MANY: rows of many pieces, a head per block, its threads in groups that
// share the pieces; otherwise as many heads as fill the block, every thread all pieces.  With 64
// ragged rows of some 5 pieces the second takes 1.0 to 2.1 us less (fewer blocks, one round of
// loads); with 2 rows of 64 pieces 2.8 us more.
constexpr int kManyRows = 32;        // from here on the second form
template <bool QBF, int D, bool MANY>
__global__ void __launch_bounds__(kJoinThreads) attend_join_kernel(const AttendParams p) {
    extern __shared__ __align__(16) float s_w[];          // MANY: [ctas] weights, then [groups][D] sums
    constexpr int kLanes = D / 4, kGroups = kJoinThreads / kLanes;
    const int first = blockIdx.x, tid = threadIdx.x, grp = tid / kLanes, d = tid % kLanes * 4;
    const int head = MANY ? blockIdx.y : blockIdx.y * kGroups + grp;
    grid_launch_dependents();
    grid_dependency_wait();
    const int row = p.meta[2 * first];
    if (row < 0) return;
    const int n = p.meta[2 * first + 1] - first + 1;
    const int per_request = p.H * p.chunks;
    const int b = row / per_request, rr = row - b * per_request;
    const int h = rr / p.chunks, chunk = rr - h * p.chunks;
    if (head >= p.heads || chunk * p.heads + head >= p.group) return;
    // piece 0 is slot 2 first + 1; piece i is slot 2 (first + i)
    auto piece = [&](int i) { return static_cast<size_t>(2 * (first + i) + (i == 0)) * p.heads + head; };
    using QT = typename std::conditional<QBF, __nv_bfloat16, __half>::type;
    QT* dst = static_cast<QT*>(p.out) +
              (static_cast<size_t>(b) * p.H * p.group + h * p.group + chunk * p.heads + head) * D + d;
    if constexpr (!MANY) {
        constexpr int kAtOnce = 8;
        float top = __int_as_float(0xff800000), sum = 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int i0 = 0; i0 < n; i0 += kAtOnce) {
            float2 ml[kAtOnce];
            float4 x[kAtOnce];
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i)
                if (i0 + i < n) {
                    ml[i] = *reinterpret_cast<const float2*>(p.part_ml + 2 * piece(i0 + i));
                    x[i] = *reinterpret_cast<const float4*>(p.part + piece(i0 + i) * D + d);
                }
            float to = top;
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i)
                if (i0 + i < n) to = fmaxf(to, ml[i].x);
            const float ref = to == __int_as_float(0xff800000) ? 0.0f : to;
            const float down = exp2_approx(top - ref);
            top = to;
            sum *= down;
            o.x *= down;
            o.y *= down;
            o.z *= down;
            o.w *= down;
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i)
                if (i0 + i < n) {
                    const float a = exp2_approx(ml[i].x - ref);
                    sum += a * ml[i].y;
                    o.x += a * x[i].x;
                    o.y += a * x[i].y;
                    o.z += a * x[i].z;
                    o.w += a * x[i].w;
                }
        }
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        *reinterpret_cast<uint2*>(dst) =
            make_uint2(pack2<QBF>(o.x * inv, o.y * inv), pack2<QBF>(o.z * inv, o.w * inv));
        return;
    }
    __shared__ float s_red[kJoinThreads / 32 + 1];
    float top = __int_as_float(0xff800000);
    for (int i = tid; i < n; i += kJoinThreads) top = fmaxf(top, p.part_ml[2 * piece(i)]);
#pragma unroll
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    if ((tid & 31) == 0) s_red[tid >> 5] = top;
    __syncthreads();
    top = s_red[0];
#pragma unroll
    for (int w = 1; w < kJoinThreads / 32; ++w) top = fmaxf(top, s_red[w]);
    const float ref = top == __int_as_float(0xff800000) ? 0.0f : top;
    __syncthreads();
    float sum = 0.0f;
    for (int i = tid; i < n; i += kJoinThreads) {
        const float a = exp2_approx(p.part_ml[2 * piece(i)] - ref);
        s_w[i] = a;
        sum += a * p.part_ml[2 * piece(i) + 1];
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if ((tid & 31) == 0) s_red[tid >> 5] = sum;
    __syncthreads();
    sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kJoinThreads / 32; ++w) sum += s_red[w];
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;

    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int i = grp; i < n; i += kGroups) {
        const float a = s_w[i];
        const float4 x = *reinterpret_cast<const float4*>(p.part + piece(i) * D + d);
        o.x += a * x.x;
        o.y += a * x.y;
        o.z += a * x.z;
        o.w += a * x.w;
    }
    float* s_o = s_w + ((p.ctas + 3) & ~3);
    *reinterpret_cast<float4*>(s_o + grp * D + d) = o;
    __syncthreads();
    if (grp == 0) {
#pragma unroll
        for (int k = 1; k < kGroups; ++k) {
            const float4 x = *reinterpret_cast<const float4*>(s_o + k * D + d);
            o.x += x.x;
            o.y += x.y;
            o.z += x.z;
            o.w += x.w;
        }
        *reinterpret_cast<uint2*>(dst) =
            make_uint2(pack2<QBF>(o.x * inv, o.y * inv), pack2<QBF>(o.z * inv, o.w * inv));
    }
}

template <bool QBF, bool I8, int D, int NT>
cudaError_t launch(const AttendParams& p, AttendForm form, cudaStream_t st) {
    using S = Shape<QBF, I8, D, NT>;
    if (form == kAttendCluster) {
        static SmemLimit limit;
        cudaError_t e = limit.ensure(attend_kernel<QBF, I8, D, NT, true>, S::kShared);
        if (e == cudaSuccess && p.ctas > 8)
            e = cudaFuncSetAttribute(attend_kernel<QBF, I8, D, NT, true>,
                                     cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(p.B * p.H * p.chunks * p.ctas);
        cfg.blockDim = dim3(kThreads);
        cfg.dynamicSmemBytes = S::kShared;
        cfg.stream = st;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = p.ctas;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = pdl_allowed() ? 2 : 1;
        return cudaLaunchKernelEx(&cfg, attend_kernel<QBF, I8, D, NT, true>, p);
    }
    static SmemLimit limit;
    cudaError_t e = limit.ensure(attend_kernel<QBF, I8, D, NT, false>, S::kShared);
    if (e != cudaSuccess) return e;
    e = launch_chained(attend_kernel<QBF, I8, D, NT, false>, dim3(p.ctas), dim3(kThreads), S::kShared, st, p);
    if (e != cudaSuccess || form == kAttendWhole) return e;
    if (p.B * p.H * p.chunks >= kManyRows) {
        constexpr int kGroups = kJoinThreads / (D / 4);
        return launch_chained(attend_join_kernel<QBF, D, false>, dim3(p.ctas, (p.heads + kGroups - 1) / kGroups),
                              dim3(kJoinThreads), 0, st, p);
    }
    const size_t smem = (((p.ctas + 3) & ~3) + kJoinThreads / (D / 4) * D) * sizeof(float);
    return launch_chained(attend_join_kernel<QBF, D, true>, dim3(p.ctas, p.heads), dim3(kJoinThreads), smem,
                          st, p);
}

template <bool QBF, bool I8>
cudaError_t launch_any(const AttendParams& p, AttendForm form, cudaStream_t st) {
    if (p.heads == 8) {
        if (p.D == 64) return launch<QBF, I8, 64, 1>(p, form, st);
        if (p.D == 128) return launch<QBF, I8, 128, 1>(p, form, st);
        return launch<QBF, I8, 256, 1>(p, form, st);
    }
    if (p.D == 64) return launch<QBF, I8, 64, 2>(p, form, st);
    if (p.D == 128) return launch<QBF, I8, 128, 2>(p, form, st);
    return launch<QBF, I8, 256, 2>(p, form, st);
}

}  // namespace attend
}  // namespace escha
