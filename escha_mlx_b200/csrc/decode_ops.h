// Launchers of the decode step's operators around the projections: page plans, the paged
// key-value cache, attention over it and sampling.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace escha {

// Element types of the boundary (escha_b200.h: ESCHA_F16 ...).
constexpr int kF16 = 0, kBF16 = 1, kF32 = 2, kI8 = 3;

// Multiprocessors of the current device.
int sm_count();

constexpr int kPlanMaxBatch = 4096;

struct PlanParams {
    int32_t* table;          // [B, W], entries of newly taken pages are written
    const int32_t* lengths;  // [B]
    const int32_t* added;    // [B]
    const int32_t* free_pages;  // [F]
    const int32_t* head;     // [1]
    int32_t* slots;          // [rows]
    int32_t* positions;      // [rows]
    int32_t* starts;         // [B + 1]
    int32_t* ends;           // [B]
    int32_t* head_out;       // [1]
    int32_t* refused;        // [1]
    int B, W, F, rows, log_page, n_pages;
};
cudaError_t launch_page_plan(const PlanParams& p, cudaStream_t st);

struct AppendParams {
    const void* k;           // [T, H, D] with strides (elements)
    const void* v;
    long k_row, k_head, v_row, v_head;
    const int32_t* slots;    // [T]
    void* k_cache;           // [n_pages, H, P, D]
    void* v_cache;
    float* k_scale;          // [n_pages, H, P], 8-bit cache only
    float* v_scale;
    int T, H, D, log_page, n_pages;
};
// 16-bit caches take rows of their own type (a copy); the 8-bit cache takes f16 or bf16 rows.
cudaError_t launch_paged_append(const AppendParams& p, int in_type, int cache_type, cudaStream_t st);

// Requests of one attention launch (their prefix of token blocks sits in shared memory).
constexpr int kAttendMaxBatch = 1024;
// Tokens that a CTA takes at a time, and the granularity of the split over the cache.
constexpr int kAttendBlock = 64;

struct AttendParams {
    const void* q;           // [B, H * group, D] with strides (elements)
    long q_row, q_head;
    const void* k_cache;     // [n_pages, H, P, D]
    const void* v_cache;
    const float* k_scale;    // [n_pages, H, P], 8-bit cache only
    const float* v_scale;
    const int32_t* table;    // [B, W]
    const int32_t* lengths;  // [B]
    void* out;               // [B, H * group, D]
    int32_t* meta;           // [ctas][2]: row that a CTA starts and leaves unfinished, last CTA of it
    float* part_ml;          // [2 * ctas][heads][2]
    float* part;             // [2 * ctas][heads][D]
    float scale_log2;        // score scale times log2(e)
    int B, H, group, chunks, heads, D, W, log_page, n_pages, ctas;
    int row_cost;            // blocks that the start of a row counts for
};
// How rows (a request's query heads of one key/value head) are shared out: a cluster each,
// equal shares that cut rows (and a join), or equal shares that cannot.
enum AttendForm { kAttendCluster, kAttendSplit, kAttendWhole };
struct AttendShape {
    AttendForm form;
    int heads;    // query heads of one work item: 8 or 16 at most
    int chunks;   // work items per key/value head
    int ctas;     // CTAs per row (cluster), or of the launch
    size_t meta_bytes, ml_bytes, part_bytes;
};
// What starting a row costs, in blocks of its cache (`bytes` per token).  Measured with 32 to 64
// ragged requests, cost 0 / 2 / 4 / 8 / 16: 512 bytes 57.8 / 54.3 / 54.4 / 54.3 / 53.7 us, 256
// bytes 87.8 / 69.4 / 69.0 / 68.8 / 69.9, 128 bytes 110 / 99 / 88 / 80 / 83, 64 bytes 117 / 108 /
// 100 / 92 / 94.
constexpr int attend_row_cost(int bytes) { return 1024 / bytes < 8 ? 1024 / bytes : 8; }
AttendShape attend_shape(int B, int H, int group, int D, int W, int log_page, int sms);
cudaError_t launch_attend(const AttendParams& p, int q_type, int cache_type, AttendForm form,
                          cudaStream_t st);

struct SampleParams {
    const void* logits;      // [B, V], rows `stride` elements apart
    const float* uniforms;   // [B]
    // per row, or NULL for the number beside it
    const float* temperature;
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    float temperature1, top_p1, min_p1;
    int top_k1;
    int64_t* tokens;         // [B]
    long stride;
    int B, V, slice;
    bool by_length;          // rows in the order of what their settings may cost
};
int sample_max_vocab(int type);
cudaError_t launch_sample(const SampleParams& p, int type, cudaStream_t st);

}  // namespace escha
