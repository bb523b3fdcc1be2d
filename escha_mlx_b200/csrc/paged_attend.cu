// Shape and dispatch of the paged attention (kernels: paged_attend.cuh, one file per types).
#include "decode_ops.h"

namespace escha {

namespace attend {
template <bool QBF, bool I8>
cudaError_t launch_any(const AttendParams& p, AttendForm form, cudaStream_t st);
extern template cudaError_t launch_any<false, false>(const AttendParams&, AttendForm, cudaStream_t);
extern template cudaError_t launch_any<true, false>(const AttendParams&, AttendForm, cudaStream_t);
extern template cudaError_t launch_any<false, true>(const AttendParams&, AttendForm, cudaStream_t);
extern template cudaError_t launch_any<true, true>(const AttendParams&, AttendForm, cudaStream_t);
}  // namespace attend

// Longest table whose rows are cut inside a cluster.  Measured with all rows of that length, 2
// heads of 256, 1 / 4 / 16 requests, cluster against split and join: 512 tokens 5.6 / 6.0 / 9.4
// us against 8.7 / 9.3 / 12.5, 2048 tokens 8.4 / 10.4 / 16.0 against 9.4 / 12.6 / 20.7, 8192
// tokens 21 / 24 / 44 against 16 / 20 / 51.  With 37 requests (clusters of 4 that do not all fit
// at once) 39 against 33 at 2048.
constexpr int kClusterTokens = 2048;
// The same for a few rows, with clusters of 16: 1 / 4 requests 9.4 / 13.6 us against 12.7 / 15.4
// at 4096 tokens, 14.5 / 18.8 against 16.7 / 20.4 at 8192, 23 / 32 against 20 / 32 at 16384; 16
// rows 28 against 20 at 4096 (not all at once either).
constexpr int kWideTokens = 8192, kWideRows = 8;

AttendShape attend_shape(int B, int H, int group, int D, int W, int log_page, int sms) {
    AttendShape s;
    s.heads = group <= 8 ? 8 : 16;
    s.chunks = (group + s.heads - 1) / s.heads;
    const long long blocks = ((static_cast<long long>(W) << log_page) + kAttendBlock - 1) / kAttendBlock;
    const long long rows = static_cast<long long>(B) * H * s.chunks, fit = 2ll * sms;   // two CTAs fit an SM
    s.form = kAttendSplit;
    if (blocks * kAttendBlock <= kClusterTokens) {
        // the most CTAs per row that are resident together (clusters do not fill the last SMs of
        // a group), if they use most of the GPU or a row has no more blocks
        s.ctas = 1;
        while (s.ctas < 8 && s.ctas < blocks && 2 * s.ctas * rows <= fit - fit / 9) s.ctas *= 2;
        if (rows <= fit && (s.ctas >= 8 || s.ctas >= blocks || s.ctas * rows >= fit - fit / 2 + fit / 24))
            s.form = kAttendCluster;
    } else if (blocks * kAttendBlock <= kWideTokens && rows <= kWideRows) {
        s.ctas = 16;
        s.form = kAttendCluster;
    }
    if (s.form != kAttendCluster) {
        // rows are cut between blocks only
        s.form = blocks > 1 ? kAttendSplit : kAttendWhole;
        s.ctas = static_cast<int>(blocks * rows < fit ? blocks * rows : fit);
    }
    const size_t pieces = s.form == kAttendSplit ? 2ull * s.ctas * s.heads : 0;
    s.meta_bytes = s.form == kAttendSplit ? (2ull * s.ctas * 4 + 15) / 16 * 16 : 0;
    s.ml_bytes = pieces * 8;
    s.part_bytes = pieces * D * 4;
    return s;
}

cudaError_t launch_attend(const AttendParams& p, int q_type, int cache_type, AttendForm form,
                          cudaStream_t st) {
    if (cache_type == kI8)
        return q_type == kBF16 ? attend::launch_any<true, true>(p, form, st)
                               : attend::launch_any<false, true>(p, form, st);
    return q_type == kBF16 ? attend::launch_any<true, false>(p, form, st)
                           : attend::launch_any<false, false>(p, form, st);
}

}  // namespace escha
