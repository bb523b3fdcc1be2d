// Shape and dispatch of the paged attention (kernels: paged_attend.cuh, one file per types).
#include "decode_ops.h"

namespace escha {

namespace attend {
template <bool QBF, bool I8>
cudaError_t launch_any(const AttendParams& p, bool split, cudaStream_t st);
extern template cudaError_t launch_any<false, false>(const AttendParams&, bool, cudaStream_t);
extern template cudaError_t launch_any<true, false>(const AttendParams&, bool, cudaStream_t);
extern template cudaError_t launch_any<false, true>(const AttendParams&, bool, cudaStream_t);
extern template cudaError_t launch_any<true, true>(const AttendParams&, bool, cudaStream_t);
}  // namespace attend

AttendShape attend_shape(int B, int H, int group, int D, int W, int log_page, int sms) {
    AttendShape s;
    s.heads = group <= 8 ? 8 : 16;
    s.chunks = (group + s.heads - 1) / s.heads;
    const long long blocks = ((static_cast<long long>(W) << log_page) + kAttendBlock - 1) / kAttendBlock;
    const long long most = blocks * B * H * s.chunks;
    s.ctas = static_cast<int>(most < 2ll * sms ? most : 2ll * sms);   // two CTAs fit an SM
    s.split = blocks > 1;          // rows are cut between blocks only
    const size_t pieces = s.split ? 2ull * s.ctas * s.heads : 0;
    s.meta_bytes = s.split ? (2ull * s.ctas * 4 + 15) / 16 * 16 : 0;
    s.ml_bytes = pieces * 8;
    s.part_bytes = pieces * D * 4;
    return s;
}

cudaError_t launch_attend(const AttendParams& p, int q_type, int cache_type, bool split,
                          cudaStream_t st) {
    if (cache_type == kI8)
        return q_type == kBF16 ? attend::launch_any<true, true>(p, split, st)
                               : attend::launch_any<false, true>(p, split, st);
    return q_type == kBF16 ? attend::launch_any<true, false>(p, split, st)
                           : attend::launch_any<false, false>(p, split, st);
}

}  // namespace escha
