// binary16 queries over a cache of 8-bit codes.
#include "paged_attend.cuh"

namespace escha {
namespace attend {
template cudaError_t launch_any<false, true>(const AttendParams&, AttendForm, cudaStream_t);
}  // namespace attend
}  // namespace escha
