// binary16 queries over a cache of the same type.
#include "paged_attend.cuh"

namespace escha {
namespace attend {
template cudaError_t launch_any<false, false>(const AttendParams&, AttendForm, cudaStream_t);
}  // namespace attend
}  // namespace escha
