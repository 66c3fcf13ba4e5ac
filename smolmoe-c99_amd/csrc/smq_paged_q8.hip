/* Attention over a paged q8 cache (smq_paged_attend.h); one source per type of cache, compiled beside each other. */
#define SMQ_ATTEND_KERNELS
#include "smq_paged_attend.h"

namespace smq {
template hipError_t launch_attend<2>(const PagedArgs &, const AttendPlan &, const float *, float *, i4 *, float *,
                                       hipStream_t);
}  // namespace smq
