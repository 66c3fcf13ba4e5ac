/* Attention over a paged f32 cache (smq_paged_attend.h); one source per type of cache, compiled beside each other. */
#define SMQ_ATTEND_KERNELS
#include "smq_paged_attend.h"

namespace smq {
template hipError_t launch_attend<0, false>(const PagedArgs &, const TreeArgs &, const AttendPlan &, const float *, float *,
                                              i4 *, float *, hipStream_t);
}  // namespace smq
