/* Attention of trees of drafted tokens over a paged f16 cache (smq_paged_attend.h). */
#define SMQ_ATTEND_KERNELS
#include "smq_paged_attend.h"

namespace smq {
template hipError_t launch_attend<1, true>(const PagedArgs &, const TreeArgs &, const AttendPlan &, const float *, float *,
                                             i4 *, float *, hipStream_t);
}  // namespace smq
