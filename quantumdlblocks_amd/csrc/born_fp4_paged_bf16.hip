// Born attention over a 4-bit paged cache, BF16 queries.
#include "born_fp4_paged.h"
#include "born_fp4_tiled.h"

namespace qdl {

template <>
hipError_t fp4_paged_fwd<BF16>(const Fp4PagedArgs& a, const Fp4Plan& plan, hipStream_t st) {
    const hipError_t e = launch_fp4_paged<BF16>(a, plan, st);
    return e != hipSuccess || plan.slots == 0 ? e : launch_fp4_tiled<BF16>(a, plan, st);
}

}  // namespace qdl
