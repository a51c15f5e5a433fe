// Born attention over a 4-bit paged cache, F32 queries.
#include "born_fp4_paged.h"
#include "born_fp4_tiled.h"

namespace qdl {

template <>
hipError_t fp4_paged_fwd<F32>(const Fp4PagedArgs& a, const Fp4Plan& plan, hipStream_t st) {
    const hipError_t e = launch_fp4_paged<F32>(a, plan, st);
    return e != hipSuccess || plan.slots == 0 ? e : launch_fp4_tiled<F32>(a, plan, st);
}

}  // namespace qdl
