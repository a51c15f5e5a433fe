// Born attention over a 4-bit paged cache, F32 queries.
#include "born_fp4_tiled.h"

namespace qdl {

template <>
hipError_t fp4_paged_fwd<F32>(const Fp4PagedArgs& a, const Fp4Plan& plan, hipStream_t st) {
    return launch_fp4<F32>(a, plan, st);
}

}  // namespace qdl
