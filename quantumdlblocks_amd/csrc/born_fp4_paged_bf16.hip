// Born attention over a 4-bit paged cache, BF16 queries.
#include "born_fp4_tiled.h"

namespace qdl {

template <>
hipError_t fp4_paged_fwd<BF16>(const Fp4PagedArgs& a, const Fp4Plan& plan, hipStream_t st) {
    return launch_fp4<BF16>(a, plan, st);
}

}  // namespace qdl
