// Born attention over a paged cache, F16 caches.
#include "born_paged.h"

namespace qdl {

template <>
hipError_t paged_fwd<F16>(const PagedArgs& a, hipStream_t st) {
    return launch_paged<F16>(a, st);
}

}  // namespace qdl
