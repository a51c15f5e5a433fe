// Born attention over a paged cache, F32 caches.
#include "born_paged.h"

namespace qdl {

template <>
hipError_t paged_fwd<F32>(const PagedArgs& a, hipStream_t st) {
    return launch_paged<F32>(a, st);
}

}  // namespace qdl
