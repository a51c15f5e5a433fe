// Born attention over a paged cache, BF16 caches.
#include "born_paged.h"

namespace qdl {

template <>
hipError_t paged_fwd<BF16>(const PagedArgs& a, hipStream_t st) {
    return launch_paged<BF16>(a, st);
}

}  // namespace qdl
