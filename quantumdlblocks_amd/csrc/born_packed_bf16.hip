// Packed Born attention, BF16 inputs.
#include "born_packed.h"

namespace qdl {

template <>
hipError_t packed_fwd<BF16>(const PackedArgs& a, const PackedPlan& plan, hipStream_t st) {
    return launch_packed_fwd<BF16>(a, plan, st);
}
template <>
hipError_t packed_bwd<BF16>(const PackedArgs& a, const PackedPlan& plan, hipStream_t st) {
    return launch_packed_bwd<BF16>(a, plan, st);
}

}  // namespace qdl
