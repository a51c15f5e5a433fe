// Packed Born attention, F16 inputs.
#include "born_packed.h"

namespace qdl {

template <>
hipError_t packed_fwd<F16>(const PackedArgs& a, const PackedPlan& plan, hipStream_t st) {
    return launch_packed_fwd<F16>(a, plan, st);
}
template <>
hipError_t packed_bwd<F16>(const PackedArgs& a, const PackedPlan& plan, hipStream_t st) {
    return launch_packed_bwd<F16>(a, plan, st);
}

}  // namespace qdl
