// Packed Born attention, F32 inputs.
#include "born_packed.h"

namespace qdl {

template <>
hipError_t packed_fwd<F32>(const PackedArgs& a, const PackedPlan& plan, hipStream_t st) {
    return launch_packed_fwd<F32>(a, plan, st);
}
template <>
hipError_t packed_bwd<F32>(const PackedArgs& a, const PackedPlan& plan, hipStream_t st) {
    return launch_packed_bwd<F32>(a, plan, st);
}

}  // namespace qdl
