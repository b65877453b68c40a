// seq_unit_fp32.hip -- the gated unit's kernels for fp32.
#include "seq_unit_kernels.hpp"

namespace seq {
hipError_t unit_forward_fp32(const UnitArgs& u, hipStream_t s) { return forward<SEQ_FP32>(u, s); }
hipError_t unit_backward_fp32(const UnitArgs& u, hipStream_t s) { return backward<SEQ_FP32>(u, s); }
}  // namespace seq
