// seq_unit_fp16.hip -- the gated unit's kernels for fp16.
#include "seq_unit_kernels.hpp"

namespace seq {
hipError_t unit_forward_fp16(const UnitArgs& u, hipStream_t s) { return forward<SEQ_FP16>(u, s); }
hipError_t unit_backward_fp16(const UnitArgs& u, hipStream_t s) { return backward<SEQ_FP16>(u, s); }
}  // namespace seq
