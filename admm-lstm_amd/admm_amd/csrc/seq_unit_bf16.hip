// seq_unit_bf16.hip -- the gated unit's kernels for bf16.
#include "seq_unit_kernels.hpp"

namespace seq {
hipError_t unit_forward_bf16(const UnitArgs& u, hipStream_t s) { return forward<SEQ_BF16>(u, s); }
hipError_t unit_backward_bf16(const UnitArgs& u, hipStream_t s) { return backward<SEQ_BF16>(u, s); }
}  // namespace seq
