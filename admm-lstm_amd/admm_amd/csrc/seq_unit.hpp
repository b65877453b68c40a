// seq_unit.hpp -- operands and work memory of the gated unit's kernels.
#pragma once
#include <stdint.h>

namespace seq {

struct UnitArgs {
  int M, D, F, act, dtype;
  const void *x, *wg, *wu;
  int64_t x_ld, w_ld, wu_ld;
  bool copy_x, copy_w;          // operands that need padded copies (f32: always, as planes)
  char *xp, *wgp, *wup;         // their copies
  int64_t D8, F8;               // row lengths of the copies, in elements
  float *pre;                   // a, then b [M, F] (NULL: not kept)
  void* y;
  // gradients
  const void* dy;
  int64_t dy_ld;
  char *dap, *dbp;              // [planes][M, F8]
  void *dx, *dwg, *dwu;
};

}  // namespace seq
