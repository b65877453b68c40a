// seq_unit_act.hpp -- the gated unit's activations.
#pragma once
#include "seq_dev.hpp"

namespace seq {
namespace {

__device__ __forceinline__ float sigmoid(float z) { return admm::sigm(z); }

// act(z), and its derivative
__device__ __forceinline__ float act(int kind, float z) {
  if (kind == SEQ_SILU) return z * sigmoid(z);
  if (kind == SEQ_GELU) return 0.5f * z * erfcf(-0.70710678118654752f * z);
  return sigmoid(z);
}
__device__ __forceinline__ void act_grad(int kind, float z, float& f, float& df) {
  if (kind == SEQ_GELU) {
    const float phi = 0.5f * erfcf(-0.70710678118654752f * z);
    f = z * phi;
    df = fmaf(z, 0.39894228040143268f * expf(-0.5f * z * z), phi);
  } else {
    const admm::SigPair s = admm::sig_pair(z);
    if (kind == SEQ_SILU) {
      f = z * s.s;
      df = s.s * fmaf(z, s.sc, 1.f);
    } else {
      f = s.s;
      df = s.s * s.sc;
    }
  }
}

}  // namespace
}  // namespace seq
