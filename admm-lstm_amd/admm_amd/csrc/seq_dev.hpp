// seq_dev.hpp -- device building blocks of the sequence-layer operators (libseqops.so), on top of admm_dev.hpp.
//
// Matrix products run on the bf16 matrix cores with operands held as sums of bf16 pieces ("planes"): a bf16 input is
// one plane, an fp16 input two (its 11 bits split 8 + 3, exact), an fp32 value three (to 2^-24 relative).  Products of
// planes i and j with i + j below the larger plane count are summed in the f32 accumulators: three per product of a
// bf16 input with an fp32 value, six for two fp32 values, at 16 times the fp32 matrix rate each.
#pragma once
#include <hip/hip_fp16.h>

#include "admm_dev.hpp"
#include "seq_ops.h"

namespace seq {

using admm::bf16x4;
using admm::bf16x8;
using admm::f32x4;
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

template <int DT> struct Elem;
template <> struct Elem<SEQ_BF16> { typedef __bf16 T; static constexpr int kPlanes = 1; };
template <> struct Elem<SEQ_FP16> { typedef _Float16 T; static constexpr int kPlanes = 2; };
template <> struct Elem<SEQ_FP32> { typedef float T; static constexpr int kPlanes = 3; };

// eight consecutive values of a row, n of them inside it (the others zero); `wide`: the row is 16-byte aligned, holds
// whole groups of eight, and may be read 16 bytes at a time
template <class T>
__device__ __forceinline__ f32x8 load8(const T* p, int n, bool wide) {
  f32x8 x;
  if (wide && n >= 8) {
    if constexpr (sizeof(T) == 4) {
      const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) { x[i] = a[i]; x[4 + i] = b[i]; }
    } else {
      typedef T T8 __attribute__((ext_vector_type(8)));
      const T8 v = *reinterpret_cast<const T8*>(p);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = (float)v[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = i < n ? (float)p[i] : 0.f;
  }
  return x;
}

// zero where every value is finite, NaN otherwise
__device__ __forceinline__ float zero_if_finite(f32x4 a) { return (a[0] * 0.f + a[1] * 0.f) + (a[2] * 0.f + a[3] * 0.f); }

// the first NP planes of eight values (the rest of each value after the NP planes is dropped)
template <int NP>
__device__ __forceinline__ void planes8(f32x8 x, bf16x8 (&p)[NP]) {
  p[0] = __builtin_convertvector(x, bf16x8);
  if constexpr (NP > 1) {
    const f32x8 r = x - admm::bf16_widen<f32x8>(p[0]);
    p[1] = __builtin_convertvector(r, bf16x8);
    if constexpr (NP > 2) p[2] = __builtin_convertvector(r - admm::bf16_widen<f32x8>(p[1]), bf16x8);
  }
}

// The same of any finite values: the first plane of those above the largest bf16 value, which would be infinite, is that value.  An
// infinity has NaN among its planes.
template <int NP>
__device__ __forceinline__ void planes8_whole(f32x8 x, bf16x8 (&p)[NP]) {
  constexpr float kMost = 0x1.fep127f;
  f32x8 c;
#pragma unroll
  for (int i = 0; i < 8; ++i) c[i] = __builtin_amdgcn_fmed3f(x[i], -kMost, kMost);
  p[0] = __builtin_convertvector(c, bf16x8);
  static_assert(NP == 3, "two planes and a remainder");
  const f32x8 r = x - admm::bf16_widen<f32x8>(p[0]);
  p[1] = __builtin_convertvector(r, bf16x8);
  p[2] = __builtin_convertvector(r - admm::bf16_widen<f32x8>(p[1]), bf16x8);
}

__device__ __forceinline__ f32x8 cat8(f32x4 a, f32x4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }

// acc += a b over the plane pairs i + j < L, the smallest terms first
template <int NA, int NB, int L>
__device__ __forceinline__ f32x4 mfma_planes(const bf16x8 (&a)[NA], const bf16x8 (&b)[NB], f32x4 acc) {
#pragma unroll
  for (int s = L - 1; s >= 0; --s)
#pragma unroll
    for (int i = 0; i < NA; ++i)
      if (s - i >= 0 && s - i < NB) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[s - i], acc, 0, 0, 0);
  return acc;
}

// acc[t] += a(t) b for R row tiles: plane pairs outside, rows inside, so that neighbouring instructions do not wait for each other
template <int NA, int NB, int L, int R, class A>
__device__ __forceinline__ void mfma_rows(const A& a, const bf16x8 (&b)[NB], f32x4 (&acc)[R]) {
#pragma unroll
  for (int s = L - 1; s >= 0; --s)
#pragma unroll
    for (int i = 0; i < NA; ++i)
      if (s - i >= 0 && s - i < NB) {
#pragma unroll
        for (int t = 0; t < R; ++t) acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a(t)[i], b[s - i], acc[t], 0, 0, 0);
      }
}

// Between matrix instructions and control flow behind which their results are read first.  The wait states that such a read needs
// are the compiler's to insert, and where two ways of different length lead to it, it has left them out on the shorter one.
__device__ __forceinline__ void mfma_settle() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_nop 15\n\ts_nop 3");
  __builtin_amdgcn_sched_barrier(0);
}

// 16 bytes a lane from global memory straight into LDS: `lds` is the wave's base, lane l's bytes land at lds + 16 l.
// The caller waits for them (vm_wait) before the barrier that hands them to other waves, and keeps other buffers' readers out by
// barriers too.  In assembly (m0: the LDS base; there is no result register) because the compiler, which cannot tell the
// buffers apart, waits for all such loads before the next transposing read of any of them.
__device__ __forceinline__ void glds16(const void* g, void* lds) {
  const uint32_t at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(at), "v"(g) : "memory");
}
// the wave's index, as a scalar
__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }
__device__ __forceinline__ void vm_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// Four rows by sixteen columns of 16-bit values, transposed on the way out of LDS: lane i of each 16 gives the address
// of row i / 4, columns 4 (i % 4)..+3, and gets the four rows of column i.
__device__ __forceinline__ bf16x4 tr4(const __bf16* p) {
  const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
  return __builtin_bit_cast(bf16x4, v);
}

// Tiles of 16-bit values in LDS: rows of W values (W = 32, 64 or 128) in pieces of eight (16 bytes), piece c of row r at
// place c ^ swz(r), so that eight neighbouring rows' pieces c lie in eight different groups of four banks.
template <int W>
__device__ __forceinline__ int tile_at(int r, int c) {
  constexpr int P = W / 8;
  const int x = P >= 8 ? r & (P - 1) & 15 : (r >> 1) & (P - 1);
  return r * W + 8 * (c ^ x);
}

}  // namespace seq
