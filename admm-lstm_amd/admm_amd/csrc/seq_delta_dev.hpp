// seq_delta_dev.hpp -- what the forward and backward kernels of the gated delta rule share: operand fragments, staging.
//
// v_mfma_f32_16x16x32_bf16: lane l = 16 g + x holds row (column) x of A (B), inner values 8 g..8 g + 7, and column x, rows
// 4 g..4 g + 3 of the result.  Two result tiles 2 s and 2 s + 1 whose row m stands for perm_row(2 s [+ 1], m) give lane l rows
// 32 s + 8 g..+7 of its column: an operand B of the next product as it stands.  So a chain of products needs no
// exchange between lanes, only the A operands' rows taken in that order.
#pragma once
#include "seq_delta.hpp"

namespace seq {
namespace {

__device__ __forceinline__ int perm_row(int t, int m) { return 32 * (t >> 1) + 8 * (m >> 2) + 4 * (t & 1) + (m & 3); }

// operand A of tile t: the lane's row, values 8 (4 s + g)..+7
template <int W, int NP, int TILE>
__device__ __forceinline__ void frag(const __bf16* base, int row, int s, int g, bf16x8 (&a)[NP]) {
  const int at = tile_at<W>(row, 4 * s + g);
#pragma unroll
  for (int i = 0; i < NP; ++i) a[i] = *reinterpret_cast<const bf16x8*>(base + i * TILE + at);
}

// operand A of tile t of the transposed tile: the lane's column perm_row(t, l % 16), rows 32 s + 8 g..+7
template <int W, int NP, int TILE>
__device__ __forceinline__ void frag_t(const __bf16* base, int t, int s, int g, int x, bf16x8 (&a)[NP]) {
  const int r = 32 * s + 8 * g + (x >> 2), c = 4 * (t >> 1) + (x & 3), h = 4 * (t & 1);
  const int lo = tile_at<W>(r, c) + h, hi = tile_at<W>(r + 4, c) + h;
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const bf16x4 u = tr4(base + i * TILE + lo), v = tr4(base + i * TILE + hi);
    a[i] = __builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7);
  }
}

// the same for the triangular tiles; frag_tri_t: columns perm_row(t, l % 16), rows 32 s + 8 g..+7
template <int NP>
__device__ __forceinline__ void frag_tri(const __bf16* base, int t, int s, int g, int x, bf16x8 (&a)[NP]) {
  const int at = t < 2 ? tile_at<32>(perm_row(t, x), g) : 32 * 32 + tile_at<64>(perm_row(t, x) - 32, 4 * s + g);
#pragma unroll
  for (int i = 0; i < NP; ++i) a[i] = *reinterpret_cast<const bf16x8*>(base + i * kTri + at);
}
template <int NP>
__device__ __forceinline__ void frag_tri_t(const __bf16* base, int t, int s, int g, int x, bf16x8 (&a)[NP]) {
  const int r = 8 * g + (x >> 2), c = 4 * (t >> 1) + (x & 3), h = 4 * (t & 1);
  const int lo = (s ? 32 * 32 + tile_at<64>(r, c) : tile_at<32>(r, c)) + h;
  const int hi = (s ? 32 * 32 + tile_at<64>(r + 4, c) : tile_at<32>(r + 4, c)) + h;
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const bf16x4 u = tr4(base + i * kTri + lo), v = tr4(base + i * kTri + hi);
    a[i] = __builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7);
  }
}
// operand B (or A, transposed) with columns 16 t + l % 16 of a tile in rows: rows 32 s + 8 g..+7
template <int W, int NP, int TILE>
__device__ __forceinline__ void frag_col(const __bf16* base, int t, int s, int g, int x, bf16x8 (&a)[NP]) {
  const int r = 32 * s + 8 * g + (x >> 2), c = 2 * t + ((x & 3) >> 1), h = 4 * (x & 1);
  const int lo = tile_at<W>(r, c) + h, hi = tile_at<W>(r + 4, c) + h;
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const bf16x4 u = tr4(base + i * TILE + lo), v = tr4(base + i * TILE + hi);
    a[i] = __builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7);
  }
}

// sum of a wave's values up to each lane, in f64: the decays' exponents are differences of such sums, and have to be
// right to 1e-7 where the sums are large (they are kept as two floats, hi + lo)
__device__ __forceinline__ double running_sum64(double sum, int lane, double& last) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const double up = __shfl_up(sum, d);
    if (lane >= d) sum += up;
  }
  last = __shfl(sum, 63);
  return sum;
}
__device__ __forceinline__ double running_sum(float v, int lane, double& last) { return running_sum64(v, lane, last); }

template <int DT, int KP, bool SAVE>
constexpr int scan_bufs() { return 2 * DeltaShape<DT, KP, SAVE>::kStage <= 160 * 1024 ? 2 : 1; }

// linear copy of a chunk's planes and vectors into LDS, 1 KB a wave at a time
template <class S, int WAVES>
__device__ __forceinline__ void stage_chunk(const DeltaArgs& a, int64_t c, int hk, int h, char* lds, int wave, int lane) {
  const char* kq = a.kq + (c * a.Hk + hk) * (int64_t)S::kKQ;
  const char* xp = a.xp + (c * a.Hv + h) * (int64_t)S::kXP;
  const char* vec = a.vec + (c * a.Hv + h) * (int64_t)S::kVec;
  for (int i = wave; i < S::kStage / 1024; i += WAVES) {
    const char* src = i < S::kKQ / 1024 ? kq + i * 1024
                      : i < (S::kKQ + S::kXP) / 1024 ? xp + (i * 1024 - S::kKQ) : vec;
    glds16(src + lane * 16, lds + i * 1024);
  }
}

template <class F>
hipError_t allow_lds(F* f, int bytes) {
  return hipFuncSetAttribute(reinterpret_cast<const void*>(f), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

}  // namespace
}  // namespace seq
