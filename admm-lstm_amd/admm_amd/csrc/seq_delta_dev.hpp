// seq_delta_dev.hpp -- what the forward and backward kernels of the gated delta rule share.
#pragma once
#include "seq_delta.hpp"

#include <type_traits>

namespace seq {
namespace {

// ---- 16-bit tiles in LDS (tile_at), whole fragments of them

// operand A (B): the lane's row (column) `row`, values 32 s + 8 g..+7
template <int W, int NP, int TILE>
__device__ __forceinline__ void frag(const __bf16* base, int row, int s, int g, bf16x8 (&a)[NP]) {
  const int at = tile_at<W>(row, 4 * s + g);
#pragma unroll
  for (int i = 0; i < NP; ++i) a[i] = *reinterpret_cast<const bf16x8*>(base + i * TILE + at);
}
// the same of the transposed tile: column perm_row(t, x), rows 32 s + 8 g..+7
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
// column 16 t + x, rows 32 s + 8 g..+7
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

// ---- fragments in the work memory and operands B in LDS

// sum over the 16 lanes of a row of the wave, in all of them: rotations within the row, which cost an addition no more time
template <int N>
__device__ __forceinline__ float add_turned(float v) {
  return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x120 + N, 0xf, 0xf, false));
}
__device__ __forceinline__ float sum16(float v) { return add_turned<1>(add_turned<2>(add_turned<4>(add_turned<8>(v)))); }

// Offsets made from these are made where they are used: worked out once before a loop they take more registers than there are
__device__ __forceinline__ void here(int& g, int& x) { asm volatile("" : "+v"(g), "+v"(x)); }

// Element `at` of an array that begins at a scalar address: with 32-bit offsets an access needs one register, not two.  at times
// the element's size is below 2^32
template <class T>
__device__ __forceinline__ T& item(T* base, uint32_t at) {
  using Byte = std::conditional_t<std::is_const_v<T>, const char, char>;
  return *reinterpret_cast<T*>(reinterpret_cast<Byte*>(base) + (uint32_t)(at * (uint32_t)sizeof(T)));
}

// keeps a branch around what hardly ever runs (the compiler would rather run both sides and select)
__device__ __forceinline__ void rare_path() { asm volatile(""); }

// sum over S inner steps of a[s] b(s), a step's plane pairs and the steps in several chains: a matrix instruction that takes the
// result of the last one waits for all of it
template <int NA, int NB, int L, int S, class B>
__device__ __forceinline__ f32x4 product(const bf16x8 (&a)[S][NA], const B& load) {
  constexpr int kChains = S >= 4 ? 4 : S == 2 ? 4 : 2;
  f32x4 acc[kChains];
#pragma unroll
  for (int c = 0; c < kChains; ++c) acc[c] = f32x4{0.f, 0.f, 0.f, 0.f};
  bf16x8 b[S][NB];
#pragma unroll
  for (int s = 0; s < S; ++s) load(s, b[s]);
  int n[S] = {};
#pragma unroll
  for (int q = L - 1; q >= 0; --q)
#pragma unroll
    for (int i = 0; i < NA; ++i)
      if (q - i >= 0 && q - i < NB) {
#pragma unroll
        for (int s = 0; s < S; ++s) {
          const int c = S >= 4 ? s % 4 : S == 2 ? 2 * s + (n[s] & 1) : n[s] & 1;
          acc[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[s][i], b[s][q - i], acc[c], 0, 0, 0);
          ++n[s];
        }
      }
  f32x4 sum = acc[0] + acc[1];
  if (kChains == 4) sum += acc[2 % kChains] + acc[3 % kChains];
  return sum;
}

// a value that is the same in all lanes, as a scalar (addresses made of it need no vector arithmetic)
__device__ __forceinline__ int64_t uniform(int64_t v) {
  return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v) |
                   (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32);
}

// base: scalar; at16: 16 * lane
template <int NP>
__device__ __forceinline__ void load_frag(const char* base, int plane, uint32_t at16, bf16x8 (&a)[NP]) {
#pragma unroll
  for (int i = 0; i < NP; ++i) a[i] = *reinterpret_cast<const bf16x8*>(base + (plane + i) * 1024 + at16);
}
// half p (rows of tile 2 s + p) of an operand B
template <int NP>
__device__ __forceinline__ void put_half(char* lds, int s, int p, int lane, f32x4 v) {
  f32x4 r = v;
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const bf16x4 b = __builtin_convertvector(r, bf16x4);
    *reinterpret_cast<bf16x4*>(lds + (s * NP + i) * 1024 + lane * 16 + 8 * p) = b;
    if (i + 1 < NP) r -= admm::bf16_widen<f32x4>(b);
  }
}
template <int NP>
__device__ __forceinline__ void put_whole(char* lds, int s, int lane, f32x8 v) {
  bf16x8 b[NP];
  planes8<NP>(v, b);
#pragma unroll
  for (int i = 0; i < NP; ++i) *reinterpret_cast<bf16x8*>(lds + (s * NP + i) * 1024 + lane * 16) = b[i];
}
// the first NB of an operand's NP planes
template <int NP, int NB = NP>
__device__ __forceinline__ void get_operand(const char* lds, int s, int lane, bf16x8 (&b)[NB]) {
#pragma unroll
  for (int i = 0; i < NB; ++i) b[i] = *reinterpret_cast<const bf16x8*>(lds + (s * NP + i) * 1024 + lane * 16);
}
// LDS writes of all waves before, LDS reads after; loads from global memory stay in flight
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// A lane's share of a chunk's rows of a tensor: rows perm_row(t, 4 g + r) of the lane's column.  The loads are unconditional
// (rows and columns outside are taken from the nearest inside, and become zeros on the way out), so that all of them are in
// flight at once; a branch around each made the compiler wait for each.
template <class T, int C>
struct ColumnRows {
  T raw[4];
  int left;   // rows of the chunk
  // p: the chunk's first row, at the lane's column or the row's last; at[r]: r rows behind the lane's first (in elements)
  __device__ __forceinline__ void load(const T* p, const int64_t (&at)[4], int64_t stride, int rows, int row0) {
    left = rows;
    if (rows == C) {
#pragma unroll
      for (int r = 0; r < 4; ++r) raw[r] = p[at[r]];
    } else {
      rare_path();
#pragma unroll
      for (int r = 0; r < 4; ++r) raw[r] = p[(row0 + r < rows ? row0 + r : rows - 1) * stride];
    }
  }
  __device__ __forceinline__ f32x4 get(bool in, int row0) const {
    f32x4 v;
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = in && row0 + r < left ? (float)raw[r] : 0.f;
    return v;
  }
};

// a lane's share of a [K, V] state: rows perm_row(t, 4 g + r) of its column, zeros outside
__device__ __forceinline__ f32x4 load_state(const float* p, int K, int V, int col, int t, int g) {
  f32x4 st = {0.f, 0.f, 0.f, 0.f};
  if (!p) return st;
  const int c = col < V ? col : V - 1, at = perm_row(t, 4 * g) * V + c, last = (K - 1) * V + c;   // K V <= 2^23
#pragma unroll
  for (int r = 0; r < 4; ++r) st[r] = p[min(at + r * V, last)];
#pragma unroll
  for (int r = 0; r < 4; ++r) st[r] = col < V && perm_row(t, 4 * g + r) < K ? st[r] : 0.f;
  return st;
}

// The value head and column tiles of this workgroup.  Workgroups are dealt out to the eight XCDs in turn: those of one sequence
// and query/key head, which read the same fragments, go to one XCD's L2.  false: none
__device__ __forceinline__ bool place_columns(const DeltaArgs& a, int groups, int64_t& n, int& h, int& hk, int& group) {
  const int share = a.Hv / a.Hk, per = share * groups;   // workgroups of a query/key head
  const int64_t unit = (int64_t)(blockIdx.x / 8 / per) * 8 + blockIdx.x % 8;
  if (unit >= a.rows.N * a.Hk) return false;
  const int at = (int)(blockIdx.x / 8 % per);
  n = unit / a.Hk;
  hk = (int)(unit % a.Hk);
  h = hk * share + at % share;
  group = at / share;
  return true;
}
// workgroups for that
inline unsigned column_blocks(const DeltaArgs& a, int groups) {
  return (unsigned)((a.rows.N * a.Hk + 7) / 8 * 8 * (a.Hv / a.Hk) * groups);
}

template <class F>
hipError_t allow_lds(F* f, int bytes) {
  return hipFuncSetAttribute(reinterpret_cast<const void*>(f), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

}  // namespace
}  // namespace seq
