// seq_unit_few.hip -- the gated unit's forward for a few rows (single tokens of a few streams).
//
// Bound by the weights, which are read once: 4 D F bytes in 16 bits, and nothing may stand between them and the matrix cores.
// A lane loads 8 rows of 8 neighbouring weights (rows 8 g..8 g + 7 of the inner axis, columns 8 x..8 x + 7) straight into
// registers, 16 bytes a row whatever their alignment, and turns its 8 x 8 block over there (32 byte permutes): fragment j then has
// the weights of columns 8 x + j as the matrix instruction wants them, and eight of those make 128 columns.  f32 weights need no
// turning over: v_mfma_f32_16x16x4_f32 takes one weight a lane, at columns 4 x + j.  The rows of x are the other operand.  (An infinity
// of f32 is made NaN, which it is as planes in the kernels of more rows: the result does not depend on the number of rows.)
// The inner axis is split over the four waves of a workgroup and over workgroups, so that the loads in flight fill the memory
// system; where it is split over workgroups their sums go through work memory and are joined by k_unit_sum, in order.
#include "seq_dev.hpp"
#include "seq_unit.hpp"
#include "seq_unit_act.hpp"

namespace seq {
namespace {

constexpr int kWavesF = 4;
constexpr int kRowS = 66;   // a register of all lanes in LDS: two banks on, so that neighbouring columns lie in different banks
template <int DT> constexpr int few_cols() { return DT == SEQ_FP32 ? 64 : 128; }   // columns of a workgroup
template <int DT> constexpr int few_frags() { return DT == SEQ_FP32 ? 4 : 8; }     // fragments side by side

typedef _Float16 h8 __attribute__((ext_vector_type(8)));

template <class V>
__device__ __forceinline__ V load_any(const void* p) {   // of any alignment
  V v;
  __builtin_memcpy(&v, p, sizeof v);
  return v;
}

// NaN for an infinity, any other value as it is
__device__ __forceinline__ float finite_or_nan(float v) { return fmaf(v, 0.f, v); }

// 16 bytes of a row of n values from value c on, zeros outside
template <class T>
__device__ __forceinline__ u32x4 load_piece(const T* row, int c, int n) {
  constexpr int N = 16 / sizeof(T);
  if (c + N <= n) return load_any<u32x4>(row + c);
  typedef T V __attribute__((ext_vector_type(N)));
  V v;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = c + i < n ? row[c + i] : (T)0;
  return __builtin_bit_cast(u32x4, v);
}

template <int DT, int MT>
__global__ __launch_bounds__(64 * kWavesF) void k_unit_few(UnitArgs u, int splits, float* sums) {
  using T = typename Elem<DT>::T;
  constexpr int NF = few_frags<DT>(), COLS = few_cols<DT>(), STEP = DT == SEQ_FP32 ? 16 : 32;   // inner values of a step
  extern __shared__ __attribute__((aligned(16))) float part[];   // [wave][MT][matrix][fragment][r][lane]
  const int lane = threadIdx.x & 63, wave = wave_id(), x = lane & 15, g = lane >> 4;
  const int groups = (u.F + COLS - 1) / COLS, group = blockIdx.x % groups, split = blockIdx.x / groups;
  const int steps = (u.D + STEP - 1) / STEP, parts = splits * kWavesF, me = split * kWavesF + wave;
  const int first = (int)((int64_t)steps * me / parts), last = (int)((int64_t)steps * (me + 1) / parts);
  const int col = group * COLS + (DT == SEQ_FP32 ? 4 : 8) * x;
  const T* const w[2] = {static_cast<const T*>(u.wg), static_cast<const T*>(u.wu)};
  const int64_t ld[2] = {u.w_ld, u.wu_ld};
  const T* xr[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) xr[m] = static_cast<const T*>(u.x) + (16 * m + x < u.M ? 16 * m + x : u.M - 1) * u.x_ld;

  f32x4 acc[MT][2][NF];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int j = 0; j < NF; ++j) acc[m][e][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  for (int s = first; s < last; ++s) {
    const int k0 = s * STEP;
    if constexpr (DT == SEQ_FP32) {
      f32x4 b[2][4];   // inner values k0 + 4 i + g
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int k = k0 + 4 * i + g;
          b[e][i] = __builtin_bit_cast(f32x4, k < u.D && col < u.F ? load_piece<T>(w[e] + k * ld[e], col, u.F) : u32x4{0, 0, 0, 0});
#pragma unroll
          for (int j = 0; j < 4; ++j) b[e][i][j] = finite_or_nan(b[e][i][j]);
        }
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int k = k0 + 4 * i + g;
          const float xv = k < u.D ? finite_or_nan(xr[m][k]) : 0.f;
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              acc[m][e][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(b[e][i][j], xv, acc[m][e][j], 0, 0, 0);
        }
    } else {
      const int k = k0 + 8 * g;
      u32x4 b[2][8];   // rows k..k + 7
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          b[e][i] = k + i < u.D && col < u.F ? load_piece<T>(w[e] + (int64_t)(k + i) * ld[e], col, u.F) : u32x4{0, 0, 0, 0};
      bf16x8 xv[MT];
#pragma unroll
      for (int m = 0; m < MT; ++m) xv[m] = __builtin_bit_cast(bf16x8, k < u.D ? load_piece<T>(xr[m], k, u.D) : u32x4{0, 0, 0, 0});
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          u32x4 t;   // column 8 x + j, rows k..k + 7
#pragma unroll
          for (int i = 0; i < 4; ++i)
            t[i] = __builtin_amdgcn_perm(b[e][2 * i + 1][j / 2], b[e][2 * i][j / 2], j & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            if constexpr (DT == SEQ_FP16)
              acc[m][e][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, t), __builtin_bit_cast(h8, xv[m]), acc[m][e][j], 0, 0, 0);
            else
              acc[m][e][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, t), xv[m], acc[m][e][j], 0, 0, 0);
          }
        }
    }
  }
  mfma_settle();
  constexpr int kPart = MT * 2 * NF * 4 * kRowS;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int j = 0; j < NF; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) part[wave * kPart + (((m * 2 + e) * NF + j) * 4 + r) * kRowS + lane] = acc[m][e][j][r];
  __syncthreads();
  // row m, column n of the group: lane 16 g + m % 16, register r and fragment j with n = NF (4 g + r) + j
  const int rows = u.M < 16 * MT ? u.M : 16 * MT;
  for (int i = threadIdx.x; i < rows * COLS; i += 64 * kWavesF) {
    const int m = i / COLS, n = i % COLS, c = group * COLS + n;
    if (c >= u.F) continue;
    float v[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int at = ((((m >> 4) * 2 + e) * NF + n % NF) * 4 + (n / NF & 3)) * kRowS + (n / NF >> 2) * 16 + (m & 15);
      v[e] = (part[at] + part[kPart + at]) + (part[2 * kPart + at] + part[3 * kPart + at]);
    }
    const int64_t to = (int64_t)m * u.F + c, MF = (int64_t)u.M * u.F;
    if (splits > 1) {
      sums[(2 * split) * MF + to] = v[0];
      sums[(2 * split + 1) * MF + to] = v[1];
    } else {
      static_cast<T*>(u.y)[to] = (T)(act(u.act, v[0]) * v[1]);
      if (u.pre) {
        u.pre[to] = v[0];
        u.pre[MF + to] = v[1];
      }
    }
  }
}

template <class T>
__global__ __launch_bounds__(256) void k_unit_sum(UnitArgs u, int splits, const float* sums) {
  const int64_t MF = (int64_t)u.M * u.F;
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < MF; i += (int64_t)gridDim.x * 256) {
    float a = 0.f, b = 0.f;
    for (int s = 0; s < splits; ++s) {
      a += sums[2 * s * MF + i];
      b += sums[(2 * s + 1) * MF + i];
    }
    static_cast<T*>(u.y)[i] = (T)(act(u.act, a) * b);
    if (u.pre) {
      u.pre[i] = a;
      u.pre[MF + i] = b;
    }
  }
}

template <int DT, int MT>
hipError_t launch(const UnitArgs& u, int splits, float* sums, hipStream_t s) {
  using T = typename Elem<DT>::T;
  constexpr int bytes = kWavesF * MT * 2 * few_frags<DT>() * 4 * kRowS * 4;
  hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(k_unit_few<DT, MT>), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != hipSuccess) return e;
  const int groups = (u.F + few_cols<DT>() - 1) / few_cols<DT>();
  k_unit_few<DT, MT><<<(unsigned)(groups * splits), 64 * kWavesF, bytes, s>>>(u, splits, sums);
  if (splits > 1) {
    const int64_t want = ((int64_t)u.M * u.F + 255) / 256;
    k_unit_sum<T><<<(unsigned)(want < 2048 ? want : 2048), 256, 0, s>>>(u, splits, sums);
  }
  return hipGetLastError();
}

}  // namespace

// Workgroups along the inner axis, 0 where tiles are faster.  Enough for three on every compute unit (for half of that with more
// than 16 rows, whose sums are twice as long), and at least two steps of 32 for each of their waves.  In us, against 64-row tiles:
// bf16, D 2048, F 8192: 1 to 16 rows 19 to 22 (28), 32 rows 25 (28); D 4096, F 1024, 32 rows: 18 (34); but D 512, F 1408, 1 to 32
// rows: 9 to 13 (7), D 1024, F 4096, 16 rows: 12 (11), so not up to D 1024.  f32, whose tiles have six products: D 512, F 1408, 32
// rows: 13 (35); D 2048, F 8192: 35 to 54 (170).  32 rows of the first with 4, 8 and 16 along the inner axis: 25, 32, 45.
int unit_few_splits(int M, int D, int F, int dtype) {
  if (M > 32 || (dtype != SEQ_FP32 && D <= 1024)) return 0;
  const int cols = dtype == SEQ_FP32 ? 64 : 128, groups = (F + cols - 1) / cols;
  const int most = D / (dtype == SEQ_FP32 ? 128 : 256), all = M > 16 ? 384 : 768, want = (all + groups - 1) / groups;
  const int s = want < most ? want : most;
  return s < 1 ? 1 : s > 32 ? 32 : s;
}

hipError_t unit_few(const UnitArgs& u, int splits, float* sums, hipStream_t s) {
  const bool two = u.M > 16;
  if (u.dtype == SEQ_BF16) return two ? launch<SEQ_BF16, 2>(u, splits, sums, s) : launch<SEQ_BF16, 1>(u, splits, sums, s);
  if (u.dtype == SEQ_FP16) return two ? launch<SEQ_FP16, 2>(u, splits, sums, s) : launch<SEQ_FP16, 1>(u, splits, sums, s);
  return two ? launch<SEQ_FP32, 2>(u, splits, sums, s) : launch<SEQ_FP32, 1>(u, splits, sums, s);
}

}  // namespace seq
