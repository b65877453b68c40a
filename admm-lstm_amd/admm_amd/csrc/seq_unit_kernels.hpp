// seq_unit_kernels.hpp -- the gated unit y = act(x Wg) * (x Wu): both projections, the activation and the product in one kernel,
// and its gradients.
//
// Forward: a workgroup forms the same tile of both projections (one tile of x in LDS serves both) and only their product
// leaves it; where gradients follow, the projections a = x Wg and b = x Wu are kept too, in f32 (rounded to 16 bits they would
// cost the gradients more than their own rounding).  Backward: da = dy b act'(a) and db = dy act(a) elementwise, then
// dx = da Wg^T + db Wu^T as one product over both, and dWg = x^T da, dWu = x^T db in one launch (in parts of the rows where the
// layer is narrow, unit_parts).  da and db are held
//   in bf16 as bf16: one rounding more than the result's own (1.4 times its error), for half the products of two planes;
//   in fp16 as two bf16 planes, 16 bits, x and W too (exactly): da has a range of its own, products of three values, and fp16 would
//     lose small gradients and overflow where dx does not.  Three products for one (seq_dev.hpp): all gradients of 8192 x 2048 x
//     8192 take 2.9 ms, with da and db in fp16 1.2 ms;
//   in f32 as three.
//
// Bound by the matrix cores where the layer is wide (12 M D F operations a training step), by the weights where there are few
// rows.  Planes of the operands are formed by a pass before, and 16-bit operands whose rows are not 16-byte aligned are copied to
// padded rows.
//
// 8192 x 2048 x 8192, bf16: forward with the projections kept 557 us (0.99 PFLOP/s; without them 465, 1.18), dx 434 us and dWg, dWu
// 450 us (1.27 and 1.22 PFLOP/s; a large library product reaches 1.41), the elementwise pass 203 us (4.6 TB/s).
//
// Compiled by one source for each type (seq_unit_bf16.hip, _fp16, _fp32), so that they compile side by side.
#pragma once
#include <type_traits>

#include "seq_gemm.hpp"
#include "seq_unit.hpp"
#include "seq_unit_act.hpp"

namespace seq {

namespace {

// rows of n values with the stride ld, as rows of n8 >= n values, the rest zero: 16-bit values as they are (NP = 1), or NP bf16
// planes (`plane` elements apart)
struct CopyJob {
  const void* src;
  __bf16* dst;
  int64_t ld, rows, n8, plane;
  int n;
};
struct CopyJobs {   // one launch for up to three operands: blockIdx.y
  CopyJob job[3];
};
template <int DT, int NP>
__global__ __launch_bounds__(256) void k_unit_copy(CopyJobs jobs) {
  const CopyJob& job = jobs.job[blockIdx.y];
  const void* const src = job.src;
  __bf16* const dst = job.dst;
  const int64_t ld = job.ld, rows = job.rows, n8 = job.n8, plane = job.plane;
  const int n = job.n;
  using T = typename Elem<DT>::T;
  const T* s = static_cast<const T*>(src);
  const int64_t pieces = n8 / 8, all = rows * pieces;
  const bool small = all < (int64_t)1 << 32;
  const bool wide = reinterpret_cast<uintptr_t>(src) % 16 == 0 && ld * (int)sizeof(T) % 16 == 0;
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    const int64_t r = small ? (uint32_t)i / (uint32_t)pieces : i / pieces, p = i - r * pieces;
    const int left = n - (int)(8 * p);
    __bf16* d = dst + r * n8 + 8 * p;
    if constexpr (NP > 1) {
      f32x8 v = {};
      if (left > 0) v = load8(s + r * ld + 8 * p, left, wide);
      bf16x8 pl[NP];
      if constexpr (DT == SEQ_FP32) planes8_whole<NP>(v, pl);
      else planes8<NP>(v, pl);
#pragma unroll
      for (int j = 0; j < NP; ++j) *reinterpret_cast<bf16x8*>(d + j * plane) = pl[j];
    } else {
      const uint16_t* h = reinterpret_cast<const uint16_t*>(s) + r * ld + 8 * p;
      uint16_t v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = j < left ? h[j] : 0;
      *reinterpret_cast<u32x4*>(d) = *reinterpret_cast<const u32x4*>(v);
    }
  }
}

// four neighbouring values of a row, n of them inside it
template <class T>
__device__ __forceinline__ void store4(T* p, f32x4 v, int n, bool wide) {
  typedef T T4 __attribute__((ext_vector_type(4)));
  if (wide && n >= 4) {
    T4 t;
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = (T)v[i];
    *reinterpret_cast<T4*>(p) = t;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) p[i] = (T)v[i];
  }
}

// v[0], v[1] of lanes 2 i and 2 i + 1 (`odd`): afterwards the even lane has both lanes' v[0], the odd one both lanes' v[1]
__device__ __forceinline__ void swap_pairs(f32x4 (&v)[2], int odd) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float send = odd ? v[0][e] : v[1][e];
    const float got = __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, send), 0xb1, 0xf, 0xf, false));
    v[0][e] = odd ? got : v[0][e];
    v[1][e] = odd ? v[1][e] : got;
  }
}

template <int DT, int ACT, int WM, int WN, int MT, int NT, bool KEEP>
__global__ __launch_bounds__(64 * WM * WN) void k_unit(GemmArgs g, typename Elem<DT>::T* y, float* pre, bool wide) {
  using G = Gemm<DT, WM, WN, MT, NT, true, false, true, false>;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63, wave = wave_id(), x = lane & 15, q = lane >> 4, wm = wave / WN, wn = wave % WN;
  int tm, tn;
  G::place(g, tm, tn);
  f32x4 acc[MT][NT];
  G::run(g, tm, tn, 0, lds, acc);
  // Where a wave has two tiles side by side, pairs of lanes swap halves of their results, so that a store holds 32 neighbouring
  // columns of a row (8192 x 2048 x 8192, bf16, projections kept: 690 us without, and 20 us more for whoever reads them)
  constexpr int kPair = NT % 4 == 0 ? 2 : 1;
  const int odd = kPair == 2 ? x & 1 : 0;
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT / 2; j += kPair) {
      const int col = tn * G::BH + 16 * (wn * (NT / 2) + j + odd) + 4 * q, n = g.N - col;
      const int row0 = tm * G::BM + 16 * (wm * MT + i) + (kPair == 2 ? x & ~1 : x);
      f32x4 a[kPair], b[kPair], r[kPair];
#pragma unroll
      for (int p = 0; p < kPair; ++p) {
        a[p] = acc[i][j + p];
        b[p] = acc[i][j + p + NT / 2];
#pragma unroll
        for (int e = 0; e < 4; ++e) r[p][e] = act(ACT, a[p][e]) * b[p][e];
      }
      if constexpr (kPair == 2) {
        swap_pairs(r, odd);
        if (KEEP) {
          swap_pairs(a, odd);
          swap_pairs(b, odd);
        }
      }
#pragma unroll
      for (int p = 0; p < kPair; ++p) {
        const int64_t at = (int64_t)(row0 + p) * g.N + col;
        if (row0 + p >= g.M || n <= 0) continue;
        store4(y + at, r[p], n, wide);
        if (KEEP) {
          store4(pre + at, a[p], n, wide);
          store4(pre + (int64_t)g.M * g.N + at, b[p], n, wide);
        }
      }
    }
}

// the matrix instructions' operands in the products of the gradients: bf16 or planes of it
template <int DT> constexpr int kGradType = DT == SEQ_FP16 ? SEQ_BF16 : DT;

// AI, BI, SPLIT as in Gemm; otherwise blockIdx.y picks the matrix B and the result, and blockIdx.z a part of the inner axis, whose
// sums go to `sums` [part][matrix][M][N] where there are several
template <int DT, int WM, int WN, int MT, int NT, bool AI, bool BI, bool SPLIT>
__global__ __launch_bounds__(64 * WM * WN) void k_unit_gemm(GemmArgs g, typename Elem<DT>::T* c0, typename Elem<DT>::T* c1, float* sums, bool wide) {
  using G = Gemm<kGradType<DT>, WM, WN, MT, NT, AI, BI, false, SPLIT>;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63, wave = wave_id(), x = lane & 15, q = lane >> 4, wm = wave / WN, wn = wave % WN;
  int tm, tn;
  G::place(g, tm, tn);
  f32x4 acc[MT][NT];
  if constexpr (!SPLIT && !AI && !BI) {
    if (gridDim.z > 1) {
      const int tiles = (g.K + kBK - 1) / kBK, first = (int)((int64_t)tiles * blockIdx.z / gridDim.z), end = (int)((int64_t)tiles * (blockIdx.z + 1) / gridDim.z);
      const int64_t k0 = (int64_t)first * kBK;
#pragma unroll
      for (int p = 0; p < 3; ++p) {
        g.a[0][p] += k0 * g.lda * 2;
        g.b[0][p] += k0 * g.ldb * 2;
        g.b[1][p] += k0 * g.ldb * 2;
      }
      g.K = (int)((int64_t)end * kBK < g.K ? (int64_t)end * kBK - k0 : g.K - k0);
    }
  }
  G::run(g, tm, tn, blockIdx.y, lds, acc);
  typename Elem<DT>::T* c = blockIdx.y ? c1 : c0;
  if (sums) sums += (2 * (int64_t)blockIdx.z + blockIdx.y) * g.M * g.N;
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int row = tm * G::BM + 16 * (wm * MT + i) + x;
    if (row >= g.M) continue;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int col = tn * G::BN + 16 * (wn * NT + j) + 4 * q, n = g.N - col;
      if (n <= 0) continue;
      if (sums) store4(sums + (int64_t)row * g.N + col, acc[i][j], n, wide);
      else store4(c + (int64_t)row * g.N + col, acc[i][j], n, wide);
    }
  }
}

__device__ __forceinline__ f32x8 once8(const float* p, int n, bool wide) {
  if (!(wide && n >= 8)) return load8(p, n, false);
  const f32x4 a = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(p)), b = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(p + 4));
  return cat8(a, b);
}
// the parts' sums [part][matrix][n], added up in order
template <class T>
__global__ __launch_bounds__(256) void k_unit_join(const float* sums, int parts, int64_t n, T* c0, T* c1) {
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < 2 * n; i += (int64_t)gridDim.x * 256) {
    float v = 0.f;
#pragma unroll 8
    for (int p = 0; p < parts; ++p) v += sums[2 * n * p + i];
    (i < n ? c0 : c1 - n)[i] = (T)v;
  }
}

// da = dy b act'(a), db = dy act(a), as rows of F8 values, in bf16 planes
template <int DT, int ACT>
__global__ __launch_bounds__(256) void k_unit_back(UnitArgs u) {
  using T = typename Elem<DT>::T;
  const int64_t pieces = u.F8 / 8, all = u.M * pieces, plane = u.M * u.F8, MF = (int64_t)u.M * u.F;
  const T* dy = static_cast<const T*>(u.dy);
  const bool small = all < (int64_t)1 << 32;   // 64-bit division takes longer than the rest
  const bool wide = u.F % 8 == 0, wide_dy = reinterpret_cast<uintptr_t>(dy) % 16 == 0 && u.dy_ld * (int)sizeof(T) % 16 == 0;
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    const int64_t r = small ? (uint32_t)i / (uint32_t)pieces : i / pieces, p = i - r * pieces;
    const int left = u.F - (int)(8 * p);
    const f32x8 a = once8(u.pre + r * u.F + 8 * p, left, wide), b = once8(u.pre + MF + r * u.F + 8 * p, left, wide);
    const f32x8 d = load8(dy + r * u.dy_ld + 8 * p, left, wide_dy);
    f32x8 da, db;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float f, df;
      act_grad(ACT, a[j], f, df);
      da[j] = j < left ? d[j] * b[j] * df : 0.f;
      db[j] = j < left ? d[j] * f : 0.f;
    }
    const int64_t at = r * u.F8 + 8 * p;
    constexpr int NP = Elem<DT>::kPlanes;
    bf16x8 pa[NP], pb[NP];
    if constexpr (DT == SEQ_FP32) {
      planes8_whole<NP>(da, pa);
      planes8_whole<NP>(db, pb);
    } else {
      planes8<NP>(da, pa);
      planes8<NP>(db, pb);
    }
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      *reinterpret_cast<bf16x8*>(reinterpret_cast<__bf16*>(u.dap) + j * plane + at) = pa[j];
      *reinterpret_cast<bf16x8*>(reinterpret_cast<__bf16*>(u.dbp) + j * plane + at) = pb[j];
    }
  }
}

unsigned blocks_for(int64_t n) {
  const int64_t want = (n + 255) / 256;
  return (unsigned)(want < 256 * 32 ? want : 256 * 32);
}

template <int DT, int NP>
void copies(const UnitArgs& u, hipStream_t s) {
  CopyJobs jobs = {};
  int count = 0;
  int64_t most = 0;
  auto add = [&](const void* src, int64_t ld, int64_t rows, int n, int64_t n8, char* dst) {
    jobs.job[count++] = {src, reinterpret_cast<__bf16*>(dst), ld, rows, n8, rows * n8, n};
    most = rows * n8 / 8 > most ? rows * n8 / 8 : most;
  };
  if (u.copy_x) add(u.x, u.x_ld, u.M, u.D, u.D8, u.xp);
  if (u.copy_w) {
    add(u.wg, u.w_ld, u.D, u.F, u.F8, u.wgp);
    add(u.wu, u.wu_ld, u.D, u.F, u.F8, u.wup);
  }
  if (most) k_unit_copy<DT, NP><<<dim3(blocks_for(most), (unsigned)count), 256, 0, s>>>(jobs);
}

template <class F>
hipError_t lds_for(F* f, int bytes) {
  return hipFuncSetAttribute(reinterpret_cast<const void*>(f), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

// planes of an operand: the tensor itself, or its copy
void planes(const char* (&p)[3], bool copied, const void* x, const char* copy, int64_t plane) {
  for (int i = 0; i < 3; ++i) p[i] = copied ? copy + i * plane * 2 : static_cast<const char*>(x);
}

// f of the activation as a constant: a tile's 64 activations a lane are straight code, three times as long with all of them in it
template <class F>
hipError_t for_act(int act, F&& f) {
  return act == SEQ_SILU ? f(std::integral_constant<int, SEQ_SILU>()) : act == SEQ_GELU ? f(std::integral_constant<int, SEQ_GELU>())
                                                                                     : f(std::integral_constant<int, SEQ_SIGMOID>());
}

void tiles(GemmArgs& g, int BM, int BN) {
  g.tiles_m = (g.M + BM - 1) / BM;
  g.tiles_n = (g.N + BN - 1) / BN;
}

template <int DT, int WM, int WN, int MT, int NT>
hipError_t launch_unit(GemmArgs g, const UnitArgs& u, hipStream_t s) {
  using T = typename Elem<DT>::T;
  using G = Gemm<DT, WM, WN, MT, NT, true, false, true, false>;
  tiles(g, G::BM, G::BH);
  const bool wide = u.F % 4 == 0;
  auto go = [&](auto* f) {
    const hipError_t e = lds_for(f, G::kLds);
    if (e == hipSuccess) f<<<(unsigned)(g.tiles_m * g.tiles_n), G::kThreads, G::kLds, s>>>(g, static_cast<T*>(u.y), u.pre, wide);
    return e;
  };
  return for_act(u.act, [&](auto act) {
    constexpr int A = decltype(act)::value;
    return u.pre ? go(k_unit<DT, A, WM, WN, MT, NT, true>) : go(k_unit<DT, A, WM, WN, MT, NT, false>);
  });
}

template <int DT, int WM, int WN, int MT, int NT, bool AI, bool BI, bool SPLIT>
hipError_t launch_gemm(GemmArgs g, void* c0, void* c1, hipStream_t s, int parts = 1, float* sums = nullptr) {
  using T = typename Elem<DT>::T;
  using G = Gemm<kGradType<DT>, WM, WN, MT, NT, AI, BI, false, SPLIT>;
  tiles(g, G::BM, G::BN);
  auto* f = k_unit_gemm<DT, WM, WN, MT, NT, AI, BI, SPLIT>;
  const hipError_t e = lds_for(f, G::kLds);
  if (e != hipSuccess) return e;
  f<<<dim3((unsigned)(g.tiles_m * g.tiles_n), c1 ? 2 : 1, (unsigned)parts), G::kThreads, G::kLds, s>>>(
      g, static_cast<T*>(c0), static_cast<T*>(c1), sums, g.N % 4 == 0);
  return hipSuccess;
}

template <int DT>
hipError_t forward(const UnitArgs& u, hipStream_t s) {
  constexpr int np = DT == SEQ_FP32 ? 3 : 1;
  copies<DT, np>(u, s);
  GemmArgs g = {};
  g.M = u.M, g.N = u.F, g.K = u.D;
  g.planes = np;
  g.lda = u.copy_x ? u.D8 : u.x_ld;
  g.ldb = u.copy_w ? u.F8 : u.w_ld;
  planes(g.a[0], u.copy_x, u.x, u.xp, u.M * u.D8);
  planes(g.b[0], u.copy_w, u.wg, u.wgp, u.D * u.F8);
  planes(g.b[1], u.copy_w, u.wu, u.wup, u.D * u.F8);
  const int tile = tile_for(u.M, 2 * (int64_t)u.F, true, 1, nullptr);
  const hipError_t e = tile == 0   ? launch_unit<DT, 2, 4, 8, 4>(g, u, s)
                       : tile == 1 ? launch_unit<DT, 2, 2, 4, 4>(g, u, s)
                       : tile == 2 ? launch_unit<DT, 2, 2, 2, 2>(g, u, s) : launch_unit<DT, 2, 4, 6, 4>(g, u, s);
  return e != hipSuccess ? e : hipGetLastError();
}

template <int DT>
hipError_t backward(const UnitArgs& u, hipStream_t s) {
  constexpr int np = Elem<DT>::kPlanes;
  hipError_t e = !u.M ? hipSuccess : for_act(u.act, [&](auto act) {
    k_unit_back<DT, decltype(act)::value><<<blocks_for(u.M * u.F8 / 8), 256, 0, s>>>(u);
    return hipGetLastError();
  });
  if (e != hipSuccess) return e;
  copies<DT, np>(u, s);
  if (u.dx) {
    GemmArgs g = {};
    g.M = u.M, g.N = u.D, g.K = u.F;
    g.planes = np;
    g.lda = u.F8;
    g.ldb = u.copy_w ? u.F8 : u.w_ld;
    planes(g.a[0], true, nullptr, u.dap, u.M * u.F8);
    planes(g.a[1], true, nullptr, u.dbp, u.M * u.F8);
    planes(g.b[0], u.copy_w, u.wg, u.wgp, u.D * u.F8);
    planes(g.b[1], u.copy_w, u.wu, u.wup, u.D * u.F8);
    const int tile = tile_for(u.M, u.D, true, 1, nullptr);
    e = tile == 0   ? launch_gemm<DT, 2, 4, 8, 4, true, true, true>(g, u.dx, nullptr, s)
        : tile == 1 ? launch_gemm<DT, 2, 2, 4, 4, true, true, true>(g, u.dx, nullptr, s)
        : tile == 2 ? launch_gemm<DT, 2, 2, 2, 2, true, true, true>(g, u.dx, nullptr, s)
                    : launch_gemm<DT, 2, 4, 6, 4, true, true, true>(g, u.dx, nullptr, s);
    if (e != hipSuccess) return e;
  }
  if (u.dwg) {
    GemmArgs g = {};
    g.M = u.D, g.N = u.F, g.K = u.M;
    g.planes = np;
    g.lda = u.copy_x ? u.D8 : u.x_ld;
    g.ldb = u.F8;
    planes(g.a[0], u.copy_x, u.x, u.xp, u.M * u.D8);
    planes(g.b[0], true, nullptr, u.dap, u.M * u.F8);
    planes(g.b[1], true, nullptr, u.dbp, u.M * u.F8);
    const UnitParts way = unit_parts(u.M, u.D, u.F, u.dtype);
    float* const sums = way.parts > 1 ? u.sums : nullptr;
    e = way.tile == 0   ? launch_gemm<DT, 2, 4, 8, 4, false, false, false>(g, u.dwg, u.dwu, s, way.parts, sums)
        : way.tile == 1 ? launch_gemm<DT, 2, 2, 4, 4, false, false, false>(g, u.dwg, u.dwu, s, way.parts, sums)
                        : launch_gemm<DT, 2, 2, 2, 2, false, false, false>(g, u.dwg, u.dwu, s, way.parts, sums);
    using T = typename Elem<DT>::T;
    const int64_t n = (int64_t)u.D * u.F;
    if (e == hipSuccess && sums) k_unit_join<T><<<blocks_for(2 * n), 256, 0, s>>>(sums, way.parts, n, static_cast<T*>(u.dwg), static_cast<T*>(u.dwu));
    if (e != hipSuccess) return e;
  }
  return hipGetLastError();
}

}  // namespace
}  // namespace seq
