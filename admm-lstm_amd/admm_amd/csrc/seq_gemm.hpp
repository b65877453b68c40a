// seq_gemm.hpp -- tiled matrix product on the 16-bit matrix cores, the core of the gated unit's kernels.
//
// C = sum over segments of A_s B_s, A_s [M, K], B_s [K, N], each operand stored along either axis: its tiles go from global
// memory straight into LDS as they are stored (16 bytes a lane, pieces swizzled), and an operand whose inner axis is not the
// contiguous one is transposed on its way out of LDS.  Segments are the two halves of an inner axis (gradient of x) and, for
// f32 operands held as three bf16 planes, the six plane pairs (seq_dev.hpp).
//
// Operands are swapped in the matrix instruction (A = B^T tile), so that a lane ends up with four neighbouring columns of one row
// of C: 8- or 16-byte stores.
#pragma once
#include "seq_dev.hpp"

namespace seq {

constexpr int kBK = 64;   // inner values of an LDS tile

struct GemmArgs {
  const char *a[2][3], *b[2][3];   // [matrix][plane]
  int64_t lda, ldb;                // in elements
  int M, N, K;
  int planes;                      // 1, or 3 (six plane pairs)
  int tiles_m, tiles_n;
};

// sources of loads that lie outside an operand: they have to add nothing
__device__ const u32x4 g_zeros = {0, 0, 0, 0};

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <int DT>
__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
  if constexpr (DT == SEQ_FP16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// An operand's tile: R rows of the outer axis by kBK of the inner one.
// INNER (inner axis contiguous): R rows of 8 pieces, piece c of row r at place c ^ (r & 7).
// else: kBK rows of R / 8 pieces, piece c of row k at place c ^ spread(k): the four rows that a transposing read takes
// together, and the next lanes' four, lie in different banks.
template <int R, bool INNER>
struct TileOf {
  static constexpr int kBytes = R * kBK * 2;
  static constexpr int kP = INNER ? kBK / 8 : R / 8;   // pieces of a row
  __device__ static int spread(int row) {
    if (INNER) return row & 7;
    return (((row & 3) << 1) | ((row >> 3 & 3) << 3)) & (kP - 1);
  }
  // element offset of the fragment with outer rows 16 t + x, inner values 32 s + 8 g..+7
  __device__ static bf16x8 frag(const __bf16* p, int t, int s, int g, int x) {
    if (INNER) {
      const int r = 16 * t + x;
      return *reinterpret_cast<const bf16x8*>(p + r * kBK + 8 * ((4 * s + g) ^ spread(r)));
    }
    const int k = 32 * s + 8 * g + (x >> 2), c = 2 * t + ((x & 3) >> 1), h = 4 * (x & 1);
    const bf16x4 u = tr4(p + k * R + 8 * (c ^ spread(k)) + h), v = tr4(p + (k + 4) * R + 8 * (c ^ spread(k + 4)) + h);
    return __builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  // Loads the tile whose first outer row is o0 and first inner value k0 of a matrix with `outer` and `inner` values: WAVES
  // waves, 1 KB at a time.  Pieces outside come from g_zeros.
  template <int WAVES>
  __device__ static void load(const char* base, int64_t ld, int o0, int k0, int outer, int inner, char* lds, int wave, int lane) {
#pragma unroll
    for (int i = 0; i < kBytes / 1024 / WAVES; ++i) {
      const int at = (i * WAVES + wave) * 64 + lane, row = at / kP, piece = (at % kP) ^ spread(row);
      const int o = INNER ? o0 + row : o0 + 8 * piece, k = INNER ? k0 + 8 * piece : k0 + row;
      const char* src = base + ((INNER ? o : k) * ld + (INNER ? k : o)) * 2;
      glds16(o < outer && k < inner ? src : reinterpret_cast<const char*>(&g_zeros), lds + (i * WAVES + wave) * 1024);
    }
  }
};

// WM x WN waves of MT x NT tiles of 16 x 16.  DUAL: two matrices B side by side (half of the tile's columns each), SPLIT: the
// inner axis is two segments (A and B of matrix 0, then of matrix 1).
template <int DT, int WM, int WN, int MT, int NT, bool AI, bool BI, bool DUAL, bool SPLIT>
struct Gemm {
  static constexpr int kWaves = WM * WN, kThreads = 64 * kWaves;
  static constexpr int BM = WM * MT * 16, BN = WN * NT * 16, BH = DUAL ? BN / 2 : BN;   // BH: columns of C in a tile
  using TA = TileOf<BM, AI>;
  using TB = TileOf<BH, BI>;
  static constexpr int kBuf = TA::kBytes + (DUAL ? 2 : 1) * TB::kBytes;
  static constexpr int kLds = 2 * kBuf;
  static_assert(TA::kBytes % (1024 * kWaves) == 0 && TB::kBytes % (1024 * kWaves) == 0, "whole loads for each wave");

  // the tile of C of this workgroup: neighbouring workgroups (of one XCD: they are dealt out in turn) share columns of B
  // and rows of A in groups of eight row tiles
  __device__ static void place(const GemmArgs& g, int& tm, int& tn) {
    const int n = g.tiles_m * g.tiles_n, id = blockIdx.x;
    const int per = n / 8, extra = n % 8, xcd = id % 8;
    const int at = xcd * per + (xcd < extra ? xcd : extra) + id / 8;
    const int group = 8 * g.tiles_n, first = at / group * 8, rows = g.tiles_m - first < 8 ? g.tiles_m - first : 8;
    tm = first + at % group % rows;
    tn = at % group / rows;
  }

  // b_of: which matrix B (not DUAL, not SPLIT).  acc[i][j]: rows 16 (wm MT + i) + x, columns 16 j' + 4 g..+3 of C
  __device__ static void run(const GemmArgs& g, int tm, int tn, int b_of, char* lds, f32x4 (&acc)[MT][NT]) {
    const int lane = threadIdx.x & 63, wave = wave_id(), x = lane & 15, q = lane >> 4;
    const int wm = wave / WN, wn = wave % WN;
    const int kt = (g.K + kBK - 1) / kBK, terms = g.planes == 1 ? 1 : 6, total = kt * terms * (SPLIT ? 2 : 1);
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto issue = [&](int it, char* buf) {
      const int seg = it / kt, k0 = (it - seg * kt) * kBK, mat = SPLIT ? seg / terms : 0, term = SPLIT ? seg % terms : seg;
      // plane pairs, smallest first: (2,0) (0,2) (1,1) (1,0) (0,1) (0,0)
      const int pa = terms == 1 ? 0 : term == 0 ? 2 : term == 2 || term == 3 ? 1 : 0;
      const int pb = terms == 1 ? 0 : term == 1 ? 2 : term == 2 || term == 4 ? 1 : 0;
      TA::template load<kWaves>(g.a[mat][pa], g.lda, tm * BM, k0, g.M, g.K, buf, wave, lane);
      TB::template load<kWaves>(g.b[SPLIT ? mat : b_of][pb], g.ldb, tn * BH, k0, g.N, g.K, buf + TA::kBytes, wave, lane);
      if (DUAL)
        TB::template load<kWaves>(g.b[1][pb], g.ldb, tn * BH, k0, g.N, g.K, buf + TA::kBytes + TB::kBytes, wave, lane);
    };
    if (total) issue(0, lds);
    for (int it = 0; it < total; ++it) {
      const char* buf = lds + (it & 1) * kBuf;
      vm_wait();
      __syncthreads();
      if (it + 1 < total) issue(it + 1, lds + ((it + 1) & 1) * kBuf);
      const __bf16* At = reinterpret_cast<const __bf16*>(buf);
#pragma unroll
      for (int s = 0; s < kBK / 32; ++s) {
        bf16x8 fb[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const int half = DUAL ? j / (NT / 2) : 0, t = DUAL ? wn * (NT / 2) + j % (NT / 2) : wn * NT + j;
          fb[j] = TB::frag(reinterpret_cast<const __bf16*>(buf + TA::kBytes + half * TB::kBytes), t, s, q, x);
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const bf16x8 fa = TA::frag(At, wm * MT + i, s, q, x);
#pragma unroll
          for (int j = 0; j < NT; ++j) acc[i][j] = mfma16<DT>(fb[j], fa, acc[i][j]);
        }
      }
    }
    mfma_settle();   // the callers store behind bounds checks
  }
};

}  // namespace seq
