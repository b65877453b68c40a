// seq_gemm.hpp -- tiled matrix product on the 16-bit matrix cores, the core of the gated unit's kernels.
//
// C = sum over segments of A_s B_s, A_s [M, K], B_s [K, N], each operand stored along either axis: its tiles go from global
// memory straight into LDS as they are stored (16 bytes a lane, pieces swizzled), and an operand whose inner axis is not the
// contiguous one is transposed on its way out of LDS.  Segments are the two halves of an inner axis (gradient of x) and the pairs
// of planes (seq_dev.hpp): six for f32 operands held as three bf16 planes, three for two planes (gradients of fp16).
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
  int planes;                      // 1, 2 (three plane pairs) or 3 (six)
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
template <int R, bool INNER, int WAVES>
struct TileOf {
  static constexpr int kBytes = R * kBK * 2;
  static constexpr int kP = INNER ? kBK / 8 : R / 8;         // pieces of a row
  static constexpr int kLoads = kBytes / 1024 / WAVES;       // of 1 KB, for each wave
  __device__ static int spread(int row) {
    if (INNER) return row & 7;
    return (((row & 3) << 1) | ((row >> 3 & 3) << 3)) & (kP - 1);
  }
  // Offsets of the lane's pieces from the tile's first value.  Outer values outside the matrix are taken from the last ones
  // inside (what they make is not stored), so that only the last tile along the inner axis needs a look at its pieces.
  uint32_t off[kLoads];
  __device__ void place(int64_t ld, int o0, int outer, int wave, int lane) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int at = (i * WAVES + wave) * 64 + lane, row = at / kP, piece = (at % kP) ^ spread(row);
      const int last = INNER ? outer - 1 - o0 : (outer + 7) / 8 * 8 - 8 - o0;
      const int o = INNER ? row : 8 * piece, k = INNER ? 8 * piece : row, oc = o < last ? o : last;
      off[i] = (uint32_t)(((INNER ? oc : k) * ld + (INNER ? k : oc)) * 2);
    }
  }
  // base: the matrix at outer value o0, inner value k0 (a scalar); inner: values left from k0 on
  __device__ void load(const char* base, int inner, char* lds, int wave, int lane) const {
    if (inner >= kBK) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) glds16(base + off[i], lds + (i * WAVES + wave) * 1024);
    } else {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int at = (i * WAVES + wave) * 64 + lane, row = at / kP, k = INNER ? 8 * ((at % kP) ^ spread(row)) : row;
        glds16(k < inner ? base + off[i] : reinterpret_cast<const char*>(&g_zeros), lds + (i * WAVES + wave) * 1024);
      }
    }
  }
};

// Where a lane finds the fragments (outer rows 16 t + x, inner values 32 s + 8 g..+7) of T tiles from t0 on
template <int R, bool INNER, int T>
struct FragsOf {
  int at[INNER ? 2 : T];
  __device__ FragsOf(int t0, int g, int x) {
    if (INNER) {
#pragma unroll
      for (int s = 0; s < 2; ++s) at[s] = ((16 * t0 + x) * kBK + 8 * ((4 * s + g) ^ (x & 7))) * 2;
    } else {
      const int k = 8 * g + (x >> 2);   // spread() is the same for rows k, k + 4 and k + 32
#pragma unroll
      for (int t = 0; t < T; ++t)
        at[t] = (k * R + 8 * ((2 * (t0 + t) + ((x & 3) >> 1)) ^ TileOf<R, false, 1>::spread(k)) + 4 * (x & 1)) * 2;
    }
  }
  __device__ bf16x8 get(const char* lds, int t, int s) const {
    if (INNER) return *reinterpret_cast<const bf16x8*>(lds + at[s] + t * 16 * kBK * 2);
    const __bf16* p = reinterpret_cast<const __bf16*>(lds + at[t] + s * 32 * R * 2);
    const bf16x4 u = tr4(p), v = tr4(p + 4 * R);
    return __builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7);
  }
};

// WM x WN waves of MT x NT tiles of 16 x 16.  DUAL: two matrices B side by side (half of the tile's columns each), SPLIT: the
// inner axis is two segments (A and B of matrix 0, then of matrix 1).
template <int DT, int WM, int WN, int MT, int NT, bool AI, bool BI, bool DUAL, bool SPLIT>
struct Gemm {
  static constexpr int kWaves = WM * WN, kThreads = 64 * kWaves;
  static constexpr int BM = WM * MT * 16, BN = WN * NT * 16, BH = DUAL ? BN / 2 : BN;   // BH: columns of C in a tile
  using TA = TileOf<BM, AI, kWaves>;
  using TB = TileOf<BH, BI, kWaves>;
  static constexpr int kBuf = TA::kBytes + (DUAL ? 2 : 1) * TB::kBytes;
  static constexpr int kLds = 2 * kBuf;
  // The next tile's loads before the first or the second half of the products.  Before the second they do not hold up the first
  // half's LDS reads: the forward of f32 operands, 2048 x 2048 x 4096, takes 335 us for 363; but they have less time to arrive: dx
  // of 8192 x 2048 x 8192, bf16, would take 525 for 505, the forward 641 for 630, and products of few tiles up to a quarter more.
  static constexpr int kIssueAt = DUAL && DT == SEQ_FP32 ? 1 : 0;
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
    const int kt = (g.K + kBK - 1) / kBK, terms = g.planes * (g.planes + 1) / 2, total = kt * terms * (SPLIT ? 2 : 1);
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    TA la;
    TB lb;
    la.place(g.lda, tm * BM, g.M, wave, lane);
    lb.place(g.ldb, tn * BH, g.N, wave, lane);
    const int64_t a0 = (AI ? (int64_t)tm * BM * g.lda : (int64_t)tm * BM) * 2, b0 = (BI ? (int64_t)tn * BH * g.ldb : (int64_t)tn * BH) * 2;
    const int64_t a_step = (AI ? kBK : kBK * g.lda) * 2, b_step = (BI ? kBK : kBK * g.ldb) * 2;
    int seg = 0, left = 0;   // segment, inner values left in it
    const char *pa = nullptr, *pb = nullptr, *pb1 = nullptr;
    auto issue = [&](char* buf) {
      if (left <= 0) {
        const int mat = SPLIT ? seg / terms : 0, term = (SPLIT ? seg % terms : seg) + 6 - terms;
        // plane pairs, smallest first: (2,0) (0,2) (1,1) (1,0) (0,1) (0,0); of two planes the last three, of one the last
        const int ia = term == 0 ? 2 : term == 2 || term == 3 ? 1 : 0;
        const int ib = term == 1 ? 2 : term == 2 || term == 4 ? 1 : 0;
        pa = g.a[mat][ia] + a0;
        pb = g.b[SPLIT ? mat : b_of][ib] + b0;
        pb1 = g.b[1][ib] + b0;
        left = g.K;
        ++seg;
      }
      la.load(pa, left, buf, wave, lane);
      lb.load(pb, left, buf + TA::kBytes, wave, lane);
      if (DUAL) lb.load(pb1, left, buf + TA::kBytes + TB::kBytes, wave, lane);
      pa += a_step, pb += b_step, pb1 += b_step, left -= kBK;
    };
    const FragsOf<BM, AI, MT> fa(wm * MT, q, x);
    constexpr int TN = DUAL ? NT / 2 : NT;
    const FragsOf<BH, BI, TN> fb(wn * TN, q, x);
    if (total) issue(lds);
    for (int it = 0; it < total; ++it) {
      const char* buf = lds + (it & 1) * kBuf;
      vm_wait();
      __syncthreads();
#pragma unroll
      for (int s = 0; s < kBK / 32; ++s) {
        if (s == kIssueAt && it + 1 < total) issue(lds + ((it + 1) & 1) * kBuf);
        bf16x8 b[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) b[j] = fb.get(buf + TA::kBytes + (DUAL ? j / TN * TB::kBytes : 0), DUAL ? j % TN : j, s);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const bf16x8 a = fa.get(buf, i, s);
#pragma unroll
          for (int j = 0; j < NT; ++j) acc[i][j] = mfma16<DT>(b[j], a, acc[i][j]);
        }
      }
    }
    mfma_settle();   // the callers store behind bounds checks
  }
};

}  // namespace seq
