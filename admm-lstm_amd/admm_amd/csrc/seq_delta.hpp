// seq_delta.hpp -- shapes, work memory and row addressing of the gated delta rule's kernels.
//
// The rule in chunks of 64 rows (G_i: the sum of g up to row i of the chunk; D_ij = exp(G_i - G_j) for i >= j, else 0):
//   the u of a chunk's rows solve  u_i + beta_i sum_{j < i} D_ij (k_i . k_j) u_j = beta_i (v_i - exp(G_i) S^T k_i),
//   so with A the strictly lower part of beta_i D_ij (k_i . k_j) and X = (I + A)^-1
//     u = X (beta (v - exp(G) K S)),   o = scale exp(G) Q S + P u with P_ij = scale D_ij (q_i . k_j),
//     S <- exp(G_63) S + K^T (exp(G_63 - G) u).
// X and P depend on q, k, g, beta alone: k_delta_prep forms them for all chunks at once.  What is left to do in order
// is four products a chunk, and every column of S, v, u and o goes its own way through them: a wave owns 16 columns
// from the first chunk to the last and exchanges nothing with the others (k_delta_scan).
// A value that is not finite would pass backwards through zeros of X and P (0 * NaN), to rows before its own.  So rows
// of k, g or beta from the first that is not finite are left out of X and P, and values of v out of the products; what
// they make NaN in truth, o from that row on and the state, is set to NaN afterwards.
#pragma once
#include "seq_dev.hpp"

namespace seq {

constexpr int kC = 64;          // rows of a chunk
// X and P are lower triangular: a plane is rows 0..31 of 32 values, then rows 32..63 of 64
constexpr int kTri = 32 * 32 + 32 * 64;
__device__ __forceinline__ int tri_at(int r, int c) { return r < 32 ? tile_at<32>(r, c) : 32 * 32 + tile_at<64>(r - 32, c); }

constexpr float kMinG = -200.f;  // exp(g) is zero in f32 far above this: lower values (-inf too) act the same

// SAVE: gradients follow, and f32 gradients (of g, beta and the state) are made of P too
template <int DT, int KP, bool SAVE>
struct DeltaShape {
  static constexpr int NP = Elem<DT>::kPlanes;
  static constexpr int NO = DT == SEQ_FP32 ? 3 : 2;    // planes of what only values of type DT are made of
  static constexpr int NPP = SAVE ? 3 : NO;            // planes of P
  static constexpr int kTile = kC * KP;                // values of one plane of K or Q
  static constexpr int kKQ = 2 * NP * kTile * 2;       // bytes of a chunk's K planes and Q planes
  static constexpr int kXP = (3 + NPP) * kTri * 2;     // bytes of a chunk's X and P planes
  static constexpr int kVec = 4 * kC * 4;              // exp(G); exp(G_63 - G); beta; exp(G_63), first row not finite
  static constexpr int kStage = kKQ + kXP + kVec;
};

// row ranges of the sequences and their chunks' places in the work memory
struct DeltaRows {
  int64_t T, N;
  int64_t per;          // chunks of a sequence (offsets == NULL)
  const void* off;
  int off64;
  __device__ int64_t at(int64_t n) const {
    const int64_t o = off64 ? static_cast<const int64_t*>(off)[n] : static_cast<const int32_t*>(off)[n];
    return o < 0 ? 0 : o > T ? T : o;
  }
  // first row (counted from the batch row's, or from the packed rows' first), rows, first chunk
  __device__ void range(int64_t n, int64_t& begin, int64_t& len, int64_t& chunk) const {
    if (!off) {
      begin = 0, len = T, chunk = n * per;
    } else {
      begin = at(n);
      const int64_t e = at(n + 1);
      len = e > begin ? e - begin : 0;
      chunk = begin / kC + n;   // no two sequences' chunks meet: a sequence of L rows has at most L / 64 + 1
    }
  }
  __device__ int64_t batch(int64_t n) const { return off ? 0 : n; }
  // the sequence of chunk c of the work memory
  __device__ int64_t find(int64_t c) const {
    if (!off) return c / per;
    int64_t lo = 0, hi = N - 1;
    while (lo < hi) {
      const int64_t m = (lo + hi + 1) >> 1;
      if (at(m) / kC + m <= c) lo = m; else hi = m - 1;
    }
    return lo;
  }
};

struct DeltaArgs {
  DeltaRows rows;
  int Hk, Hv, K, V, VP;   // VP: V rounded up to 16
  float scale;
  bool wide_q, wide_k;
  const void *q, *k, *v;
  const float *g, *beta;
  int64_t qs[3], ks[3], vs[3], gs[3], bs[3];
  const float* initial;
  int64_t chunks;
  char* kq;      // [chunk][Hk] planes of K, then of Q
  char* xp;      // [chunk][Hv] planes of X, then of P
  char* vec;     // [chunk][Hv]
  float* s0;     // [chunk][Hv][KP][VP] the state at each chunk's start (saved = 1)
  float* u;      // [chunk][Hv][64][VP]
  void* o;
  float* final;
};

struct DeltaGradArgs {
  DeltaArgs f;
  float* ds;     // [chunk][Hv][KP][VP] gradient of the state at each chunk's end
  float* dr;     // [chunk][Hv][64][VP] gradient of beta (v - exp(G) K S)
  float *dq32, *dk32;   // [rows][Hv][K]: shares of the value heads where Hv > Hk
  const void* d_o;
  const float* d_final;
  void *dq, *dk, *dv;
  float *dg, *dbeta, *d_initial;
};

}  // namespace seq
