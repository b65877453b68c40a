// seq_delta.hpp -- shapes, work memory and row addressing of the gated delta rule's kernels.
//
// The rule in chunks of C = 64 rows (32 where no sequence is longer).  G_i is the sum of g up to row i of the chunk, G the
// whole chunk's, D_ij = exp(G_i - G_j) for i >= j, else 0:
//   the u of a chunk's rows solve  u_i + beta_i sum_{j < i} D_ij (k_i . k_j) u_j = beta_i (v_i - exp(G_i) S^T k_i),
//   so with A the strictly lower part of beta_i D_ij (k_i . k_j) and X = (I + A)^-1
//     u = X (beta (v - exp(G_i) K S)),   o = scale exp(G_i) Q S + P u with P_ij = scale D_ij (q_i . k_j),
//     S <- exp(G) S + K^T (exp(G - G_i) u).
// X and P depend on q, k, g, beta alone: k_delta_prep forms them for all chunks at once.  What is left to do in order is
// four products a chunk (k_delta_scan), in which every column of S, v, u and o goes its own way.
// A value that is not finite would pass backwards through zeros of X and P (0 * NaN), to rows before its own.  So rows
// of k, g or beta from the first that is not finite are left out of X and P, and values of v out of the products; what
// they make NaN in truth, o from that row on and the state, is set to NaN afterwards.
//
// v_mfma_f32_16x16x32_bf16: lane l = 16 g + x holds row (column) x of A (B), inner values 8 g..8 g + 7, and column x, rows
// 4 g..4 g + 3 of the result.  Result tile t stands for rows perm_row(t, m), m = 0..15: the tiles 2 s and 2 s + 1 then give
// lane l rows 32 s + 8 g..+7 of its column, which is an operand B of the next product as it stands.
//
// The A operands lie in the work memory as the matrix instructions take them ("fragments": 64 lanes of 16 bytes, 1 KB a
// plane), written once by k_delta_prep: a wave loads them with coalesced 16-byte loads straight into registers.
#pragma once
#include "seq_dev.hpp"

namespace seq {

constexpr float kMinG = -200.f;  // exp(g) is zero in f32 far above this: lower values (-inf too) act the same

// SAVE: gradients follow, and f32 gradients (of g, beta and the state) are made of P too
template <int DT, int KP, int C_, bool SAVE>
struct DeltaShape {
  static constexpr int C = C_;
  static constexpr int NP = Elem<DT>::kPlanes;
  static constexpr int NO = DT == SEQ_FP32 ? 3 : 2;    // planes of what only values of type DT are made of
  static constexpr int NPP = SAVE ? 3 : NO;            // planes of P
  static constexpr int RT = C / 16, KT = KP / 16;      // tiles of 16 rows of a chunk, of the state
  static constexpr int KS = KP / 32, CS = C / 32;      // inner steps of 32 over K, over the chunk's rows
  static constexpr int TRI = C == 64 ? 6 : 2;          // fragments of a lower triangular C x C matrix
  // fragments (of NP planes) of a chunk and query/key head: K by rows, Q by rows, K^T and (SAVE) Q^T by state tiles
  static constexpr int fK = 0, fQ = RT * KS, fKT = 2 * RT * KS, fQT = fKT + KT * CS, fEnd = SAVE ? fQT + KT * CS : fQT;
  static constexpr int kKQ = fEnd * NP * 1024;
  // planes of a chunk and value head: X, P, and (SAVE) X^T, P^T
  static constexpr int pX = 0, pP = 3 * TRI, pXT = pP + NPP * TRI, pPT = pXT + 3 * TRI, pEnd = SAVE ? pPT + 3 * TRI : pXT;
  static constexpr int kXP = pEnd * 1024;
};
constexpr int kVec = 4 * 64 * 4;   // exp(G_i); exp(G - G_i); beta; exp(G), first row that is not finite

__device__ __forceinline__ int perm_row(int t, int m) { return 32 * (t >> 1) + 8 * (m >> 2) + 4 * (t & 1) + (m & 3); }
// fragment of a lower triangular matrix: tile t of its rows, inner step s <= t / 2; of its transpose: t of its columns, s >= t / 2
__device__ constexpr int tri_frag(int t, int s) { return t < 2 ? t : 2 + 2 * (t - 2) + s; }
__device__ constexpr int tri_frag_t(int t, int s) { return t < 2 ? 2 * t + s : t + 2; }   // (C = 64)

// row ranges of the sequences and their chunks' places in the work memory
struct DeltaRows {
  int C;
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
      chunk = begin / C + n;   // no two sequences' chunks meet: a sequence of L rows has at most L / C + 1
    }
  }
  __device__ int64_t batch(int64_t n) const { return off ? 0 : n; }
  // the sequence of chunk c of the work memory
  __device__ int64_t find(int64_t c) const {
    if (!off) return c / per;
    int64_t lo = 0, hi = N - 1;
    while (lo < hi) {
      const int64_t m = (lo + hi + 1) >> 1;
      if (at(m) / C + m <= c) lo = m; else hi = m - 1;
    }
    return lo;
  }
};

// columns of a state that a workgroup of the single-token kernel takes (seq_step.hip has the measurements)
inline int step_cols(int64_t heads, int V) { return V < 96 || heads < 1024 ? 32 : 128; }

struct DeltaOutside {
  int n;
  void* p[5];
  int64_t row[5];   // bytes of a row
};

struct DeltaArgs {
  DeltaRows rows;
  int Hk, Hv, K, V, VP;   // VP: V rounded up to 16
  float scale;
  bool wide_q, wide_k;
  bool wide_cols;         // two column tiles a workgroup
  const void *q, *k, *v;
  const float *g, *beta;
  int64_t qs[3], ks[3], vs[3], gs[3], bs[3];
  const float* initial;
  int64_t chunks;
  char* kq;      // [chunk][Hk] fragments
  char* xp;      // [chunk][Hv] fragments
  char* vec;     // [chunk][Hv]
  float* s0;     // [chunk][Hv][KP][VP] the state at each chunk's start (SAVE)
  float* u;      // [chunk][Hv][C][VP]
  void* o;
  float* final;
};

struct DeltaGradArgs {
  DeltaArgs f;
  float* ds;     // [chunk][Hv][KP][VP] gradient of the state at each chunk's end
  float* dr;     // [chunk][Hv][C][VP] gradient of beta (v - exp(G_i) K S)
  float *dq32, *dk32;   // [rows][Hv][K]: shares of the value heads where Hv > Hk
  const void* d_o;
  const float* d_final;
  void *dq, *dk, *dv;
  float *dg, *dbeta, *d_initial;
};

}  // namespace seq
