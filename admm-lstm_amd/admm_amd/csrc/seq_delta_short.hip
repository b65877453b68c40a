// seq_delta_short.hip -- the gated delta rule for sequences of at most 32 rows: forward and backward in one kernel each.
//
// One chunk is the whole sequence (seq_delta.hpp and seq_delta_grad.hip have the formulas), so nothing has to go through work
// memory: a workgroup takes one sequence and value head, forms X and P in LDS, and its four waves take 16 columns each of S, v, u
// and o through all products at once.  The backward kernel forms all that again (reading q, k, v and the initial state a second
// time costs less than writing and reading it back) and goes on to the gradients; what it sums over the value axis passes
// through LDS 64 columns at a time.
//
// Bound by the latency of the chain of products, two to four waves on a SIMD; what had cost most was registers spilled to
// scratch memory (offsets that the compiler worked out before the loops).  f32, forward and forward with backward, in us, against
// the kernels over chunks of 32 rows with their work memory: 2048 sequences of 32 rows, 4 heads of 64 x 64: 144 and 550 (321 and
// 1024); 1024 of 32 rows, 4 heads of 128 x 128: 210 and 946 (493 and 1565); 256 of them, V = 512: 184 and 736 (405 and 1333);
// 1024 of 8 rows: 184 and 887 (475 and 1517); 8 sequences: 10 (14).  At memory's rate the first would take 50 and 210; at the clocks
// of a program that goes on it takes 135 and 523.
#include "seq_delta_dev.hpp"

namespace seq {
namespace {

constexpr int kS = 32;          // rows of the chunk
constexpr int kSld = kS + 4;    // row length of the f32 tiles
constexpr int kMat = kS * kS;   // values of a plane of X, P, m or n

template <int DT, int KP, bool GRAD>
struct ShortLds {
  static constexpr int NP = Elem<DT>::kPlanes, NO = DT == SEQ_FP32 ? 3 : 2, NPP = GRAD ? 3 : NO, KT = KP / 16, KS = KP / 32;
  static constexpr int kTile = kS * KP, kCol = 64 * kS;   // values of a plane of K; of 64 columns of u, dR or do
  static constexpr int most(int a, int b) { return a > b ? a : b; }
  // K and Q; X and P; the decays; A and X in f32 and, when these are no longer read, the columns of u, dR and do, then m and n
  static constexpr int kq = 0, xp = kq + 2 * NP * kTile * 2, vec = xp + (3 + NPP) * kMat * 2, A = vec + 8 * kS * 4, X = A + kS * kSld * 4,
                       cols = A, sums = A + most(2 * kS * kSld * 4, GRAD ? most((6 + NP) * kCol * 2, 2 * NO * kMat * 2) : 0),
                       bytes = sums + (GRAD ? (4 * 4 * kS + 3 * 3 * 16 + 8) * 4 : 0);
};

struct ShortVec {   // in LDS
  float ghi[kS], glo[kS], into[kS], left[kS], beta[kS], all, bad, pad[kS - 2];
  int kbad[kS];
};

// K and Q as planes, X and P as planes and the decays, all in LDS; kk and qk: k_i . k_j and q_i . k_j of the wave's tile, rows
// 16 ti + 4 g.., columns 16 tj + x (waves 0..2: tiles (0, 0), (1, 0), (1, 1))
template <int DT, int KP, bool GRAD>
__device__ __forceinline__ void short_prep(const DeltaArgs& a, int64_t n, int h, int hk, char* lds, f32x4& kk, f32x4& qk) {
  using L = ShortLds<DT, KP, GRAD>;
  using T = typename Elem<DT>::T;
  constexpr int NP = L::NP, kTile = L::kTile;
  __bf16* const kq = reinterpret_cast<__bf16*>(lds);
  float* const A = reinterpret_cast<float*>(lds + L::A);
  float* const X = reinterpret_cast<float*>(lds + L::X);
  ShortVec* const sv = reinterpret_cast<ShortVec*>(lds + L::vec);
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_id(), m = lane & 15, g = lane >> 4;
  const int rows = (int)a.rows.T;
  constexpr int P = KP / 8, N = kS * P * 2 / 256 < 1 ? 1 : kS * P * 2 / 256;   // pieces of eight for a thread: K, then Q
  f32x8 v[N];
  float odd[N], any = 0.f;
  const T* base[2] = {static_cast<const T*>(a.k) + n * a.ks[0] + hk * a.ks[2], static_cast<const T*>(a.q) + n * a.qs[0] + hk * a.qs[2]};
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int e = tid + 256 * i, w = e / (kS * P), r = e / P % kS, p = e % P, left = a.K - 8 * p;
    v[i] = f32x8{};
    if (r < rows && left > 0) v[i] = load8(base[w] + r * (w ? a.qs[1] : a.ks[1]) + 8 * p, left, w ? a.wide_q : a.wide_k);
  }
  if (tid < kS) sv->kbad[tid] = 0;
  lds_barrier();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int e = tid + 256 * i, w = e / (kS * P), r = e / P % kS, p = e % P;
    odd[i] = w ? 0.f : zero_if_finite(v[i].lo) + zero_if_finite(v[i].hi);
    any += odd[i];
    bf16x8 pl[NP];
    planes8<NP>(v[i], pl);
#pragma unroll
    for (int j = 0; j < NP; ++j) *reinterpret_cast<bf16x8*>(kq + (w * NP + j) * kTile + tile_at<KP>(r, p)) = pl[j];
  }
  if (__ballot(any != 0.f)) {   // rows of k that are not finite: marked, and zeros
    rare_path();
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (odd[i] != 0.f) sv->kbad[(tid + 256 * i) / P % kS] = 1;
  }
  lds_barrier();
  if (__ballot(sv->kbad[lane % kS])) {
    rare_path();
    for (int e = tid; e < kS * P * NP; e += 256) {
      const int r = e / (P * NP);
      if (sv->kbad[r]) *reinterpret_cast<u32x4*>(kq + e / P % NP * kTile + tile_at<KP>(r, e % P)) = u32x4{0, 0, 0, 0};
    }
    lds_barrier();
  }
  if (wave == 3) {
    const bool in = lane < rows;
    float gv = in ? a.g[n * a.gs[0] + lane * a.gs[1] + h * a.gs[2]] : 0.f;
    float bv = in ? a.beta[n * a.bs[0] + lane * a.bs[1] + h * a.bs[2]] : 0.f;
    gv = gv < kMinG ? kMinG : gv;
    const uint64_t bits = __ballot((gv - gv) + (bv - bv) != 0.f || (lane < kS && sv->kbad[lane < kS ? lane : 0]));
    const int bad = bits ? __ffsll((unsigned long long)bits) - 1 : kS;
    if (lane >= bad) gv = bv = 0.f;
    double last;
    const double sum = running_sum(gv, lane, last);
    const float hi = (float)sum;
    if (lane < kS) {
      sv->ghi[lane] = hi;
      sv->glo[lane] = (float)(sum - (double)hi);
      sv->into[lane] = expf((float)sum);
      sv->left[lane] = expf((float)(last - sum));
      sv->beta[lane] = bv;
      sv->all = expf((float)last);
      sv->bad = (float)bad;
    }
  }
  const int ti = wave > 0, tj = wave > 1;
  kk = qk = f32x4{0.f, 0.f, 0.f, 0.f};
  if (wave < 3) {
#pragma unroll
    for (int s = 0; s < L::KS; ++s) {
      bf16x8 ka[NP], qa[NP], kb[NP];
      frag<KP, NP, kTile>(kq, 16 * ti + m, s, g, ka);
      frag<KP, NP, kTile>(kq + NP * kTile, 16 * ti + m, s, g, qa);
      frag<KP, NP, kTile>(kq, 16 * tj + m, s, g, kb);
      kk = mfma_planes<NP, NP, 3>(ka, kb, kk);
      qk = mfma_planes<NP, NP, 3>(qa, kb, qk);
    }
  }
  mfma_settle();
  lds_barrier();
  float pv[4];
  const int c = wave < 3 ? 16 * tj + m : 16 + m, r0 = wave < 3 ? 16 * ti + 4 * g : 4 * g;   // wave 3: the zeros right of the diagonal
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int row = r0 + r;
    const bool lower = c <= row;
    const float d = lower ? expf((sv->ghi[row] - sv->ghi[c]) + (sv->glo[row] - sv->glo[c])) : 0.f;
    A[row * kSld + c] = c < row ? sv->beta[row] * d * kk[r] : 0.f;
    X[row * kSld + c] = 0.f;
    pv[r] = lower ? a.scale * d * qk[r] : 0.f;
  }
  lds_barrier();
  // X = (I + A)^-1, as in k_delta_prep
  if (wave == 0) {
    if (g < 2) {
      float x[16];
      const float* blk = A + (16 * g) * kSld + 16 * g;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float t = i == m ? 1.f : 0.f;
#pragma unroll
        for (int q = 0; q < (i + 3) / 4; ++q) {
          const f32x4 w = *reinterpret_cast<const f32x4*>(blk + i * kSld + 4 * q);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (4 * q + j < i) t = fmaf(-w[j], x[4 * q + j], t);
        }
        x[i] = t;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) X[(16 * g + i) * kSld + 16 * g + m] = x[i];
    }
    // [X11 0; -X22 A21 X11  X22]; A's upper right tile holds A21 X11 meanwhile.  One wave: its own LDS writes are in order
    f32x4 y = {0.f, 0.f, 0.f, 0.f}, z = y;
    for (int k = 0; k < 16; k += 4)
      y = __builtin_amdgcn_mfma_f32_16x16x4f32(A[(16 + m) * kSld + k + g], X[(k + g) * kSld + m], y, 0, 0, 0);
#pragma unroll
    for (int r = 0; r < 4; ++r) A[(4 * g + r) * kSld + 16 + m] = y[r];
    for (int k = 0; k < 16; k += 4)
      z = __builtin_amdgcn_mfma_f32_16x16x4f32(X[(16 + m) * kSld + 16 + k + g], A[(k + g) * kSld + 16 + m], z, 0, 0, 0);
#pragma unroll
    for (int r = 0; r < 4; ++r) X[(16 + 4 * g + r) * kSld + m] = -z[r];
  }
  lds_barrier();
  // planes of X, and of P (where A was: all of A has been read)
#pragma unroll
  for (int r = 0; r < 4; ++r) A[(r0 + r) * kSld + c] = pv[r];
  lds_barrier();
  __bf16* const xp = reinterpret_cast<__bf16*>(lds + L::xp);
  {
    const int w = tid / 128, r = tid / 4 % 32, p = tid % 4;
    const float* src = (w ? A : X) + r * kSld + 8 * p;
    bf16x8 pl[3];
    planes8<3>(cat8(*reinterpret_cast<const f32x4*>(src), *reinterpret_cast<const f32x4*>(src + 4)), pl);
#pragma unroll
    for (int j = 0; j < 3; ++j)
      if (!w || j < L::NPP) *reinterpret_cast<bf16x8*>(xp + (w * 3 + j) * kMat + tile_at<kS>(r, p)) = pl[j];
  }
  lds_barrier();
}

// perm_row(t, 4 g + r) = 8 g + step(t) + r
__device__ constexpr int step(int t) { return 32 * (t >> 1) + 4 * (t & 1); }

// A lane's rows perm_row(t, 4 g + r), t < N, of its column: fetched at addresses inside, so that no branch separates the loads,
// and zeros outside when they are taken
template <class T, int N>
struct ShortRows {
  T raw[N][4];
  __device__ __forceinline__ void fetch(const T* p, uint32_t stride, int rows, int c, int g) {
    const uint32_t at = 8 * g * stride + c, last = (rows - 1) * stride + c;
#pragma unroll
    for (int t = 0; t < N; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) raw[t][r] = item(p, min(at + (step(t) + r) * stride, last));
  }
  __device__ __forceinline__ void take(int rows, bool in, int g, f32x4 (&v)[N]) const {
#pragma unroll
    for (int t = 0; t < N; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) v[t][r] = in && 8 * g + step(t) + r < rows ? (float)raw[t][r] : 0.f;
  }
};

__device__ __forceinline__ f32x4 vec4(const float* v, int t, int g) { return *reinterpret_cast<const f32x4*>(v + perm_row(t, 4 * g)); }

// u of the wave's 16 columns, from S and v: u = X (beta (v - exp(G_i) K S)); bad: the first row of the column that is not finite
template <int DT, int KP, bool GRAD>
__device__ __forceinline__ void short_u(const char* lds, const f32x4 (&st)[KP / 16], const f32x4 (&v)[2], int g, int x, f32x4 (&u)[2], int& bad) {
  using L = ShortLds<DT, KP, GRAD>;
  constexpr int NP = L::NP;
  const __bf16* K = reinterpret_cast<const __bf16*>(lds);
  const __bf16* X = reinterpret_cast<const __bf16*>(lds + L::xp);
  const ShortVec* sv = reinterpret_cast<const ShortVec*>(lds + L::vec);
  f32x4 ks[2] = {};
#pragma unroll
  for (int s = 0; s < L::KS; ++s) {
    bf16x8 sp[3], fa[2][NP];
    planes8<3>(cat8(st[2 * s], st[2 * s + 1]), sp);
#pragma unroll
    for (int t = 0; t < 2; ++t) frag<KP, NP, L::kTile>(K, perm_row(t, x), s, g, fa[t]);
    mfma_rows<NP, 3, 3, 2>([&](int t) -> const bf16x8(&)[NP] { return fa[t]; }, sp, ks);
  }
  bad = (int)sv->bad;
  int mine = kS;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    ks[t] = vec4(sv->beta, t, g) * (v[t] - vec4(sv->into, t, g) * ks[t]);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const bool odd = ks[t][r] * 0.f != 0.f;   // not a - a, which contracts to the rounding error of a product
      ks[t][r] = odd ? 0.f : ks[t][r];
      mine = odd ? min(mine, perm_row(t, 4 * g + r)) : mine;
    }
  }
  mine = min(mine, __shfl_xor(mine, 16));
  mine = min(mine, __shfl_xor(mine, 32));
  bad = min(bad, mine);
  bf16x8 rp[3], fx[2][3];
  planes8<3>(cat8(ks[0], ks[1]), rp);
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    frag<kS, 3, kMat>(X, perm_row(t, x), 0, g, fx[t]);
    u[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  mfma_rows<3, 3, 3, 2>([&](int t) -> const bf16x8(&)[3] { return fx[t]; }, rp, u);
}

template <int DT, int KP>
__global__ __launch_bounds__(256, 2) void k_delta_short(DeltaArgs a) {
  using L = ShortLds<DT, KP, false>;
  using T = typename Elem<DT>::T;
  constexpr int NP = L::NP, NO = L::NO, KT = L::KT;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63, wave = wave_id();
  int x = lane & 15, g = lane >> 4;
  const int64_t n = blockIdx.x / a.Hv;
  const int h = (int)(blockIdx.x % a.Hv), hk = h / (a.Hv / a.Hk), rows = (int)a.rows.T;
  const int64_t head = n * a.Hv + h;
  const float* s0 = a.initial ? a.initial + head * a.K * a.V : nullptr;
  const T* v_in = static_cast<const T*>(a.v) + n * a.vs[0] + h * a.vs[2];
  T* const o_out = static_cast<T*>(a.o) + ((int64_t)n * rows * a.Hv + h) * a.V;
  float* const final = a.final + head * a.K * a.V;
  const uint32_t orow = a.Hv * a.V;
  f32x4 kk, qk;
  ShortRows<float, KT> sn = {};
  ShortRows<T, 2> vn;
  auto fetch = [&](int c0) {   // ahead of their use
    const int c = min(c0 + x, a.V - 1);
    if (s0) sn.fetch(s0, a.V, a.K, c, g);
    vn.fetch(v_in, (uint32_t)a.vs[1], rows, c, g);
  };
  fetch(16 * wave);
  short_prep<DT, KP, false>(a, n, h, hk, lds, kk, qk);
  const __bf16* K = reinterpret_cast<const __bf16*>(lds);
  const __bf16* Q = K + NP * L::kTile;
  const __bf16* P = reinterpret_cast<const __bf16*>(lds + L::xp) + 3 * kMat;
  const ShortVec* sv = reinterpret_cast<const ShortVec*>(lds + L::vec);
  const float nan = __builtin_nanf("");
  for (int c0 = 16 * wave; c0 < a.V; c0 += 64) {
    here(g, x);
    const int col = c0 + x;
    const bool in = col < a.V;
    f32x4 st[KT], v[2], u[2], o[2] = {};
    sn.take(a.K, in, g, st);
    vn.take(rows, in, g, v);
    if (c0 + 64 < a.V) fetch(c0 + 64);
    int bad;
    short_u<DT, KP, false>(lds, st, v, g, x, u, bad);
    // o = scale exp(G_i) Q S + P u
#pragma unroll
    for (int s = 0; s < L::KS; ++s) {
      bf16x8 sp[NO], fa[2][NP];
      planes8<NO>(cat8(st[2 * s], st[2 * s + 1]), sp);
#pragma unroll
      for (int t = 0; t < 2; ++t) frag<KP, NP, L::kTile>(Q, perm_row(t, x), s, g, fa[t]);
      mfma_rows<NP, NO, NO, 2>([&](int t) -> const bf16x8(&)[NP] { return fa[t]; }, sp, o);
    }
    {
      bf16x8 up[NO], fp[2][NO];
      planes8<NO>(cat8(u[0], u[1]), up);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        frag<kS, NO, kMat>(P, perm_row(t, x), 0, g, fp[t]);
        o[t] *= a.scale * vec4(sv->into, t, g);
      }
      mfma_rows<NO, NO, NO, 2>([&](int t) -> const bf16x8(&)[NO] { return fp[t]; }, up, o);
    }
    // S <- exp(G) S + K^T (exp(G - G_i) u), NaN in a column that is no longer finite
    {
      bf16x8 up[3], ft[KT][NP];
      planes8<3>(cat8(vec4(sv->left, 0, g) * u[0], vec4(sv->left, 1, g) * u[1]), up);
      const float all = bad < kS ? nan : sv->all;
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        frag_t<KP, NP, L::kTile>(K, t, 0, g, x, ft[t]);
        st[t] *= all;
      }
      mfma_rows<NP, 3, 3, KT>([&](int t) -> const bf16x8(&)[NP] { return ft[t]; }, up, st);
    }
    mfma_settle();
    if (in) {
      const uint32_t oat = 8 * g * orow + col, fat = 8 * g * a.V + col;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = 8 * g + step(t) + r;
          if (row < rows) item(o_out, oat + (step(t) + r) * orow) = (T)(row >= bad ? nan : o[t][r]);
        }
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (8 * g + step(t) + r < a.K) item(final, fat + (step(t) + r) * a.V) = st[t][r];
    }
  }
}

template <int NP, int TILE>
__device__ __forceinline__ float joined(const __bf16* p) {
  float v = (float)p[(NP - 1) * TILE];
#pragma unroll
  for (int i = NP - 2; i >= 0; --i) v += (float)p[i * TILE];
  return v;
}

// Names as in k_delta_back and k_delta_grad.
// K = 128: one wave a SIMD, with the registers of two (two of them spilled 230 registers each, and took 2197 for 946 us)
template <int DT, int KP>
__global__ __launch_bounds__(256, KP == 128 ? 1 : 2) void k_delta_short_grad(DeltaGradArgs ga, bool wide_s) {
  using L = ShortLds<DT, KP, true>;
  using T = typename Elem<DT>::T;
  constexpr int NP = L::NP, NO = L::NO, KT = L::KT, NT = KT >= 4 ? KT / 4 : 1, kTile = L::kTile, kCol = L::kCol;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const DeltaArgs& a = ga.f;
  const int lane = threadIdx.x & 63, wave = wave_id();
  int x = lane & 15, g = lane >> 4;
  const int64_t n = blockIdx.x / a.Hv;
  const int h = (int)(blockIdx.x % a.Hv), hk = h / (a.Hv / a.Hk), rows = (int)a.rows.T;
  const int64_t head = n * a.Hv + h, first = (n * rows * a.Hv + h) * a.V;
  const uint32_t orow = a.Hv * a.V;
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  const float* s0 = a.initial ? a.initial + head * a.K * a.V : nullptr;
  const float* df = ga.d_final ? ga.d_final + head * a.K * a.V : nullptr;
  const T* v_in = static_cast<const T*>(a.v) + n * a.vs[0] + h * a.vs[2];
  const T* do_in = static_cast<const T*>(ga.d_o) + first;
  float* const di_out = ga.d_initial ? ga.d_initial + head * a.K * a.V : nullptr;
  T* const dv_out = static_cast<T*>(ga.dv) + first;
  f32x4 kk, qk;
  ShortRows<float, KT> sn = {}, dn = {};
  ShortRows<T, 2> vn, on;
  auto fetch = [&](int v0) {   // ahead of their use
    const int c = min(v0 + 16 * wave + x, a.V - 1);
    if (s0) sn.fetch(s0, a.V, a.K, c, g);
    if (df) dn.fetch(df, a.V, a.K, c, g);
    vn.fetch(v_in, (uint32_t)a.vs[1], rows, c, g);
    on.fetch(do_in, orow, rows, c, g);
  };
  fetch(0);
  short_prep<DT, KP, true>(a, n, h, hk, lds, kk, qk);
  const __bf16* K = reinterpret_cast<const __bf16*>(lds);
  const __bf16* Q = K + NP * kTile;
  const __bf16* X = reinterpret_cast<const __bf16*>(lds + L::xp);
  const __bf16* P = X + 3 * kMat;
  const ShortVec* sv = reinterpret_cast<const ShortVec*>(lds + L::vec);
  __bf16* const cu = reinterpret_cast<__bf16*>(lds + L::cols);   // planes [64 columns][32 rows] of u, dR, do
  __bf16* const cr = cu + 3 * kCol;
  __bf16* const co = cr + 3 * kCol;
  const float nan = __builtin_nanf("");

  const bool active = wave * NT < KT;
  // rows kd of S and dS, eight columns of step s
  f32x8 sr[NT], dr8[NT];
  auto fetch_rows = [&](const float* p, int c, f32x8 (&to)[NT]) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      to[j] = f32x8{};
      if (!p) continue;
      const int kd = 16 * (wave * NT + j) + x, row = min(kd, a.K - 1) * a.V;
      const bool in = active && kd < a.K;
      if (wide_s) {
        const f32x4 lo = *reinterpret_cast<const f32x4*>(p + row + min(c, a.V - 4));
        const f32x4 hi = *reinterpret_cast<const f32x4*>(p + row + min(c + 4, a.V - 4));
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          to[j][r] = in && c < a.V ? lo[r] : 0.f;
          to[j][4 + r] = in && c + 4 < a.V ? hi[r] : 0.f;
        }
      } else {
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const float one = p[row + min(c + r, a.V - 1)];
          to[j][r] = in && c + r < a.V ? one : 0.f;
        }
      }
    }
  };
  f32x4 X1[2][NT], Y[2][NT], Z[2][NT], M = zero, N = zero;
  float rv[2][4] = {}, dot = 0.f;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) X1[i][j] = Y[i][j] = Z[i][j] = zero;

  for (int v0 = 0; v0 < a.V; v0 += 64) {
    here(g, x);
    const int col = v0 + 16 * wave + x;
    const bool in = col < a.V;
    if (v0 + 16 * wave < a.V) {
      f32x4 st[KT], ds[KT], v[2], d[2], u[2], du[2], dr[2] = {zero, zero};
      sn.take(a.K, in, g, st);
      dn.take(a.K, in, g, ds);
      vn.take(rows, in, g, v);
      on.take(rows, in, g, d);
      int bad;
      short_u<DT, KP, true>(lds, st, v, g, x, u, bad);
      mfma_settle();
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) u[t][r] = perm_row(t, 4 * g + r) >= bad ? nan : u[t][r];
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) dot = fmaf(st[t][r], ds[t][r], dot);
      // du = exp(G - G_i) K dS + P^T do
      du[0] = du[1] = zero;
#pragma unroll
      for (int s = 0; s < L::KS; ++s) {
        bf16x8 sp[3], fa[2][NP];
        planes8<3>(cat8(ds[2 * s], ds[2 * s + 1]), sp);
#pragma unroll
        for (int t = 0; t < 2; ++t) frag<KP, NP, kTile>(K, perm_row(t, x), s, g, fa[t]);
        mfma_rows<NP, 3, 3, 2>([&](int t) -> const bf16x8(&)[NP] { return fa[t]; }, sp, du);
      }
      bf16x8 dp[NP], fp[2][3];
      planes8<NP>(cat8(d[0], d[1]), dp);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        du[t] *= vec4(sv->left, t, g);
        frag_t<kS, 3, kMat>(P, t, 0, g, x, fp[t]);
      }
      mfma_rows<3, NP, 3, 2>([&](int t) -> const bf16x8(&)[3] { return fp[t]; }, dp, du);
      // dR = X^T du
      bf16x8 p3[3];
      planes8<3>(cat8(du[0], du[1]), p3);
#pragma unroll
      for (int t = 0; t < 2; ++t) frag_t<kS, 3, kMat>(X, t, 0, g, x, fp[t]);
      mfma_rows<3, 3, 3, 2>([&](int t) -> const bf16x8(&)[3] { return fp[t]; }, p3, dr);
      mfma_settle();
      // u, dR and do for the sums over the columns
#pragma unroll
      for (int j = 0; j < NP; ++j) *reinterpret_cast<bf16x8*>(co + j * kCol + tile_at<kS>(16 * wave + x, g)) = dp[j];
      planes8<3>(cat8(dr[0], dr[1]), p3);
#pragma unroll
      for (int j = 0; j < 3; ++j) *reinterpret_cast<bf16x8*>(cr + j * kCol + tile_at<kS>(16 * wave + x, g)) = p3[j];
      planes8<3>(cat8(u[0], u[1]), p3);
#pragma unroll
      for (int j = 0; j < 3; ++j) *reinterpret_cast<bf16x8*>(cu + j * kCol + tile_at<kS>(16 * wave + x, g)) = p3[j];
      // dv, and the initial state's gradient
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const f32x4 dv = vec4(sv->beta, t, g) * dr[t];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = 8 * g + step(t) + r;
          rv[t][r] = fmaf(dr[t][r], v[t][r], rv[t][r]);
          if (in && row < rows) item(dv_out, 8 * g * orow + col + (step(t) + r) * orow) = (T)dv[r];
        }
        d[t] *= a.scale * vec4(sv->into, t, g);
        dr[t] = -vec4(sv->into, t, g) * dv;
      }
      if (di_out) {
        bf16x8 ep[3], rp[3];
        planes8<3>(cat8(d[0], d[1]), ep);
        planes8<3>(cat8(dr[0], dr[1]), rp);
#pragma unroll
        for (int t = 0; t < KT; ++t) {
          bf16x8 fa[NP];
          ds[t] *= sv->all;
          frag_t<KP, NP, kTile>(Q, t, 0, g, x, fa);
          ds[t] = mfma_planes<NP, 3, 3>(fa, ep, ds[t]);
          frag_t<KP, NP, kTile>(K, t, 0, g, x, fa);
          ds[t] = mfma_planes<NP, 3, 3>(fa, rp, ds[t]);
        }
        mfma_settle();
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if (in && 8 * g + step(t) + r < a.K) item(di_out, 8 * g * a.V + col + (step(t) + r) * a.V) = ds[t][r];
          }
      }
    } else {
      const bf16x8 none = {};
#pragma unroll
      for (int j = 0; j < 6 + NP; ++j) *reinterpret_cast<bf16x8*>(cu + j * kCol + tile_at<kS>(16 * wave + x, g)) = none;
    }
    here(g, x);
    fetch_rows(s0, v0 + 8 * g, sr);
    fetch_rows(df, v0 + 8 * g, dr8);
    lds_barrier();
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if (s == 1) {
        fetch_rows(s0, v0 + 32 + 8 * g, sr);
        fetch_rows(df, v0 + 32 + 8 * g, dr8);
      }
      if (wave < 3) {   // the tile of kk and qk
        bf16x8 fo[NP], fr[3], fu[3];
        frag_col<kS, NP, kCol>(co, wave > 0, s, g, x, fo);
        frag_col<kS, 3, kCol>(cr, wave > 0, s, g, x, fr);
        frag_col<kS, 3, kCol>(cu, wave > 1, s, g, x, fu);
        M = mfma_planes<NP, 3, 3>(fo, fu, M);
        N = mfma_planes<3, 3, 3>(fr, fu, N);
      }
      if (active) {
        bf16x8 sp[NT][3], dp[NT][3];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          planes8<3>(sr[j], sp[j]);
          planes8<3>(dr8[j], dp[j]);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {   // one row tile's operands at a time: more do not fit in the registers
          bf16x8 fo[NP], fr[3], fu[3];
          frag_col<kS, NP, kCol>(co, i, s, g, x, fo);
          frag_col<kS, 3, kCol>(cr, i, s, g, x, fr);
          frag_col<kS, 3, kCol>(cu, i, s, g, x, fu);
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            X1[i][j] = mfma_planes<NP, 3, 3>(fo, sp[j], X1[i][j]);
            Y[i][j] = mfma_planes<3, 3, 3>(fr, sp[j], Y[i][j]);
            Z[i][j] = mfma_planes<3, 3, 3>(fu, dp[j], Z[i][j]);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
    mfma_settle();
    if (v0 + 64 < a.V) fetch(v0 + 64);
    lds_barrier();   // the next columns, or m and n, go where these were
  }

  float* const qx = reinterpret_cast<float*>(lds + L::sums);   // by wave and row: q . X, k . Y, k . Z, dR . v
  float *const ky = qx + 4 * kS, *const kz = ky + 4 * kS, *const rw = kz + 4 * kS;
  float *const rs = rw + 4 * kS, *const rb = rs + 3 * 16, *const cs = rb + 3 * 16, *const dots = cs + 3 * 16;   // by tile
  __bf16* const mt_ = cu;
  __bf16* const nt_ = mt_ + NO * kMat;
  {
    const int ti = wave > 0, tj = wave > 1;
    const int c = wave < 3 ? 16 * tj + x : 16 + x, r0 = wave < 3 ? 16 * ti + 4 * g : 4 * g;
    float csum = 0.f;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = r0 + r;
      const float d = row >= c ? expf((sv->ghi[row] - sv->ghi[c]) + (sv->glo[row] - sv->glo[c])) : 0.f;
      const float mv = row >= c ? a.scale * d * M[r] : 0.f;
      const float nb = row > c ? -d * N[r] : 0.f, nn = sv->beta[row] * nb;
      const float e = row > c ? fmaf(mv, qk[r], nn * kk[r]) : 0.f;
      csum += e;
      const float se = sum16(e), sb = sum16(row > c ? nb * kk[r] : 0.f);
      if (x == 0 && wave < 3) {
        rs[wave * 16 + 4 * g + r] = se;
        rb[wave * 16 + 4 * g + r] = sb;
      }
      const int at = tile_at<kS>(row, c >> 3) + (c & 7);
      float rm = mv, rn = nn;
#pragma unroll
      for (int p = 0; p < NO; ++p) {
        const __bf16 bm = (__bf16)rm, bn = (__bf16)rn;
        mt_[p * kMat + at] = bm;
        nt_[p * kMat + at] = bn;
        rm -= (float)bm;
        rn -= (float)bn;
      }
    }
    csum += __shfl_xor(csum, 16);
    csum += __shfl_xor(csum, 32);
    if (g == 0 && wave < 3) cs[wave * 16 + x] = csum;
  }
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float s = sum16(rv[t][r]);
      if (x == 0) rw[wave * kS + perm_row(t, 4 * g + r)] = s;
    }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) dot += __shfl_xor(dot, d);
  if (lane == 0) dots[wave] = dot;
  // q . X, k . Y, k . Z; what dq and dk have of the states
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = 16 * i + 4 * g + r;
      float sq = 0.f, sy = 0.f, sz = 0.f;
      if (active) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const int kd = 16 * (wave * NT + j) + x, at = tile_at<KP>(row, kd >> 3) + (kd & 7);
          const float kv = joined<NP, kTile>(K + at), qv = joined<NP, kTile>(Q + at);
          const float xs = a.scale * sv->into[row] * X1[i][j][r], ys = sv->into[row] * Y[i][j][r], zs = sv->left[row] * Z[i][j][r];
          sq = fmaf(qv, xs, sq);
          sy = fmaf(kv, ys, sy);
          sz = fmaf(kv, zs, sz);
          X1[i][j][r] = xs;
          Y[i][j][r] = fmaf(-sv->beta[row], ys, zs);
        }
      }
      sq = sum16(sq), sy = sum16(sy), sz = sum16(sz);
      if (x == 0) {
        qx[wave * kS + row] = sq;
        ky[wave * kS + row] = sy;
        kz[wave * kS + row] = sz;
      }
    }
  lds_barrier();
  if (active) {
    const int64_t at32 = (n * rows * a.Hv + h) * a.K, at16 = (n * rows * a.Hk + hk) * a.K;
    float *const dq32 = ga.dq32 + at32, *const dk32 = ga.dk32 + at32;
    T *const dq = static_cast<T*>(ga.dq) + at16, *const dk = static_cast<T*>(ga.dk) + at16;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      bf16x8 kb[NP], qb[NP];
      frag_col<KP, NP, kTile>(K, wave * NT + j, 0, g, x, kb);
      frag_col<KP, NP, kTile>(Q, wave * NT + j, 0, g, x, qb);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        bf16x8 fa[NO];
        frag<kS, NO, kMat>(mt_, 16 * i + x, 0, g, fa);
        X1[i][j] = mfma_planes<NO, NP, NO>(fa, kb, X1[i][j]);
        frag<kS, NO, kMat>(nt_, 16 * i + x, 0, g, fa);
        Y[i][j] = mfma_planes<NO, NP, NO>(fa, kb, Y[i][j]);
        frag_col<kS, NO, kMat>(mt_, i, 0, g, x, fa);
        Y[i][j] = mfma_planes<NO, NP, NO>(fa, qb, Y[i][j]);
        frag_col<kS, NO, kMat>(nt_, i, 0, g, x, fa);
        Y[i][j] = mfma_planes<NO, NP, NO>(fa, kb, Y[i][j]);
      }
    }
    mfma_settle();
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 16 * i + 4 * g + r;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const int kd = 16 * (wave * NT + j) + x;
          if (row >= rows || kd >= a.K) continue;
          if (ga.dq32) {
            const uint32_t at = row * (uint32_t)(a.Hv * a.K) + kd;
            item(dq32, at) = X1[i][j][r];
            item(dk32, at) = Y[i][j][r];
          } else {
            const uint32_t at = row * (uint32_t)(a.Hk * a.K) + kd;
            item(dq, at) = (T)X1[i][j][r];
            item(dk, at) = (T)Y[i][j][r];
          }
        }
      }
  }
  if (wave == 0) {
    const int at = lane < kS ? lane : 0, lo = at & 15;
    auto waves = [&](const float* p) { return lane < kS ? (p[at] + p[kS + at]) + (p[2 * kS + at] + p[3 * kS + at]) : 0.f; };
    auto tile_rows = [&](const float* p) { return at < 16 ? p[lo] : p[16 + lo] + p[32 + lo]; };
    const float y = waves(ky), z = waves(kz), cols = at < 16 ? cs[lo] + cs[16 + lo] : cs[32 + lo];
    const double own = lane < kS ? (double)tile_rows(rs) - cols + waves(qx) - sv->beta[at] * y - z : 0.0;
    double tail, zall;
    const double upto = running_sum64(own, lane, tail);
    running_sum64(z, lane, zall);
    const double end = zall + (double)sv->all * ((dots[0] + dots[1]) + (dots[2] + dots[3]));
    if (lane < rows) {
      const int64_t to = (n * rows + lane) * a.Hv + h;
      const float graw = a.g[n * a.gs[0] + lane * a.gs[1] + h * a.gs[2]];
      ga.dg[to] = graw < kMinG ? 0.f : (float)(end + tail - upto + own);
      ga.dbeta[to] = waves(rw) - y + tile_rows(rb);
    }
  }
}

template <int DT, int KP>
hipError_t forward(const DeltaArgs& a, hipStream_t s) {
  constexpr int bytes = ShortLds<DT, KP, false>::bytes;
  const hipError_t e = allow_lds(k_delta_short<DT, KP>, bytes);
  if (e != hipSuccess) return e;
  k_delta_short<DT, KP><<<(unsigned)(a.rows.N * a.Hv), 256, bytes, s>>>(a);
  return hipGetLastError();
}
template <int DT, int KP>
hipError_t backward(const DeltaGradArgs& ga, bool wide_s, hipStream_t s) {
  constexpr int bytes = ShortLds<DT, KP, true>::bytes;
  const hipError_t e = allow_lds(k_delta_short_grad<DT, KP>, bytes);
  if (e != hipSuccess) return e;
  k_delta_short_grad<DT, KP><<<(unsigned)(ga.f.rows.N * ga.f.Hv), 256, bytes, s>>>(ga, wide_s);
  return hipGetLastError();
}
template <int DT>
hipError_t forward(const DeltaArgs& a, int KP, hipStream_t s) {
  return KP == 32 ? forward<DT, 32>(a, s) : KP == 64 ? forward<DT, 64>(a, s) : forward<DT, 128>(a, s);
}
template <int DT>
hipError_t backward(const DeltaGradArgs& ga, int KP, bool wide_s, hipStream_t s) {
  return KP == 32 ? backward<DT, 32>(ga, wide_s, s) : KP == 64 ? backward<DT, 64>(ga, wide_s, s) : backward<DT, 128>(ga, wide_s, s);
}

}  // namespace

hipError_t delta_short_forward(const DeltaArgs& a, int dtype, int KP, hipStream_t s) {
  return dtype == SEQ_BF16 ? forward<SEQ_BF16>(a, KP, s) : dtype == SEQ_FP16 ? forward<SEQ_FP16>(a, KP, s) : forward<SEQ_FP32>(a, KP, s);
}
hipError_t delta_short_backward(const DeltaGradArgs& ga, int dtype, int KP, bool wide_s, hipStream_t s) {
  return dtype == SEQ_BF16 ? backward<SEQ_BF16>(ga, KP, wide_s, s)
         : dtype == SEQ_FP16 ? backward<SEQ_FP16>(ga, KP, wide_s, s) : backward<SEQ_FP32>(ga, KP, wide_s, s);
}

}  // namespace seq
