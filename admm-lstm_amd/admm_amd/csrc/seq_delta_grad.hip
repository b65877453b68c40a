// seq_delta_grad.hip -- gradients of the gated delta rule (seq_delta.hpp has the forward's formulas and names).
//
// With dS the gradient of the state behind a chunk, do that of o, R = beta (v - exp(G_i) K S) and u = X R:
//     du = P^T do + exp(G - G_i) K dS,   dR = X^T du,   dv = beta dR,
//     dS <- exp(G) dS + scale Q^T (exp(G_i) do) - K^T (exp(G_i) beta dR).
// Again only these products run in order (backwards), and again each column by itself: k_delta_back, the mirror image of
// k_delta_scan.  It leaves dS and dR of every chunk; all other gradients follow chunk by chunk (k_delta_grad), from products
// over the value axis, with M = do u^T, N = dR u^T, and masked by i >= j (M) and i > j (N):
//     m = scale D M,  n = -beta_i D N,
//     dq = scale exp(G_i) do S^T + m K
//     dk = exp(G - G_i) u dS^T - exp(G_i) beta dR S^T + m^T Q + (n + n^T) K
//     dbeta_i = dR_i . v_i - exp(G_i) k_i . (S dR_i) - sum_j D_ij N_ij (k_i . k_j)
//     dG_i = q_i . (scale exp(G_i) S do_i) - beta_i exp(G_i) k_i . (S dR_i) - exp(G - G_i) k_i . (dS u_i)
//            + sum_{j < i} (m q.k + n k.k)_ij - sum_{j > i} (m q.k + n k.k)_ji
//     dG += exp(G) <S, dS> + sum_i exp(G - G_i) k_i . (dS u_i),    dg_t = dG + sum_{i >= t} dG_i.
// (The diagonal has no decay in it: it would cancel in dG_i, but leave its rounding in a dg that strong decays make small.)
#include "seq_delta_dev.hpp"

namespace seq {
namespace {

// As in k_delta_scan, HW of C / 16 waves keep TW tiles of dS each and form their share of K dS, and wave w takes rows
// perm_row(w, .) of du and dR.  As many more waves form what does not depend on dS, P^T do and scale Q^T (exp(G_i) do), one
// chunk ahead.
//
// Bound as k_delta_scan is: 3.2 us a chunk (32 chunks, 256 column tiles of 128 x 128, bf16: 102 us).
template <int DT, int KP, int C, int NC>
struct Back {
  using S = DeltaShape<DT, KP, C, true>;
  static constexpr int TW = S::KT >= 2 * S::RT ? S::KT / S::RT : 2, HW = S::KT / TW;
  // shares of K dS; do, and scale exp(G_i) do, as operands; du; exp(G_i) beta dR; P^T do; scale Q^T (exp(G_i) do), twice   (KB)
  static constexpr int bK = 0, bO = HW * S::RT, bE = bO + S::CS * S::NP, bU = bE + S::CS * 3, bR = bU + S::CS * 3,
                       bP = bR + S::CS * 3, bQ = bP + S::RT, bEnd = bQ + 2 * S::KT;
  static constexpr int bytes = NC * bEnd * 1024;
};

template <int DT, int KP, int C, int NC>
__global__ __launch_bounds__(8 * C, 2) void k_delta_back(DeltaGradArgs ga) {
  using S = DeltaShape<DT, KP, C, true>;
  using B = Back<DT, KP, C, NC>;
  using T = typename Elem<DT>::T;
  constexpr int NP = S::NP, TW = B::TW, HW = B::HW;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const DeltaArgs& a = ga.f;
  const int lane = threadIdx.x & 63, wave = wave_id(), w = wave % S::RT, x = lane & 15, g = lane >> 4;
  const int groups = (a.VP / 16 + NC - 1) / NC;
  int64_t n;
  int h, hk, group;
  if (!place_columns(a, groups, n, h, hk, group)) return;
  const int64_t head = n * a.Hv + h;
  const int col0 = group * NC * 16 + x;
  int64_t begin, len, c0;
  a.rows.range(n, begin, len, c0);
  begin = uniform(begin), len = uniform(len), c0 = uniform(c0);
  const int nc = (int)((len + C - 1) / C);
  const int row0 = perm_row(w, 4 * g);
  const uint32_t at16 = lane * 16;

  const int64_t last = c0 + (nc > 0 ? nc - 1 : 0);
  const char* kq = a.kq + (last * a.Hk + hk) * (int64_t)S::kKQ;
  const char* xp = a.xp + (last * a.Hv + h) * (int64_t)S::kXP;
  const char* vec = a.vec + (last * a.Hv + h) * (int64_t)kVec;
  const int64_t kq_step = (int64_t)a.Hk * S::kKQ, xp_step = (int64_t)a.Hv * S::kXP, vec_step = (int64_t)a.Hv * kVec;
  const int64_t orow = (int64_t)a.Hv * a.V, first = ((a.rows.batch(n) * a.rows.T + begin) * a.Hv + h) * (int64_t)a.V;
  bool in[NC];
#pragma unroll
  for (int i = 0; i < NC; ++i) in[i] = col0 + 16 * i < a.V;
  auto part = [&](int i, int b) { return lds + (i * B::bEnd + b) * 1024; };
  // fragment of the transposed triangular matrices; below the diagonal there is none
  auto tri_t = [&](int s) { return C == 32 ? w : tri_frag_t(w, s); };
  bf16x8 ft[TW][S::CS][NP], fx[S::CS][3];   // K^T and X^T, or Q^T and P^T
#pragma unroll
  for (int s = 0; s < S::CS; ++s)
#pragma unroll
    for (int i = 0; i < 3; ++i) fx[s][i] = bf16x8{};
  auto load_t = [&](int f) {
#pragma unroll
    for (int t = 0; t < TW; ++t)
#pragma unroll
      for (int s = 0; s < S::CS; ++s) load_frag<NP>(kq, (f + (w * TW + t) * S::CS + s) * NP, at16, ft[t][s]);
  };
  auto load_x = [&](int p) {
#pragma unroll
    for (int s = 0; s < S::CS; ++s)
      if (s >= w / 2) load_frag<3>(xp, p + 3 * tri_t(s), at16, fx[s]);
  };

  const bool holds = w < HW;
  if (wave < S::RT) {   // ---- dS
    f32x4 ds[NC][TW];
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
      for (int t = 0; t < TW; ++t)
        ds[i][t] = load_state(ga.d_final && holds ? ga.d_final + head * a.K * a.V : nullptr, a.K, a.V, col0 + 16 * i, w * TW + t, g);
    T* dvp[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) dvp[i] = static_cast<T*>(ga.dv) + first + col0 + 16 * i + row0 * orow;
    bf16x8 fk[S::RT][TW / 2][NP];
    struct { f32x4 into, left, beta; float all; } f, fnext;
    auto load_k = [&]() {
      if (!holds) return;
#pragma unroll
      for (int t = 0; t < S::RT; ++t)
#pragma unroll
        for (int s = 0; s < TW / 2; ++s) load_frag<NP>(kq, (S::fK + t * S::KS + w * (TW / 2) + s) * NP, at16, fk[t][s]);
    };
    auto load_vec = [&]() {
      const float* p = reinterpret_cast<const float*>(vec);
      fnext.into = *reinterpret_cast<const f32x4*>(p + row0);
      fnext.left = *reinterpret_cast<const f32x4*>(p + 64 + row0);
      fnext.beta = *reinterpret_cast<const f32x4*>(p + 128 + row0);
      fnext.all = p[192];
    };
    auto put_share = [&]() {   // (where the wave has tiles of dS)
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        f32x4 ks[S::RT];
#pragma unroll
        for (int t = 0; t < S::RT; ++t) ks[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < TW / 2; ++s) {
          bf16x8 sp[3];
          planes8<3>(cat8(ds[i][2 * s], ds[i][2 * s + 1]), sp);
          mfma_rows<NP, 3, 3, S::RT>([&](int t) -> const bf16x8(&)[NP] { return fk[t][s]; }, sp, ks);
        }
#pragma unroll
        for (int t = 0; t < S::RT; ++t) *reinterpret_cast<f32x4*>(part(i, B::bK) + (t * HW + w) * 1024 + at16) = ks[t];
      }
    };
    if (nc > 0) {
      load_k();
      load_vec();
      load_x(S::pXT);
      if (holds) {
        load_t(S::fKT);
        put_share();
      }
      lds_barrier();   // (the other waves exchange the last chunk's do)
      lds_barrier();
    }
    for (int ci = nc - 1; ci >= 0; --ci) {
      const bool more = ci > 0;
      const int64_t ch = (c0 + ci) * a.Hv + h;
      const int rows = (int)(len - (int64_t)ci * C < C ? len - (int64_t)ci * C : C);
      lds_barrier();
      // du = exp(G - G_i) K dS + P^T do
      f = fnext;
      if (more) vec -= vec_step;
      load_vec();
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        f32x4 k = *reinterpret_cast<const f32x4*>(part(i, B::bK) + w * HW * 1024 + at16);
#pragma unroll
        for (int j = 1; j < HW; ++j) k += *reinterpret_cast<const f32x4*>(part(i, B::bK) + (w * HW + j) * 1024 + at16);
        put_half<3>(part(i, B::bU), w / 2, w & 1, lane, f.left * k + *reinterpret_cast<const f32x4*>(part(i, B::bP) + w * 1024 + at16));
      }
      if (more) kq -= kq_step;
      load_k();
      if (holds) {
        float* p = ga.ds + ch * (int64_t)KP * a.VP + col0;
#pragma unroll
        for (int i = 0; i < NC; ++i)
#pragma unroll
          for (int t = 0; t < TW; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (col0 + 16 * i < a.VP) p[perm_row(w * TW + t, 4 * g + r) * a.VP + 16 * i] = ds[i][t][r];
      }
      lds_barrier();
      // dR = X^T du
      f32x4 dr[NC];
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        dr[i] = product<3, 3, 3, S::CS>(fx, [&](int s, bf16x8(&b)[3]) { get_operand<3>(part(i, B::bU), s, lane, b); });
        put_half<3>(part(i, B::bR), w / 2, w & 1, lane, -f.into * (f.beta * dr[i]));
      }
      if (more) xp -= xp_step;
      load_x(S::pXT);
      lds_barrier();
      // dS <- exp(G) dS + scale Q^T (exp(G_i) do) - K^T (exp(G_i) beta dR)
      if (holds) {
#pragma unroll
        for (int i = 0; i < NC; ++i) {
          const char* q = part(i, B::bQ) + (ci & 1) * S::KT * 1024;
#pragma unroll
          for (int t = 0; t < TW; ++t) ds[i][t] = f.all * ds[i][t] + *reinterpret_cast<const f32x4*>(q + (w * TW + t) * 1024 + at16);
#pragma unroll
          for (int s = 0; s < S::CS; ++s) {
            bf16x8 rp[3];
            get_operand<3>(part(i, B::bR), s, lane, rp);
            mfma_rows<NP, 3, 3, TW>([&](int t) -> const bf16x8(&)[NP] { return ft[t][s]; }, rp, ds[i]);
          }
        }
        put_share();   // behind no branch: it reads the products' results first
        load_t(S::fKT);
      }
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        float* p = ga.dr + (ch * C + row0) * (int64_t)a.VP + col0 + 16 * i;
        T* dv = dvp[i] + (int64_t)ci * C * orow;
        const f32x4 bd = f.beta * dr[i];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (col0 + 16 * i < a.VP) p[r * a.VP] = dr[i][r];
          if (in[i] && row0 + r < rows) dv[r * orow] = (T)bd[r];
        }
      }
    }
    if (ga.d_initial && holds) {
#pragma unroll
      for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int t = 0; t < TW; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int kd = perm_row(w * TW + t, 4 * g + r);
            if (in[i] && kd < a.K) ga.d_initial[(head * a.K + kd) * a.V + col0 + 16 * i] = ds[i][t][r];
          }
    }
  } else {   // ---- what depends on do alone, of chunk ci while the others are at ci + 1
    const T* dop[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) dop[i] = static_cast<const T*>(ga.d_o) + first + (in[i] ? col0 + 16 * i : a.V - 1);
    int64_t drow[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) drow[r] = (row0 + r) * orow;
    ColumnRows<T, C> d[NC];
    f32x4 into;
    auto load_do = [&](int ci) {
      const int64_t left_rows = len - (int64_t)ci * C;
#pragma unroll
      for (int i = 0; i < NC; ++i) d[i].load(dop[i] + (int64_t)ci * C * orow, drow, orow, (int)(left_rows < C ? left_rows : C), row0);
      into = *reinterpret_cast<const f32x4*>(vec + row0 * 4);
    };
    if (nc > 0) {
      load_do(nc - 1);
      load_x(S::pPT);
      if (holds) load_t(S::fQT);
    }
    // three barriers a chunk, as the others; before the first chunk and without the first one
    for (int ci = nc - 1; ci >= 0; --ci) {
      const bool more = ci > 0;
      if (ci < nc - 1) lds_barrier();
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const f32x4 v = d[i].get(in[i], row0);
        put_half<NP>(part(i, B::bO), w / 2, w & 1, lane, v);
        put_half<3>(part(i, B::bE), w / 2, w & 1, lane, (a.scale * into) * v);
      }
      if (more) kq -= kq_step, xp -= xp_step, vec -= vec_step;
      load_do(more ? ci - 1 : ci);
      lds_barrier();
#pragma unroll
      for (int i = 0; i < NC; ++i)
        *reinterpret_cast<f32x4*>(part(i, B::bP) + w * 1024 + at16) =
            product<3, NP, 3, S::CS>(fx, [&](int s, bf16x8(&b)[NP]) { get_operand<NP>(part(i, B::bO), s, lane, b); });
      load_x(S::pPT);
      lds_barrier();
      if (holds) {
#pragma unroll
        for (int i = 0; i < NC; ++i) {
          f32x4 q[TW];
#pragma unroll
          for (int t = 0; t < TW; ++t) q[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int s = 0; s < S::CS; ++s) {
            bf16x8 ep[3];
            get_operand<3>(part(i, B::bE), s, lane, ep);
            mfma_rows<NP, 3, 3, TW>([&](int t) -> const bf16x8(&)[NP] { return ft[t][s]; }, ep, q);
          }
#pragma unroll
          for (int t = 0; t < TW; ++t)
            *reinterpret_cast<f32x4*>(part(i, B::bQ) + ((ci & 1) * S::KT + w * TW + t) * 1024 + at16) = q[t];
        }
        load_t(S::fQT);
      }
    }
    if (nc > 0) {   // the others' last chunk
      lds_barrier();
      lds_barrier();
      lds_barrier();
    }
  }
}

// ----------------------------------------------------------------------------------- the rest, chunk by chunk

constexpr int kSlice = 32;              // values of v taken at a time

template <int DT, int KP, int C>
struct GradLds {
  using S = DeltaShape<DT, KP, C, true>;
  static constexpr int kST = C * kSlice, kMT = C * C;   // values of a staged plane, of a plane of m or n
  static constexpr int stage = (S::NP + 6) * kST * 2, mats = 2 * S::NO * kMT * 2;
  static constexpr int kq = 0, work = 2 * S::NP * C * KP * 2, vec = work + (stage > mats ? stage : mats);
  // G hi, G lo, beta, exp(G), exp(G_63 - G), dR . v, column sums; row sums of m q.k + n k.k, of -D N k.k, of q X, k Y, k Z
  // by wave; <S, dS> by wave
  static constexpr int bytes = vec + (7 + 5 * S::RT) * C * 4 + 32;
};


template <int NP, int TILE>
__device__ __forceinline__ float whole(const __bf16* p) {
  float v = (float)p[(NP - 1) * TILE];
#pragma unroll
  for (int i = NP - 2; i >= 0; --i) v += (float)p[i * TILE];
  return v;
}

// A workgroup takes one chunk and value head: 32 columns of v at a time into LDS as planes, a wave for 16 rows of M and N and a
// share of K's columns.  Bound by the latency of its products; at 64 rows it keeps to 256 registers, so that two workgroups of four
// waves are on a unit, though heads of 128 spill 47 registers a lane for that (f32: 67).  1024 chunks and heads of 128 x 128, bf16: 119
// us (one workgroup at a time took 1.36 times as long); the 295 MB that it moves would take 58 us.
template <int DT, int KP, int C>
__global__ __launch_bounds__(4 * C, C == 64 ? 2 : 1) void k_delta_grad(DeltaGradArgs ga, bool wide_v, bool wide_o) {
  using S = DeltaShape<DT, KP, C, true>;
  using L = GradLds<DT, KP, C>;
  using T = typename Elem<DT>::T;
  constexpr int NP = S::NP, NO = S::NO, RT = S::RT, kST = L::kST, kMT = L::kMT, kTile = C * KP;
  constexpr int NT = S::KT >= RT ? S::KT / RT : 1;   // 16-column tiles of K a wave owns
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const DeltaArgs& a = ga.f;
  __bf16* const Kt = reinterpret_cast<__bf16*>(lds);
  __bf16* const Qt = Kt + NP * kTile;
  __bf16* const dO = reinterpret_cast<__bf16*>(lds + L::work);
  __bf16* const dR = dO + NP * kST;
  __bf16* const uu = dR + 3 * kST;
  __bf16* const mt_ = reinterpret_cast<__bf16*>(lds + L::work);   // m, n: after the value axis is done
  __bf16* const nt_ = mt_ + NO * kMT;
  float* const ghi = reinterpret_cast<float*>(lds + L::vec);
  float *const glo = ghi + C, *const bet = ghi + 2 * C, *const into = ghi + 3 * C, *const left = ghi + 4 * C;
  float *const rv = ghi + 5 * C, *const cols = ghi + 6 * C, *const rsum = ghi + 7 * C, *const rnb = rsum + RT * C;
  float *const qx = rnb + RT * C, *const ky = qx + RT * C, *const kz = ky + RT * C, *const sds = kz + RT * C;

  const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
  int x = lane & 15, g = lane >> 4;
  const int64_t c = blockIdx.x / a.Hv;
  const int h = (int)(blockIdx.x % a.Hv), hk = h / (a.Hv / a.Hk);
  const int64_t n = a.rows.find(c);
  int64_t begin, len, chunk0;
  a.rows.range(n, begin, len, chunk0);
  const int64_t t0 = (c - chunk0) * C;
  if (t0 < 0 || t0 >= len) return;
  const int rows = (int)(len - t0 < C ? len - t0 : C);
  const int64_t bt = a.rows.batch(n), r0 = begin + t0, ch = c * a.Hv + h;

  {   // K and Q rows from their fragments
    const char* kq = a.kq + (c * a.Hk + hk) * (int64_t)S::kKQ + lane * 16;
#pragma unroll 4
    for (int f = wave; f < 2 * RT * S::KS * NP; f += RT) {
      const int e = f / NP, t = e / S::KS % RT, s = e % S::KS, w = e / (RT * S::KS);
      *reinterpret_cast<bf16x8*>(Kt + (w * NP + f % NP) * kTile + tile_at<KP>(perm_row(t, x), 4 * s + g)) =
          *reinterpret_cast<const bf16x8*>(kq + f * 1024);
    }
  }
  float graw = 0.f;
  if (wave == 0) {
    graw = lane < rows ? a.g[bt * a.gs[0] + (r0 + lane) * a.gs[1] + h * a.gs[2]] : 0.f;
    double last;
    const double sum = running_sum(graw < kMinG ? kMinG : graw, lane, last);
    const float hi = (float)sum;
    const float* vec = reinterpret_cast<const float*>(a.vec + ch * (int64_t)kVec);
    if (lane < C) {
      ghi[lane] = hi;
      glo[lane] = (float)(sum - (double)hi);
      into[lane] = vec[lane];
      left[lane] = vec[64 + lane];
      bet[lane] = vec[128 + lane];
    }
  }

  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  f32x4 X1[RT][NT], Y[RT][NT], Z[RT][NT], M[RT], N[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    M[i] = N[i] = zero;
#pragma unroll
    for (int j = 0; j < NT; ++j) X1[i][j] = Y[i][j] = Z[i][j] = zero;
  }
  const float* s0 = a.s0 + ch * (int64_t)KP * a.VP;
  const float* dse = ga.ds + ch * (int64_t)KP * a.VP;
  const bool active = wave * NT < S::KT;
  float dot = 0.f, rdot = 0.f;
  {
    const int row = tid >> 2, p = tid & 3;
    const float* rp = ga.dr + (ch * C + row) * (int64_t)a.VP + 8 * p;
    const float* up = a.u + (ch * C + row) * (int64_t)a.VP + 8 * p;
    const T* op = static_cast<const T*>(ga.d_o) + ((bt * a.rows.T + r0 + row) * a.Hv + h) * (int64_t)a.V + 8 * p;
    const T* vp = static_cast<const T*>(a.v) + bt * a.vs[0] + (r0 + row) * a.vs[1] + h * a.vs[2] + 8 * p;
    const int at = tile_at<kSlice>(row, p);
    for (int v0 = 0; v0 < a.VP; v0 += kSlice) {
      const int lv = a.V - v0 - 8 * p;
      f32x8 dov = {}, drv = {}, uv = {}, vv = {};
      here(g, x);
      f32x8 sv[NT] = {}, dv[NT] = {};
      if (active && v0 + 8 * g < a.VP) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const uint32_t o = (16 * (wave * NT + j) + x) * a.VP + v0 + 8 * g;
          sv[j] = load8(&item(s0, o), 8, true);
          dv[j] = load8(&item(dse, o), 8, true);
        }
      }
      if (v0 + 8 * p < a.VP) {
        drv = load8(rp + v0, 8, true);
        uv = load8(up + v0, 8, true);
        if (row < rows && lv > 0) {
          dov = load8(op + v0, lv, wide_o);
          vv = load8(vp + v0, lv, wide_v);
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) rdot = fmaf(drv[i], vv[i], rdot);
      bf16x8 po[NP], p3[3];
      lds_barrier();   // the last slice is done with
      planes8<NP>(dov, po);
#pragma unroll
      for (int i = 0; i < NP; ++i) *reinterpret_cast<bf16x8*>(dO + i * kST + at) = po[i];
      planes8<3>(drv, p3);
#pragma unroll
      for (int i = 0; i < 3; ++i) *reinterpret_cast<bf16x8*>(dR + i * kST + at) = p3[i];
      planes8<3>(uv, p3);
#pragma unroll
      for (int i = 0; i < 3; ++i) *reinterpret_cast<bf16x8*>(uu + i * kST + at) = p3[i];
      lds_barrier();
      bf16x8 fu[3];
      frag<kSlice, 3, kST>(uu, 16 * wave + x, 0, g, fu);
      bf16x8 sp[NT][3], dp[NT][3];
      if (active) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
#pragma unroll
          for (int i = 0; i < 8; ++i) dot = fmaf(sv[j][i], dv[j][i], dot);
          planes8<3>(sv[j], sp[j]);
          planes8<3>(dv[j], dp[j]);
        }
      }
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        bf16x8 fo[NP], fr[3], fi[3];
        frag<kSlice, NP, kST>(dO, 16 * i + x, 0, g, fo);
        frag<kSlice, 3, kST>(dR, 16 * i + x, 0, g, fr);
        if (i >= wave) {
          M[i] = mfma_planes<NP, 3, 3>(fo, fu, M[i]);
          N[i] = mfma_planes<3, 3, 3>(fr, fu, N[i]);
        }
        if (active) {
          frag<kSlice, 3, kST>(uu, 16 * i + x, 0, g, fi);
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            X1[i][j] = mfma_planes<NP, 3, 3>(fo, sp[j], X1[i][j]);
            Y[i][j] = mfma_planes<3, 3, 3>(fr, sp[j], Y[i][j]);
            Z[i][j] = mfma_planes<3, 3, 3>(fi, dp[j], Z[i][j]);
          }
        }
        __builtin_amdgcn_sched_barrier(0);   // (the next row tile's operands would not fit in the registers too)
      }
    }
  }
  mfma_settle();
  rdot += __shfl_xor(rdot, 1);
  rdot += __shfl_xor(rdot, 2);
  if ((tid & 3) == 0) rv[tid >> 2] = rdot;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) dot += __shfl_xor(dot, d);
  if (lane == 0) sds[wave] = dot;
  lds_barrier();   // K and Q are in; the staged values are done with

  here(g, x);
  // m and n: the lane's column j = 16 wave + x, rows 16 i + 4 g..+3
  {
    const int j = 16 * wave + x;
    f32x4 qk[RT], kk[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) qk[i] = kk[i] = zero;
#pragma unroll
    for (int s = 0; s < KP / 32; ++s) {
      bf16x8 kb[NP], fa[NP];
      frag<KP, NP, kTile>(Kt, j, s, g, kb);
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        if (i < wave) continue;
        frag<KP, NP, kTile>(Qt, 16 * i + x, s, g, fa);
        qk[i] = mfma_planes<NP, NP, 3>(fa, kb, qk[i]);
        frag<KP, NP, kTile>(Kt, 16 * i + x, s, g, fa);
        kk[i] = mfma_planes<NP, NP, 3>(fa, kb, kk[i]);
      }
    }
    mfma_settle();
    float csum = 0.f;
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 16 * i + 4 * g + r;
        const float d = row >= j ? expf((ghi[row] - ghi[j]) + (glo[row] - glo[j])) : 0.f;
        const float m = row >= j ? a.scale * d * M[i][r] : 0.f;
        const float nb = row > j ? -d * N[i][r] : 0.f;
        const float nn = bet[row] * nb;
        const float e = row > j ? fmaf(m, qk[i][r], nn * kk[i][r]) : 0.f;
        csum += e;
        const float rs = sum16(e), rb = sum16(row > j ? nb * kk[i][r] : 0.f);
        if (x == 0) {
          rsum[wave * C + row] = rs;
          rnb[wave * C + row] = rb;
        }
        const int at = tile_at<C>(row, j >> 3) + (j & 7);
        float rm = m, rn = nn;
#pragma unroll
        for (int p = 0; p < NO; ++p) {
          const __bf16 bm = (__bf16)rm, bn = (__bf16)rn;
          mt_[p * kMT + at] = bm;
          nt_[p * kMT + at] = bn;
          rm -= (float)bm;
          rn -= (float)bn;
        }
      }
    csum += __shfl_xor(csum, 16);
    csum += __shfl_xor(csum, 32);
    if (g == 0) cols[j] = csum;
  }
  lds_barrier();

  here(g, x);
  // dq and dk: the lane's column 16 (wave NT + j) + x, rows 16 i + 4 g..+3
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = 16 * i + 4 * g + r;
      float sq = 0.f, sy = 0.f, sz = 0.f;
      if (active) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const int kd = 16 * (wave * NT + j) + x;
          const int at = tile_at<KP>(row, kd >> 3) + (kd & 7);
          const float kv = whole<NP, kTile>(Kt + at), qv = whole<NP, kTile>(Qt + at);
          const float xs = a.scale * into[row] * X1[i][j][r], ys = into[row] * Y[i][j][r], zs = left[row] * Z[i][j][r];
          sq = fmaf(qv, xs, sq);
          sy = fmaf(kv, ys, sy);
          sz = fmaf(kv, zs, sz);
          X1[i][j][r] = xs;
          Y[i][j][r] = fmaf(-bet[row], ys, zs);
        }
      }
      sq = sum16(sq), sy = sum16(sy), sz = sum16(sz);
      if (x == 0) {
        qx[wave * C + row] = sq;
        ky[wave * C + row] = sy;
        kz[wave * C + row] = sz;
      }
    }
  if (active) {
#pragma unroll
    for (int s = 0; s < S::CS; ++s) {
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        bf16x8 kb[NP], qb[NP];
        frag_col<KP, NP, kTile>(Kt, wave * NT + j, s, g, x, kb);
        frag_col<KP, NP, kTile>(Qt, wave * NT + j, s, g, x, qb);
#pragma unroll
        for (int i = 0; i < RT; ++i) {
          bf16x8 fa[NO];
          if (s <= i / 2) {   // rows i of m and n have columns up to the diagonal
            frag<C, NO, kMT>(mt_, 16 * i + x, s, g, fa);
            X1[i][j] = mfma_planes<NO, NP, NO>(fa, kb, X1[i][j]);
            frag<C, NO, kMT>(nt_, 16 * i + x, s, g, fa);
            Y[i][j] = mfma_planes<NO, NP, NO>(fa, kb, Y[i][j]);
          }
          if (s >= i / 2) {
            frag_col<C, NO, kMT>(mt_, i, s, g, x, fa);
            Y[i][j] = mfma_planes<NO, NP, NO>(fa, qb, Y[i][j]);
            frag_col<C, NO, kMT>(nt_, i, s, g, x, fa);
            Y[i][j] = mfma_planes<NO, NP, NO>(fa, kb, Y[i][j]);
          }
        }
      }
    }
    mfma_settle();
    const int64_t first = bt * a.rows.T + r0;
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 16 * i + 4 * g + r;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const int kd = 16 * (wave * NT + j) + x;
          if (row >= rows || kd >= a.K) continue;
          if (ga.dq32) {
            const int64_t at = ((first + row) * a.Hv + h) * a.K + kd;
            ga.dq32[at] = X1[i][j][r];
            ga.dk32[at] = Y[i][j][r];
          } else {
            const int64_t at = ((first + row) * a.Hk + hk) * a.K + kd;
            static_cast<T*>(ga.dq)[at] = (T)X1[i][j][r];
            static_cast<T*>(ga.dk)[at] = (T)Y[i][j][r];
          }
        }
      }
  }
  lds_barrier();
  if (wave == 0) {
    const int at = lane < C ? lane : 0;
    auto waves = [&](const float* p) {
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < RT; ++i) v += p[i * C + at];
      return lane < C ? v : 0.f;
    };
    const float y = waves(ky), z = waves(kz);
    // columns right of the diagonal tile hold zeros in rsum and rnb: every wave writes every row
    const double own = lane < C ? (double)waves(rsum) - cols[at] + waves(qx) - bet[at] * y - z : 0.0;
    double tail, zall;
    const double upto = running_sum64(own, lane, tail);
    running_sum64(z, lane, zall);
    const float all = reinterpret_cast<const float*>(a.vec + ch * (int64_t)kVec)[192];
    float dots = 0.f;
#pragma unroll
    for (int i = 0; i < RT; ++i) dots += sds[i];
    const double end = zall + (double)all * dots;
    if (lane < rows) {
      const int64_t to = (bt * a.rows.T + r0 + lane) * a.Hv + h;
      ga.dg[to] = graw < kMinG ? 0.f : (float)(end + tail - upto + own);
      ga.dbeta[to] = rv[lane] - y + waves(rnb);
    }
  }
}

// shares of the value heads of one query/key head, added up in order
template <class T>
__global__ void k_delta_heads(const float* dq32, const float* dk32, T* dq, T* dk, int64_t n, int group, int K) {
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t at = i / K * group * K + i % K;
    float q = 0.f, k = 0.f;
    for (int e = 0; e < group; ++e) {
      q += dq32[at + (int64_t)e * K];
      k += dk32[at + (int64_t)e * K];
    }
    dq[i] = (T)q;
    dk[i] = (T)k;
  }
}

template <int DT, int KP, int C, int NC>
hipError_t back(const DeltaGradArgs& ga, hipStream_t s) {
  constexpr int bytes = Back<DT, KP, C, NC>::bytes;
  const DeltaArgs& a = ga.f;
  const hipError_t e = allow_lds(k_delta_back<DT, KP, C, NC>, bytes);
  if (e != hipSuccess) return e;
  const int groups = (a.VP / 16 + NC - 1) / NC;
  k_delta_back<DT, KP, C, NC><<<column_blocks(a, groups), 8 * C, bytes, s>>>(ga);
  return hipGetLastError();
}

template <int DT, int KP, int C>
hipError_t backward(const DeltaGradArgs& ga, bool wide_v, bool wide_o, hipStream_t s) {
  constexpr int bytes = GradLds<DT, KP, C>::bytes;
  const DeltaArgs& a = ga.f;
  hipError_t e = a.wide_cols ? back<DT, KP, C, 2>(ga, s) : back<DT, KP, C, 1>(ga, s);
  if (e != hipSuccess) return e;
  e = allow_lds(k_delta_grad<DT, KP, C>, bytes);
  if (e != hipSuccess) return e;
  if (a.chunks) k_delta_grad<DT, KP, C><<<(unsigned)(a.chunks * a.Hv), 4 * C, bytes, s>>>(ga, wide_v, wide_o);
  return hipGetLastError();
}

template <class T>
void heads(const DeltaGradArgs& ga, hipStream_t s) {
  const DeltaArgs& a = ga.f;
  const int64_t rows = a.rows.off ? a.rows.T : a.rows.N * a.rows.T, n = rows * a.Hk * a.K, want = (n + 255) / 256;
  if (n) k_delta_heads<T><<<(unsigned)(want < 8192 ? want : 8192), 256, 0, s>>>(
             ga.dq32, ga.dk32, static_cast<T*>(ga.dq), static_cast<T*>(ga.dk), n, a.Hv / a.Hk, a.K);
}

template <int DT, int KP>
hipError_t backward(const DeltaGradArgs& ga, bool wide_v, bool wide_o, hipStream_t s) {
  return ga.f.rows.C == 32 ? backward<DT, KP, 32>(ga, wide_v, wide_o, s) : backward<DT, KP, 64>(ga, wide_v, wide_o, s);
}

template <int DT>
hipError_t backward(const DeltaGradArgs& ga, int KP, bool wide_v, bool wide_o, hipStream_t s) {
  return KP == 32 ? backward<DT, 32>(ga, wide_v, wide_o, s)
         : KP == 64 ? backward<DT, 64>(ga, wide_v, wide_o, s) : backward<DT, 128>(ga, wide_v, wide_o, s);
}

}  // namespace

hipError_t delta_backward(const DeltaGradArgs& ga, int dtype, int KP, bool wide_v, bool wide_o, hipStream_t s) {
  return dtype == SEQ_BF16 ? backward<SEQ_BF16>(ga, KP, wide_v, wide_o, s)
         : dtype == SEQ_FP16 ? backward<SEQ_FP16>(ga, KP, wide_v, wide_o, s)
                             : backward<SEQ_FP32>(ga, KP, wide_v, wide_o, s);
}

// dq and dk of the query/key heads from their value heads' shares
hipError_t delta_heads(const DeltaGradArgs& ga, int dtype, hipStream_t s) {
  if (dtype == SEQ_BF16) heads<__bf16>(ga, s);
  else if (dtype == SEQ_FP16) heads<_Float16>(ga, s);
  else heads<float>(ga, s);
  return hipGetLastError();
}

}  // namespace seq
