// seq_delta_grad.hip -- gradients of the gated delta rule (seq_delta.hpp has the forward's formulas and names).
//
// With dS the gradient of the state behind a chunk, do that of o, R = beta (v - exp(G) K S) and u = X R:
//     du = P^T do + exp(G_63 - G) K dS,   dR = X^T du,   dv = beta dR,
//     dS <- exp(G_63) dS + scale Q^T (exp(G) do) - K^T (exp(G) beta dR).
// Again only these products run in order (backwards), and again each column by itself: k_delta_back, the mirror image of
// k_delta_scan.  It leaves dS and dR of every chunk; all other gradients follow chunk by chunk (k_delta_grad), from products
// over the value axis, with M = do u^T, N = dR u^T, and masked by i >= j (M) and i > j (N):
//     m = scale D M,  n = -beta_i D N,
//     dq = scale exp(G) do S^T + m K
//     dk = exp(G_63 - G) u dS^T - exp(G) beta dR S^T + m^T Q + (n + n^T) K
//     dbeta_i = dR_i . v_i - exp(G_i) k_i . (S dR_i) - sum_j D_ij N_ij (k_i . k_j)
//     dG_i = q_i . (scale exp(G_i) S do_i) - beta_i exp(G_i) k_i . (S dR_i) - exp(G_63 - G_i) k_i . (dS u_i)
//            + sum_j (m q.k + n k.k)_ij - sum_j (m q.k + n k.k)_ji
//     dG_63 += exp(G_63) <S, dS> + sum_i exp(G_63 - G_i) k_i . (dS u_i),    dg_t = sum_{i >= t} dG_i.
#include "seq_delta_dev.hpp"

namespace seq {
namespace {

template <int DT, int KP, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void k_delta_back(DeltaGradArgs ga) {
  using S = DeltaShape<DT, KP, true>;
  using T = typename Elem<DT>::T;
  constexpr int NP = S::NP, NB = scan_bufs<DT, KP, true>(), KS = KP / 32;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const DeltaArgs& a = ga.f;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, x = lane & 15, g = lane >> 4;
  const int vg = (a.VP / 16 + WAVES - 1) / WAVES;
  const int64_t heads = a.rows.N * a.Hv;
  const int64_t head = (int64_t)(blockIdx.x / 8 / vg) * 8 + blockIdx.x % 8;
  if (head >= heads) return;
  const int64_t n = head / a.Hv;
  const int h = (int)(head % a.Hv), hk = h / (a.Hv / a.Hk);
  const int col = ((int)(blockIdx.x / 8 % vg) * WAVES + wave) * 16 + x;
  const bool in = col < a.V;
  int64_t begin, len, c0;
  a.rows.range(n, begin, len, c0);
  const int64_t nc = (len + kC - 1) / kC;

  f32x4 ds[KP / 16];
#pragma unroll
  for (int t = 0; t < KP / 16; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int kd = perm_row(t, 4 * g + r);
      ds[t][r] = ga.d_final && in && kd < a.K ? ga.d_final[(head * a.K + kd) * a.V + col] : 0.f;
    }
  const int64_t first = ((a.rows.batch(n) * a.rows.T + begin) * a.Hv + h) * (int64_t)a.V + col;
  const int64_t orow = (int64_t)a.Hv * a.V;
  const T* dop = static_cast<const T*>(ga.d_o) + first;
  T* dvp = static_cast<T*>(ga.dv) + first;
  f32x4 d[4];
  auto load_do = [&](int64_t t0) {
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int64_t row = t0 + perm_row(t, 4 * g + r);
        d[t][r] = in && row < len ? (float)dop[row * orow] : 0.f;
      }
  };
  if (nc > 0) {
    stage_chunk<S, WAVES>(a, c0 + nc - 1, hk, h, lds, wave, lane);
    load_do((nc - 1) * kC);
  }
  for (int64_t ci = nc - 1; ci >= 0; --ci) {
    const char* buf = lds + (NB == 2 ? ((nc - 1 - ci) & 1) * S::kStage : 0);
    vm_wait();
    __syncthreads();
    f32x4 dc[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) dc[t] = d[t];
    if (ci > 0) {
      if (NB == 2) stage_chunk<S, WAVES>(a, c0 + ci - 1, hk, h, lds + ((nc - ci) & 1) * S::kStage, wave, lane);
      load_do((ci - 1) * kC);
    }
    const __bf16* Kt = reinterpret_cast<const __bf16*>(buf);
    const __bf16* Qt = Kt + NP * S::kTile;
    const __bf16* Xt = reinterpret_cast<const __bf16*>(buf + S::kKQ);
    const __bf16* Pt = Xt + 3 * kTri;
    const float* vec = reinterpret_cast<const float*>(buf + S::kKQ + S::kXP);
    const int64_t ch = (c0 + ci) * a.Hv + h;
    if (col < a.VP) {
      float* p = ga.ds + ch * (int64_t)KP * a.VP + col;
#pragma unroll
      for (int t = 0; t < KP / 16; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) p[(int64_t)perm_row(t, 4 * g + r) * a.VP] = ds[t][r];
    }
    // du = exp(G_63 - G) K dS + P^T do
    f32x4 du[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) du[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      bf16x8 sp[3];
      planes8<3>(cat8(ds[2 * s], ds[2 * s + 1]), sp);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        bf16x8 fa[NP];
        frag<KP, NP, S::kTile>(Kt, perm_row(t, x), s, g, fa);
        du[t] = mfma_planes<NP, 3, 3>(fa, sp, du[t]);
      }
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) du[t] *= *reinterpret_cast<const f32x4*>(vec + kC + perm_row(t, 4 * g));
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      bf16x8 dp[NP];
      planes8<NP>(cat8(dc[2 * s], dc[2 * s + 1]), dp);
#pragma unroll
      for (int t = 0; t < 2 + 2 * s; ++t) {
        bf16x8 fa[3];
        frag_tri_t(Pt, t, s, g, x, fa);
        du[t] = mfma_planes<3, NP, 3>(fa, dp, du[t]);
      }
    }
    // dR = X^T du
    f32x4 dr[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) dr[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      bf16x8 dp[3];
      planes8<3>(cat8(du[2 * s], du[2 * s + 1]), dp);
#pragma unroll
      for (int t = 0; t < 2 + 2 * s; ++t) {
        bf16x8 fa[3];
        frag_tri_t(Xt, t, s, g, x, fa);
        dr[t] = mfma_planes<3, 3, 3>(fa, dp, dr[t]);
      }
    }
    if (col < a.VP) {
      float* p = ga.dr + ch * (int64_t)kC * a.VP + col;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) p[(int64_t)perm_row(t, 4 * g + r) * a.VP] = dr[t][r];
    }
    const float all = vec[3 * kC];
#pragma unroll
    for (int t = 0; t < KP / 16; ++t) ds[t] *= all;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int i0 = perm_row(t, 4 * g);
      const f32x4 into = *reinterpret_cast<const f32x4*>(vec + i0), b = *reinterpret_cast<const f32x4*>(vec + 2 * kC + i0);
      const f32x4 dv = b * dr[t];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int64_t row = ci * kC + i0 + r;
        if (in && row < len) dvp[row * orow] = (T)dv[r];
      }
      dc[t] *= a.scale * into;
      dr[t] = -into * dv;
    }
    // dS <- exp(G_63) dS + scale Q^T (exp(G) do) - K^T (exp(G) beta dR)
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      bf16x8 dp[3], rp[3];
      planes8<3>(cat8(dc[2 * s], dc[2 * s + 1]), dp);
      planes8<3>(cat8(dr[2 * s], dr[2 * s + 1]), rp);
#pragma unroll
      for (int t = 0; t < KP / 16; ++t) {
        bf16x8 fa[NP];
        frag_t<KP, NP, S::kTile>(Qt, t, s, g, x, fa);
        ds[t] = mfma_planes<NP, 3, 3>(fa, dp, ds[t]);
        frag_t<KP, NP, S::kTile>(Kt, t, s, g, x, fa);
        ds[t] = mfma_planes<NP, 3, 3>(fa, rp, ds[t]);
      }
    }
    if (NB == 1 && ci > 0) {
      __syncthreads();
      stage_chunk<S, WAVES>(a, c0 + ci - 1, hk, h, lds, wave, lane);
    }
  }
  if (ga.d_initial && in) {
#pragma unroll
    for (int t = 0; t < KP / 16; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int kd = perm_row(t, 4 * g + r);
        if (kd < a.K) ga.d_initial[(head * a.K + kd) * a.V + col] = ds[t][r];
      }
  }
}

// ----------------------------------------------------------------------------------- the rest, chunk by chunk

constexpr int kSlice = 32;              // values of v taken at a time
constexpr int kST = kC * kSlice;        // values of a staged plane
constexpr int kMT = kC * kC;            // values of a plane of m or n

template <int DT, int KP>
struct GradLds {
  using S = DeltaShape<DT, KP, true>;
  static constexpr int stage = (S::NP + 6) * kST * 2, mats = 2 * S::NO * kMT * 2;
  static constexpr int kq = 0, work = S::kKQ, vec = work + (stage > mats ? stage : mats);
  // G hi, G lo, beta, exp(G), exp(G_63 - G), dR . v, column sums; row sums of m q.k + n k.k, of -D N k.k, of q X, k Y, k Z
  // by wave; <S, dS> by wave
  static constexpr int bytes = vec + (7 + 5 * 4) * kC * 4 + 4 * 4 + 16;
};

__device__ __forceinline__ float sum16(float v) {
#pragma unroll
  for (int d = 1; d < 16; d *= 2) v += __shfl_xor(v, d);
  return v;
}

template <int NP, int TILE>
__device__ __forceinline__ float whole(const __bf16* p) {
  float v = (float)p[(NP - 1) * TILE];
#pragma unroll
  for (int i = NP - 2; i >= 0; --i) v += (float)p[i * TILE];
  return v;
}

template <int DT, int KP>
__global__ __launch_bounds__(256) void k_delta_grad(DeltaGradArgs ga, bool wide_v, bool wide_o) {
  using S = DeltaShape<DT, KP, true>;
  using L = GradLds<DT, KP>;
  using T = typename Elem<DT>::T;
  constexpr int NP = S::NP, NO = S::NO, NT = KP >= 64 ? KP / 64 : 1;   // 16-column tiles of K a wave owns
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const DeltaArgs& a = ga.f;
  __bf16* const Kt = reinterpret_cast<__bf16*>(lds);
  __bf16* const Qt = Kt + NP * S::kTile;
  __bf16* const dO = reinterpret_cast<__bf16*>(lds + L::work);
  __bf16* const dR = dO + NP * kST;
  __bf16* const uu = dR + 3 * kST;
  __bf16* const mt_ = reinterpret_cast<__bf16*>(lds + L::work);   // m, n: after the value axis is done
  __bf16* const nt_ = mt_ + NO * kMT;
  float* const ghi = reinterpret_cast<float*>(lds + L::vec);
  float *const glo = ghi + kC, *const bet = ghi + 2 * kC, *const into = ghi + 3 * kC, *const left = ghi + 4 * kC;
  float *const rv = ghi + 5 * kC, *const cols = ghi + 6 * kC, *const rsum = ghi + 7 * kC, *const rnb = rsum + 4 * kC;
  float *const qx = rnb + 4 * kC, *const ky = qx + 4 * kC, *const kz = ky + 4 * kC, *const sds = kz + 4 * kC;

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, x = lane & 15, g = lane >> 4;
  const int64_t c = blockIdx.x / a.Hv;
  const int h = (int)(blockIdx.x % a.Hv), hk = h / (a.Hv / a.Hk);
  const int64_t n = a.rows.find(c);
  int64_t begin, len, chunk0;
  a.rows.range(n, begin, len, chunk0);
  const int64_t t0 = (c - chunk0) * kC;
  if (t0 < 0 || t0 >= len) return;
  const int rows = (int)(len - t0 < kC ? len - t0 : kC);
  const int64_t bt = a.rows.batch(n), r0 = begin + t0, ch = c * a.Hv + h;

  const char* kq = a.kq + (c * a.Hk + hk) * (int64_t)S::kKQ;
  for (int i = wave; i < S::kKQ / 1024; i += 4) glds16(kq + i * 1024 + lane * 16, lds + i * 1024);
  float graw = 0.f;
  if (wave == 0) {
    graw = lane < rows ? a.g[bt * a.gs[0] + (r0 + lane) * a.gs[1] + h * a.gs[2]] : 0.f;
    double last;
    const double sum = running_sum(graw < kMinG ? kMinG : graw, lane, last);
    const float hi = (float)sum;
    const float* vec = reinterpret_cast<const float*>(a.vec + ch * (int64_t)S::kVec);
    ghi[lane] = hi;
    glo[lane] = (float)(sum - (double)hi);
    into[lane] = vec[lane];
    left[lane] = vec[kC + lane];
    bet[lane] = vec[2 * kC + lane];
  }

  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  f32x4 X1[4][NT], Y[4][NT], Z[4][NT], M[4], N[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    M[i] = N[i] = zero;
#pragma unroll
    for (int j = 0; j < NT; ++j) X1[i][j] = Y[i][j] = Z[i][j] = zero;
  }
  const float* s0 = a.s0 + ch * (int64_t)KP * a.VP;
  const float* dse = ga.ds + ch * (int64_t)KP * a.VP;
  const bool active = wave * NT * 16 < KP;
  float dot = 0.f, rdot = 0.f;
  {
    const int row = tid >> 2, p = tid & 3;
    const float* rp = ga.dr + (ch * kC + row) * (int64_t)a.VP + 8 * p;
    const float* up = a.u + (ch * kC + row) * (int64_t)a.VP + 8 * p;
    const T* op = static_cast<const T*>(ga.d_o) + ((bt * a.rows.T + r0 + row) * a.Hv + h) * (int64_t)a.V + 8 * p;
    const T* vp = static_cast<const T*>(a.v) + bt * a.vs[0] + (r0 + row) * a.vs[1] + h * a.vs[2] + 8 * p;
    const int at = tile_at<kSlice>(row, p);
    for (int v0 = 0; v0 < a.VP; v0 += kSlice) {
      const int lv = a.V - v0 - 8 * p;
      f32x8 dov = {}, drv = {}, uv = {}, vv = {};
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
      __syncthreads();   // the last slice is done with
      planes8<NP>(dov, po);
#pragma unroll
      for (int i = 0; i < NP; ++i) *reinterpret_cast<bf16x8*>(dO + i * kST + at) = po[i];
      planes8<3>(drv, p3);
#pragma unroll
      for (int i = 0; i < 3; ++i) *reinterpret_cast<bf16x8*>(dR + i * kST + at) = p3[i];
      planes8<3>(uv, p3);
#pragma unroll
      for (int i = 0; i < 3; ++i) *reinterpret_cast<bf16x8*>(uu + i * kST + at) = p3[i];
      __syncthreads();
      bf16x8 fu[3];
      frag<kSlice, 3, kST>(uu, 16 * wave + x, 0, g, fu);
      bf16x8 sp[NT][3], dp[NT][3];
      if (active) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          f32x8 sv = {}, dv = {};
          if (v0 + 8 * g < a.VP) {
            const int64_t o = (int64_t)(16 * (wave * NT + j) + x) * a.VP + v0 + 8 * g;
            sv = load8(s0 + o, 8, true);
            dv = load8(dse + o, 8, true);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) dot = fmaf(sv[i], dv[i], dot);
          planes8<3>(sv, sp[j]);
          planes8<3>(dv, dp[j]);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
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
      }
    }
  }
  rdot += __shfl_xor(rdot, 1);
  rdot += __shfl_xor(rdot, 2);
  if ((tid & 3) == 0) rv[tid >> 2] = rdot;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) dot += __shfl_xor(dot, d);
  if (lane == 0) sds[wave] = dot;
  vm_wait();
  __syncthreads();   // K and Q are in; the staged values are done with

  // m and n: the lane's column j = 16 wave + x, rows 16 i + 4 g..+3
  {
    const int j = 16 * wave + x;
    f32x4 qk[4], kk[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) qk[i] = kk[i] = zero;
#pragma unroll
    for (int s = 0; s < KP / 32; ++s) {
      bf16x8 kb[NP], fa[NP];
      frag<KP, NP, S::kTile>(Kt, j, s, g, kb);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i < wave) continue;
        frag<KP, NP, S::kTile>(Qt, 16 * i + x, s, g, fa);
        qk[i] = mfma_planes<NP, NP, 3>(fa, kb, qk[i]);
        frag<KP, NP, S::kTile>(Kt, 16 * i + x, s, g, fa);
        kk[i] = mfma_planes<NP, NP, 3>(fa, kb, kk[i]);
      }
    }
    float csum = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 16 * i + 4 * g + r;
        const float d = row >= j ? expf((ghi[row] - ghi[j]) + (glo[row] - glo[j])) : 0.f;
        const float m = row >= j ? a.scale * d * M[i][r] : 0.f;
        const float nb = row > j ? -d * N[i][r] : 0.f;
        const float nn = bet[row] * nb;
        const float e = row >= j ? fmaf(m, qk[i][r], nn * kk[i][r]) : 0.f;
        csum += e;
        const float rs = sum16(e), rb = sum16(row > j ? nb * kk[i][r] : 0.f);
        if (x == 0) {
          rsum[wave * kC + row] = rs;
          rnb[wave * kC + row] = rb;
        }
        const int at = tile_at<kC>(row, j >> 3) + (j & 7);
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
  __syncthreads();

  // dq and dk: the lane's column 16 (wave NT + j) + x, rows 16 i + 4 g..+3
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = 16 * i + 4 * g + r;
      float sq = 0.f, sy = 0.f, sz = 0.f;
      if (active) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const int kd = 16 * (wave * NT + j) + x;
          const int at = tile_at<KP>(row, kd >> 3) + (kd & 7);
          const float kv = whole<NP, S::kTile>(Kt + at), qv = whole<NP, S::kTile>(Qt + at);
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
        qx[wave * kC + row] = sq;
        ky[wave * kC + row] = sy;
        kz[wave * kC + row] = sz;
      }
    }
  if (active) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        bf16x8 kb[NP], qb[NP];
        frag_col<KP, NP, S::kTile>(Kt, wave * NT + j, s, g, x, kb);
        frag_col<KP, NP, S::kTile>(Qt, wave * NT + j, s, g, x, qb);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          bf16x8 fa[NO];
          if (s <= i / 2) {   // rows i of m and n have columns up to the diagonal
            frag<kC, NO, kMT>(mt_, 16 * i + x, s, g, fa);
            X1[i][j] = mfma_planes<NO, NP, NO>(fa, kb, X1[i][j]);
            frag<kC, NO, kMT>(nt_, 16 * i + x, s, g, fa);
            Y[i][j] = mfma_planes<NO, NP, NO>(fa, kb, Y[i][j]);
          }
          if (s >= i / 2) {
            frag_col<kC, NO, kMT>(mt_, i, s, g, x, fa);
            Y[i][j] = mfma_planes<NO, NP, NO>(fa, qb, Y[i][j]);
            frag_col<kC, NO, kMT>(nt_, i, s, g, x, fa);
            Y[i][j] = mfma_planes<NO, NP, NO>(fa, kb, Y[i][j]);
          }
        }
      }
    }
    const int64_t first = bt * a.rows.T + r0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
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
  __syncthreads();
  if (wave == 0) {
    auto waves = [&](const float* p) { return (p[lane] + p[kC + lane]) + (p[2 * kC + lane] + p[3 * kC + lane]); };
    const float y = waves(ky), z = waves(kz);
    // columns right of the diagonal tile hold zeros in rsum and rnb: every wave writes every row
    const double own = (double)waves(rsum) - cols[lane] + waves(qx) - bet[lane] * y - z;
    double tail, zall;
    const double upto = running_sum64(own, lane, tail);
    running_sum64(z, lane, zall);
    const float all = reinterpret_cast<const float*>(a.vec + ch * (int64_t)S::kVec)[3 * kC];
    const double end = zall + (double)all * ((sds[0] + sds[1]) + (sds[2] + sds[3]));
    if (lane < rows) {
      const int64_t at = (bt * a.rows.T + r0 + lane) * a.Hv + h;
      ga.dg[at] = graw < kMinG ? 0.f : (float)(end + tail - upto + own);
      ga.dbeta[at] = rv[lane] - y + waves(rnb);
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

template <int DT, int KP>
hipError_t backward(const DeltaGradArgs& ga, bool wide_v, bool wide_o, hipStream_t s) {
  using S = DeltaShape<DT, KP, true>;
  using T = typename Elem<DT>::T;
  constexpr int W = 4, bytes = scan_bufs<DT, KP, true>() * S::kStage, glds = GradLds<DT, KP>::bytes;
  const DeltaArgs& a = ga.f;
  hipError_t e = allow_lds(k_delta_back<DT, KP, W>, bytes);
  if (e != hipSuccess) return e;
  e = allow_lds(k_delta_grad<DT, KP>, glds);
  if (e != hipSuccess) return e;
  const int64_t vg = (a.VP / 16 + W - 1) / W, heads = (a.rows.N * a.Hv + 7) / 8 * 8;
  k_delta_back<DT, KP, W><<<(unsigned)(heads * vg), 64 * W, bytes, s>>>(ga);
  if (a.chunks) k_delta_grad<DT, KP><<<(unsigned)(a.chunks * a.Hv), 256, glds, s>>>(ga, wide_v, wide_o);
  if (ga.dq32) {
    const int64_t rows = a.rows.off ? a.rows.T : a.rows.N * a.rows.T, n = rows * a.Hk * a.K;
    const int64_t want = (n + 255) / 256;
    if (n) k_delta_heads<T><<<(unsigned)(want < 8192 ? want : 8192), 256, 0, s>>>(
               ga.dq32, ga.dk32, static_cast<T*>(ga.dq), static_cast<T*>(ga.dk), n, a.Hv / a.Hk, a.K);
  }
  return hipGetLastError();
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

}  // namespace seq
