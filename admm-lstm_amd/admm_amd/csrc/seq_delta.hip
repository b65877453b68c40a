// seq_delta.hip -- the gated delta rule over whole sequences (seq_delta.hpp has the mathematics).
#include "seq_delta_dev.hpp"

namespace seq {
namespace {

// ------------------------------------------------------------------------------------------------- per chunk: X, P

constexpr int kLd = kC + 4;   // row length of the f32 64 x 64 tiles in LDS
constexpr int kLdY = 36;

template <int DT, int KP, bool SAVE>
constexpr int prep_lds() {
  using S = DeltaShape<DT, KP, SAVE>;
  const int mats = 2 * kC * kLd * 4 + 32 * kLdY * 4 + S::kXP;
  return (S::kKQ > mats ? S::kKQ : mats) + 4 * kC * 4;
}

// f32 product of 16 x 16 tiles, inner length 16 n: C += A B with A(m, k) = a[m * lda + k], B(k, n) = b[k * ldb + n]
__device__ __forceinline__ f32x4 mm16(const float* a, int lda, const float* b, int ldb, int n, int lane, f32x4 acc) {
  const int m = lane & 15, g = lane >> 4;
  for (int k = 0; k < 16 * n; k += 4)
    acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[m * lda + k + g], b[(k + g) * ldb + m], acc, 0, 0, 0);
  return acc;
}

template <int DT, int KP, bool SAVE>
__global__ __launch_bounds__(256) void k_delta_prep(DeltaArgs a) {
  using S = DeltaShape<DT, KP, SAVE>;
  using T = typename Elem<DT>::T;
  constexpr int NP = S::NP;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  __bf16* kq = reinterpret_cast<__bf16*>(lds);
  float* const A = reinterpret_cast<float*>(lds);           // after the Gram products: over K and Q
  float* const X = A + kC * kLd;
  float* const Y = X + kC * kLd;
  __bf16* const xp = reinterpret_cast<__bf16*>(Y + 32 * kLdY);
  float* const ghi = reinterpret_cast<float*>(lds + prep_lds<DT, KP, SAVE>() - 4 * kC * 4);
  float* const glo = ghi + kC;
  float* const bet = glo + kC;
  int* const kbad = reinterpret_cast<int*>(bet + kC);   // rows of k that hold a NaN or infinity

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, m = lane & 15, g = lane >> 4;
  const int64_t c = blockIdx.x / a.Hk;
  const int hk = (int)(blockIdx.x % a.Hk);
  const int64_t n = a.rows.find(c);
  int64_t begin, len, chunk0;
  a.rows.range(n, begin, len, chunk0);
  const int64_t t0 = (c - chunk0) * kC;
  if (t0 < 0 || t0 >= len) return;
  const int rows = (int)(len - t0 < kC ? len - t0 : kC);
  const int64_t bt = a.rows.batch(n), r0 = begin + t0;

  // K and Q rows as planes, in LDS and in the work memory
  if (tid < kC) kbad[tid] = 0;
  __syncthreads();
  {
    const T* kp = static_cast<const T*>(a.k) + bt * a.ks[0] + r0 * a.ks[1] + hk * a.ks[2];
    const T* qp = static_cast<const T*>(a.q) + bt * a.qs[0] + r0 * a.qs[1] + hk * a.qs[2];
    for (int i = tid; i < 2 * kC * (KP / 8); i += 256) {
      const int w = i / (kC * (KP / 8)), r = i / (KP / 8) % kC, p = i % (KP / 8);
      const T* src = w ? qp + (int64_t)r * a.qs[1] : kp + (int64_t)r * a.ks[1];
      f32x8 x = {};
      const int left = a.K - 8 * p;
      if (r < rows && left > 0) x = load8(src + 8 * p, left, w ? a.wide_q : a.wide_k);
      if (!w && zero_if_finite(x.lo) + zero_if_finite(x.hi) != 0.f) kbad[r] = 1;
      bf16x8 pl[NP];
      planes8<NP>(x, pl);
#pragma unroll
      for (int j = 0; j < NP; ++j)
        *reinterpret_cast<bf16x8*>(kq + (w * NP + j) * S::kTile + tile_at<KP>(r, p)) = pl[j];
    }
  }
  __syncthreads();
  for (int i = tid; i < kC * NP * (KP / 8); i += 256) {
    const int r = i / (NP * (KP / 8)), j = i / (KP / 8) % NP;
    if (kbad[r]) *reinterpret_cast<u32x4*>(kq + j * S::kTile + tile_at<KP>(r, i % (KP / 8))) = u32x4{0, 0, 0, 0};
  }
  __syncthreads();
  {
    u32x4* dst = reinterpret_cast<u32x4*>(a.kq + (c * a.Hk + hk) * (int64_t)S::kKQ);
    for (int i = tid; i < S::kKQ / 16; i += 256) dst[i] = reinterpret_cast<const u32x4*>(lds)[i];
  }
  // k_i . k_j and q_i . k_j, rows 16 wave..+15, columns up to the diagonal tile
  f32x4 kk[4], qk[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) kk[j] = qk[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < KP / 32; ++s) {
    bf16x8 ka[NP], qa[NP];
    frag<KP, NP, S::kTile>(kq, 16 * wave + m, s, g, ka);
    frag<KP, NP, S::kTile>(kq + NP * S::kTile, 16 * wave + m, s, g, qa);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j > wave) continue;
      bf16x8 kb[NP];
      frag<KP, NP, S::kTile>(kq, 16 * j + m, s, g, kb);
      kk[j] = mfma_planes<NP, NP, 3>(ka, kb, kk[j]);
      qk[j] = mfma_planes<NP, NP, 3>(qa, kb, qk[j]);
    }
  }

  const int group = a.Hv / a.Hk;
  for (int e = 0; e < group; ++e) {
    const int h = hk * group + e;
    const int64_t ch = c * a.Hv + h;
    __syncthreads();   // K, Q (first round) or the last head's tiles are done with
    if (wave == 0) {
      const bool in = lane < rows;
      float gv = in ? a.g[bt * a.gs[0] + (r0 + lane) * a.gs[1] + h * a.gs[2]] : 0.f;
      float bv = in ? a.beta[bt * a.bs[0] + (r0 + lane) * a.bs[1] + h * a.bs[2]] : 0.f;
      gv = gv < kMinG ? kMinG : gv;
      const uint64_t odd = __ballot((gv - gv) + (bv - bv) != 0.f || kbad[lane]);
      const int bad = odd ? __ffsll((unsigned long long)odd) - 1 : kC;
      if (lane >= bad) gv = bv = 0.f;
      double last;
      const double sum = running_sum(gv, lane, last);
      const float hi = (float)sum;
      ghi[lane] = hi;
      glo[lane] = (float)(sum - (double)hi);
      bet[lane] = bv;
      float* vec = reinterpret_cast<float*>(a.vec + ch * (int64_t)S::kVec);
      vec[lane] = expf((float)sum);
      vec[kC + lane] = expf((float)(last - sum));
      vec[2 * kC + lane] = bv;
      vec[3 * kC + lane] = lane == 1 ? (float)bad : expf((float)last);
    }
    __syncthreads();
    for (int i = tid; i < kC * kLd; i += 256) X[i] = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 16 * wave + 4 * g + r, col = 16 * j + m;
        const bool lower = col <= row;
        const float d = lower ? expf((ghi[row] - ghi[col]) + (glo[row] - glo[col])) : 0.f;
        A[row * kLd + col] = col < row ? bet[row] * d * kk[j][r] : 0.f;
        const float p = lower ? a.scale * d * qk[j][r] : 0.f;
        if (row >= 32 || col < 32) {
          __bf16* pp = xp + 3 * kTri + tri_at(row, col >> 3) + (col & 7);
          const __bf16 p0 = (__bf16)p;
          const float q1 = p - (float)p0;
          const __bf16 p1 = (__bf16)q1;
          pp[0] = p0;
          pp[kTri] = p1;
          if constexpr (S::NPP > 2) pp[2 * kTri] = (__bf16)(q1 - (float)p1);
        }
      }
    }
    __syncthreads();
    // X = (I + A)^-1: the four diagonal 16 x 16 blocks by substitution (a lane has one column), then joined in pairs
    if (wave == 0) {
      float x[16];
      const float* blk = A + (16 * g) * kLd + 16 * g;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float t = i == m ? 1.f : 0.f;
#pragma unroll
        for (int j = 0; j < i; ++j) t = fmaf(-blk[i * kLd + j], x[j], t);
        x[i] = t;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) X[(16 * g + i) * kLd + 16 * g + m] = x[i];
    }
    __syncthreads();
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    if (wave < 2) {   // [X11 0; -X22 A21 X11  X22], 16 rows each
      const float* a21 = A + (32 * wave + 16) * kLd + 32 * wave;
      const f32x4 y = mm16(a21, kLd, X + 32 * wave * kLd + 32 * wave, kLd, 1, lane, zero);
#pragma unroll
      for (int r = 0; r < 4; ++r) Y[(16 * wave + 4 * g + r) * kLdY + m] = y[r];
    }
    __syncthreads();
    if (wave < 2) {
      const f32x4 z = mm16(X + (32 * wave + 16) * kLd + 32 * wave + 16, kLd, Y + 16 * wave * kLdY, kLdY, 1, lane, zero);
#pragma unroll
      for (int r = 0; r < 4; ++r) X[(32 * wave + 16 + 4 * g + r) * kLd + 32 * wave + m] = -z[r];
    }
    __syncthreads();
    const int ti = wave >> 1, tj = wave & 1;
    {
      const f32x4 y = mm16(A + (32 + 16 * ti) * kLd, kLd, X + 16 * tj, kLd, 2, lane, zero);
#pragma unroll
      for (int r = 0; r < 4; ++r) Y[(16 * ti + 4 * g + r) * kLdY + 16 * tj + m] = y[r];
    }
    __syncthreads();
    {
      const f32x4 z = mm16(X + (32 + 16 * ti) * kLd + 32, kLd, Y + 16 * tj, kLdY, 2, lane, zero);
#pragma unroll
      for (int r = 0; r < 4; ++r) X[(32 + 16 * ti + 4 * g + r) * kLd + 16 * tj + m] = -z[r];
    }
    __syncthreads();
    for (int i = tid; i < kC * kC / 8; i += 256) {
      const int r = i >> 3, p = i & 7;
      if (r < 32 && p >= 4) continue;
      const f32x4* src = reinterpret_cast<const f32x4*>(X + r * kLd + 8 * p);
      bf16x8 pl[3];
      planes8<3>(cat8(src[0], src[1]), pl);
#pragma unroll
      for (int j = 0; j < 3; ++j) *reinterpret_cast<bf16x8*>(xp + j * kTri + tri_at(r, p)) = pl[j];
    }
    __syncthreads();
    u32x4* dst = reinterpret_cast<u32x4*>(a.xp + ch * (int64_t)S::kXP);
    for (int i = tid; i < S::kXP / 16; i += 256) dst[i] = reinterpret_cast<const u32x4*>(xp)[i];
  }
}

// --------------------------------------------------------------------------------------------- chunk after chunk

template <int DT, int KP, int WAVES, bool SAVE>
__global__ __launch_bounds__(64 * WAVES) void k_delta_scan(DeltaArgs a) {
  using S = DeltaShape<DT, KP, SAVE>;
  using T = typename Elem<DT>::T;
  constexpr int NP = S::NP, NO = S::NO, NB = scan_bufs<DT, KP, SAVE>(), KS = KP / 32;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, x = lane & 15, g = lane >> 4;
  // workgroups go to the eight XCDs in turn: those of one head (which read the same planes) share one XCD's L2
  const int vg = (a.VP / 16 + WAVES - 1) / WAVES;
  const int64_t heads = a.rows.N * a.Hv;
  const int64_t head = (int64_t)(blockIdx.x / 8 / vg) * 8 + blockIdx.x % 8;
  if (head >= heads) return;
  const int64_t n = head / a.Hv;
  const int h = (int)(head % a.Hv), hk = h / (a.Hv / a.Hk);
  const int col = ((int)(blockIdx.x / 8 % vg) * WAVES + wave) * 16 + x;   // the lane's column
  const bool in = col < a.V;
  int64_t begin, len, c0;
  a.rows.range(n, begin, len, c0);
  const int64_t nc = (len + kC - 1) / kC;

  f32x4 st[KP / 16];   // tile t, register r: row perm_row(t, 4 g + r) of the state
#pragma unroll
  for (int t = 0; t < KP / 16; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int kd = perm_row(t, 4 * g + r);
      st[t][r] = a.initial && in && kd < a.K ? a.initial[(head * a.K + kd) * a.V + col] : 0.f;
    }

  const T* vp = static_cast<const T*>(a.v) + a.rows.batch(n) * a.vs[0] + begin * a.vs[1] + h * a.vs[2] + col;
  T* op = static_cast<T*>(a.o) + ((a.rows.batch(n) * a.rows.T + begin) * a.Hv + h) * (int64_t)a.V + col;
  const int64_t orow = (int64_t)a.Hv * a.V;
  f32x4 v[4];   // rows perm_row(t, 4 g + r) of the chunk
  auto load_v = [&](int64_t t0) {
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int64_t row = t0 + perm_row(t, 4 * g + r);
        v[t][r] = in && row < len ? (float)vp[row * a.vs[1]] : 0.f;
      }
  };
  if (nc > 0) {
    stage_chunk<S, WAVES>(a, c0, hk, h, lds, wave, lane);
    load_v(0);
  }
  for (int64_t ci = 0; ci < nc; ++ci) {
    const char* buf = lds + (NB == 2 ? (ci & 1) * S::kStage : 0);
    vm_wait();
    __syncthreads();
    f32x4 vc[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) vc[t] = v[t];
    if (ci + 1 < nc) {
      if (NB == 2) stage_chunk<S, WAVES>(a, c0 + ci + 1, hk, h, lds + ((ci + 1) & 1) * S::kStage, wave, lane);
      load_v((ci + 1) * kC);
    }
    const __bf16* Kt = reinterpret_cast<const __bf16*>(buf);
    const __bf16* Qt = Kt + NP * S::kTile;
    const __bf16* Xt = reinterpret_cast<const __bf16*>(buf + S::kKQ);
    const __bf16* Pt = Xt + 3 * kTri;
    const float* vec = reinterpret_cast<const float*>(buf + S::kKQ + S::kXP);
    const int64_t ch = (c0 + ci) * a.Hv + h;
    if (SAVE && col < a.VP) {
      float* s0 = a.s0 + ch * (int64_t)KP * a.VP + col;
#pragma unroll
      for (int t = 0; t < KP / 16; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) s0[(int64_t)perm_row(t, 4 * g + r) * a.VP] = st[t][r];
    }
    // K S and Q S
    f32x4 ks[4], o[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) ks[t] = o[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      bf16x8 sp[3];
      planes8<3>(cat8(st[2 * s], st[2 * s + 1]), sp);
      bf16x8 so[NO];
#pragma unroll
      for (int i = 0; i < NO; ++i) so[i] = sp[i];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        bf16x8 fa[NP];
        frag<KP, NP, S::kTile>(Kt, perm_row(t, x), s, g, fa);
        ks[t] = mfma_planes<NP, 3, 3>(fa, sp, ks[t]);
        frag<KP, NP, S::kTile>(Qt, perm_row(t, x), s, g, fa);
        o[t] = mfma_planes<NP, NO, NO>(fa, so, o[t]);
      }
    }
    // beta (v - exp(G) K S), and u = X of it
    bf16x8 rp[2][3];
    int bad = (int)vec[3 * kC + 1];
    float odd = 0.f;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int i0 = perm_row(t, 4 * g);
      const f32x4 into = *reinterpret_cast<const f32x4*>(vec + i0), b = *reinterpret_cast<const f32x4*>(vec + 2 * kC + i0);
      ks[t] = b * (vc[t] - into * ks[t]);
      o[t] = (a.scale * into) * o[t];
      odd += zero_if_finite(ks[t]);
    }
    if (__ballot(odd != 0.f)) {
#pragma unroll
      for (int t = 3; t >= 0; --t)
#pragma unroll
        for (int r = 3; r >= 0; --r)
          if (ks[t][r] - ks[t][r] != 0.f) {
            ks[t][r] = 0.f;
            const int row = perm_row(t, 4 * g + r);
            bad = row < bad ? row : bad;
          }
      bad = min(bad, __shfl_xor(bad, 16));
      bad = min(bad, __shfl_xor(bad, 32));
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) planes8<3>(cat8(ks[2 * s], ks[2 * s + 1]), rp[s]);
    f32x4 u[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      u[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s <= t / 2; ++s) {
        bf16x8 fa[3];
        frag_tri(Xt, t, s, g, x, fa);
        u[t] = mfma_planes<3, 3, 3>(fa, rp[s], u[t]);
      }
    }
    const float nan = __builtin_nanf("");
    if (SAVE && col < a.VP) {
      float* us = a.u + ch * (int64_t)kC * a.VP + col;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) us[(int64_t)perm_row(t, 4 * g + r) * a.VP] = perm_row(t, 4 * g + r) >= bad ? nan : u[t][r];
    }
    // o += P u
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      bf16x8 up[NO];
      planes8<NO>(cat8(u[2 * s], u[2 * s + 1]), up);
#pragma unroll
      for (int t = 2 * s; t < 4; ++t) {
        bf16x8 fa[NO];
        frag_tri(Pt, t, s, g, x, fa);
        o[t] = mfma_planes<NO, NO, NO>(fa, up, o[t]);
      }
    }
    // S <- exp(G_63) S + K^T (exp(G_63 - G) u)
    const float all = vec[3 * kC];
#pragma unroll
    for (int t = 0; t < KP / 16; ++t) st[t] *= all;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      bf16x8 up[3];
      const f32x4 l0 = *reinterpret_cast<const f32x4*>(vec + kC + perm_row(2 * s, 4 * g));
      const f32x4 l1 = *reinterpret_cast<const f32x4*>(vec + kC + perm_row(2 * s + 1, 4 * g));
      planes8<3>(cat8(l0 * u[2 * s], l1 * u[2 * s + 1]), up);
#pragma unroll
      for (int t = 0; t < KP / 16; ++t) {
        bf16x8 fa[NP];
        frag_t<KP, NP, S::kTile>(Kt, t, s, g, x, fa);
        st[t] = mfma_planes<NP, 3, 3>(fa, up, st[t]);
      }
    }
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int64_t row = ci * kC + perm_row(t, 4 * g + r);
        if (in && row < len) op[row * orow] = (T)(perm_row(t, 4 * g + r) >= bad ? nan : o[t][r]);
      }
    if (bad < kC) {
#pragma unroll
      for (int t = 0; t < KP / 16; ++t) st[t] = f32x4{nan, nan, nan, nan};
    }
    if (NB == 1 && ci + 1 < nc) {
      __syncthreads();
      stage_chunk<S, WAVES>(a, c0 + ci + 1, hk, h, lds, wave, lane);
    }
  }
  if (in) {
#pragma unroll
    for (int t = 0; t < KP / 16; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int kd = perm_row(t, 4 * g + r);
        if (kd < a.K) a.final[(head * a.K + kd) * a.V + col] = st[t][r];
      }
  }
}

// rows of packed sequences that belong to none: before the first and behind the last.  row: bytes of a row
__global__ void k_delta_outside(DeltaRows rows, void* p, int64_t row) {
  const int64_t first = rows.at(0), last = rows.at(rows.N);
  const int64_t n = (first + (rows.T - (last > first ? last : first))) * row;
  char* q = static_cast<char*>(p);
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i * 2 < n; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t b = i * 2;
    const int64_t at = b < first * row ? b : b - first * row + (last > first ? last : first) * row;
    *reinterpret_cast<uint16_t*>(q + at) = 0;
  }
}

template <int DT, int KP, bool SAVE>
hipError_t forward(const DeltaArgs& a, hipStream_t s) {
  using S = DeltaShape<DT, KP, SAVE>;
  constexpr int W = 4;
  hipError_t e = allow_lds(k_delta_prep<DT, KP, SAVE>, prep_lds<DT, KP, SAVE>());
  if (e != hipSuccess) return e;
  constexpr int bytes = scan_bufs<DT, KP, SAVE>() * S::kStage;
  e = allow_lds(k_delta_scan<DT, KP, W, SAVE>, bytes);
  if (e != hipSuccess) return e;
  if (a.chunks) k_delta_prep<DT, KP, SAVE><<<(unsigned)(a.chunks * a.Hk), 256, (unsigned)prep_lds<DT, KP, SAVE>(), s>>>(a);
  const int64_t vg = (a.VP / 16 + W - 1) / W, heads = (a.rows.N * a.Hv + 7) / 8 * 8;
  k_delta_scan<DT, KP, W, SAVE><<<(unsigned)(heads * vg), 64 * W, bytes, s>>>(a);
  return hipGetLastError();
}

template <int DT, int KP>
hipError_t forward(const DeltaArgs& a, bool save, hipStream_t s) {
  return save ? forward<DT, KP, true>(a, s) : forward<DT, KP, false>(a, s);
}

template <int DT>
hipError_t forward(const DeltaArgs& a, int KP, bool save, hipStream_t s) {
  return KP == 32 ? forward<DT, 32>(a, save, s) : KP == 64 ? forward<DT, 64>(a, save, s) : forward<DT, 128>(a, save, s);
}

}  // namespace

hipError_t delta_outside(const DeltaRows& rows, void* p, int64_t row_bytes, hipStream_t s) {
  k_delta_outside<<<64, 256, 0, s>>>(rows, p, row_bytes);
  return hipGetLastError();
}

hipError_t delta_forward(const DeltaArgs& a, int dtype, int KP, bool save, hipStream_t s) {
  return dtype == SEQ_BF16 ? forward<SEQ_BF16>(a, KP, save, s)
         : dtype == SEQ_FP16 ? forward<SEQ_FP16>(a, KP, save, s) : forward<SEQ_FP32>(a, KP, save, s);
}

}  // namespace seq
