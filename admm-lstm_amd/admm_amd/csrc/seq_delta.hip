// seq_delta.hip -- the gated delta rule over whole sequences (seq_delta.hpp has the mathematics).
#include "seq_delta_dev.hpp"

namespace seq {
namespace {

// ------------------------------------------------------------------------------------------------- per chunk: X, P

constexpr int kLdY = 36;

template <int DT, int KP, int C, bool SAVE>
struct PrepLds {
  using S = DeltaShape<DT, KP, C, SAVE>;
  static constexpr int ld = C + 4;                 // row length of the f32 tiles
  static constexpr int kq = 2 * S::NP * C * KP * 2, mats = (2 * C * ld + (C / 2) * kLdY) * 4;
  static constexpr int vec = kq > mats ? kq : mats;
  static constexpr int bytes = vec + 4 * C * 4;
};

// f32 product of 16 x 16 tiles, inner length 16 n: A(m, k) = a[m * lda + k], B(k, n) = b[k * ldb + n]
__device__ __forceinline__ f32x4 mm16(const float* a, int lda, const float* b, int ldb, int n, int lane) {
  const int m = lane & 15, g = lane >> 4;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int k = 0; k < 16 * n; k += 4)
    acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[m * lda + k + g], b[(k + g) * ldb + m], acc, 0, 0, 0);
  return acc;
}

// eight values of a f32 tile as planes: of row r, columns c..c + 7, or (T) of column r, rows c..c + 7
template <int NP, bool T>
__device__ __forceinline__ void tile_planes(const float* m, int ld, int r, int c, bf16x8 (&p)[NP]) {
  f32x8 v;
  if (T) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = m[(c + i) * ld + r];
  } else {
    v = cat8(*reinterpret_cast<const f32x4*>(m + r * ld + c), *reinterpret_cast<const f32x4*>(m + r * ld + c + 4));
  }
  planes8<NP>(v, p);
}

// Bound by the chain of small products, exchanges and barriers of a chunk: several workgroups on a compute unit cover for each
// other, so the f32 tiles lie where K and Q were, and fragments are cut straight from them.
// 128 chunks of 16 query/key and 32 value heads of 128, bf16: 73 us, about 15 us of it one workgroup's way through; 230 MB written.
template <int DT, int KP, int C, bool SAVE>
__global__ __launch_bounds__(4 * C, DT == SEQ_FP32 ? 2 : 3) void k_delta_prep(DeltaArgs a) {
  using S = DeltaShape<DT, KP, C, SAVE>;
  using L = PrepLds<DT, KP, C, SAVE>;
  using T = typename Elem<DT>::T;
  constexpr int NP = S::NP, W = S::RT, kThreads = 64 * W, kLd = L::ld, kTile = C * KP;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  __bf16* const kq = reinterpret_cast<__bf16*>(lds);
  float* const A = reinterpret_cast<float*>(lds);           // after the Gram products: over K and Q; later P
  float* const X = A + C * kLd;
  float* const Y = X + C * kLd;
  float* const ghi = reinterpret_cast<float*>(lds + L::vec);
  float* const glo = ghi + C;
  float* const bet = glo + C;
  int* const kbad = reinterpret_cast<int*>(bet + C);   // rows of k that hold a NaN or infinity

  const int tid = threadIdx.x, lane = tid & 63, wave = wave_id(), m = lane & 15, g = lane >> 4;
  const int64_t c = blockIdx.x / a.Hk;
  const int hk = (int)(blockIdx.x % a.Hk);
  const int64_t n = a.rows.find(c);
  int64_t begin, len, chunk0;
  a.rows.range(n, begin, len, chunk0);
  const int64_t t0 = (c - chunk0) * C;
  if (t0 < 0 || t0 >= len) return;
  const int rows = (int)(len - t0 < C ? len - t0 : C);
  const int64_t bt = a.rows.batch(n), r0 = begin + t0;

  // the first head's decays and strengths; later ones are fetched while the one before is worked on
  const bool own = wave == 0 && lane < rows;
  float gn = 0.f, bn = 0.f;
  auto fetch = [&](int h) {
    gn = own ? a.g[bt * a.gs[0] + (r0 + lane) * a.gs[1] + h * a.gs[2]] : 0.f;
    bn = own ? a.beta[bt * a.bs[0] + (r0 + lane) * a.bs[1] + h * a.bs[2]] : 0.f;
  };
  const int group = a.Hv / a.Hk;
  fetch(hk * group);

  // K and Q rows as planes in LDS
  {
    constexpr int N = C * (KP / 8) / kThreads;   // pieces of eight of each, for a thread
    const T* kp = static_cast<const T*>(a.k) + bt * a.ks[0] + r0 * a.ks[1] + hk * a.ks[2];
    const T* qp = static_cast<const T*>(a.q) + bt * a.qs[0] + r0 * a.qs[1] + hk * a.qs[2];
    const int p = tid % (KP / 8), left = a.K - 8 * p;
    f32x8 v[2][N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = tid / (KP / 8) + i * (kThreads / (KP / 8));
      v[0][i] = v[1][i] = f32x8{};
      if (r < rows && left > 0) {
        v[0][i] = load8(kp + r * a.ks[1] + 8 * p, left, a.wide_k);
        v[1][i] = load8(qp + r * a.qs[1] + 8 * p, left, a.wide_q);
      }
    }
    if (tid < C) kbad[tid] = 0;
    lds_barrier();
    float odd[N], any = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = tid / (KP / 8) + i * (kThreads / (KP / 8));
      odd[i] = zero_if_finite(v[0][i].lo) + zero_if_finite(v[0][i].hi);
      any += odd[i];
      bf16x8 pl[NP];
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        planes8<NP>(v[w][i], pl);
#pragma unroll
        for (int j = 0; j < NP; ++j) *reinterpret_cast<bf16x8*>(kq + (w * NP + j) * kTile + tile_at<KP>(r, p)) = pl[j];
      }
    }
    if (__ballot(any != 0.f)) {   // rows of k that are not finite: marked, and zeros
      rare_path();
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (odd[i] != 0.f) kbad[tid / (KP / 8) + i * (kThreads / (KP / 8))] = 1;
    }
    lds_barrier();
    if (__ballot(kbad[lane % C])) {
      rare_path();
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int r = tid / (KP / 8) + i * (kThreads / (KP / 8));
        if (!kbad[r]) continue;
#pragma unroll
        for (int j = 0; j < NP; ++j) *reinterpret_cast<u32x4*>(kq + j * kTile + tile_at<KP>(r, p)) = u32x4{0, 0, 0, 0};
      }
      lds_barrier();
    }
  }
  // their fragments
  {
    char* dst = a.kq + (c * a.Hk + hk) * (int64_t)S::kKQ + lane * 16;
    for (int f = wave; f < S::fEnd; f += W) {
      bf16x8 v[NP];
      if (f < S::fKT) {
        const int e = f < S::fQ ? f : f - S::fQ;
        frag<KP, NP, kTile>(kq + (f < S::fQ ? 0 : NP * kTile), perm_row(e / S::KS, m), e % S::KS, g, v);
      } else {
        const int e = f < S::fQT ? f - S::fKT : f - S::fQT;
        frag_t<KP, NP, kTile>(kq + (f < S::fQT ? 0 : NP * kTile), e / S::CS, e % S::CS, g, m, v);
      }
#pragma unroll
      for (int j = 0; j < NP; ++j) *reinterpret_cast<bf16x8*>(dst + (f * NP + j) * 1024) = v[j];
    }
  }
  // k_i . k_j and q_i . k_j, rows 16 wave..+15, columns up to the diagonal tile
  f32x4 kk[S::RT], qk[S::RT];
#pragma unroll
  for (int j = 0; j < S::RT; ++j) kk[j] = qk[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < S::KS; ++s) {
    bf16x8 ka[NP], qa[NP];
    frag<KP, NP, kTile>(kq, 16 * wave + m, s, g, ka);
    frag<KP, NP, kTile>(kq + NP * kTile, 16 * wave + m, s, g, qa);
#pragma unroll
    for (int j = 0; j < S::RT; ++j) {
      if (j > wave) continue;
      bf16x8 kb[NP];
      frag<KP, NP, kTile>(kq, 16 * j + m, s, g, kb);
      kk[j] = mfma_planes<NP, NP, 3>(ka, kb, kk[j]);
      qk[j] = mfma_planes<NP, NP, 3>(qa, kb, qk[j]);
    }
  }
  mfma_settle();

  for (int e = 0; e < group; ++e) {
    const int h = hk * group + e;
    const int64_t ch = c * a.Hv + h;
    if (wave == 0) {
      float gv = gn, bv = bn;
      gv = gv < kMinG ? kMinG : gv;
      const uint64_t odd = __ballot((gv - gv) + (bv - bv) != 0.f || (lane < C && kbad[lane < C ? lane : 0]));
      const int bad = odd ? __ffsll((unsigned long long)odd) - 1 : C;
      if (lane >= bad) gv = bv = 0.f;
      double last;
      const double sum = running_sum(gv, lane, last);
      const float hi = (float)sum;
      if (lane < C) {
        ghi[lane] = hi;
        glo[lane] = (float)(sum - (double)hi);
        bet[lane] = bv;
      }
      float* vec = reinterpret_cast<float*>(a.vec + ch * (int64_t)kVec);
      vec[lane] = expf((float)sum);
      vec[64 + lane] = expf((float)(last - sum));
      vec[128 + lane] = bv;
      vec[192 + lane] = lane == 1 ? (float)bad : expf((float)last);
    }
    lds_barrier();   // and K, Q (first round) or the last head's tiles are done with
    if (e + 1 < group) fetch(h + 1);
    float pv[S::RT][4];
#pragma unroll
    for (int j = 0; j < S::RT; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 16 * wave + 4 * g + r, col = 16 * j + m;
        const bool lower = col <= row;
        const float d = lower ? expf((ghi[row] - ghi[col]) + (glo[row] - glo[col])) : 0.f;
        A[row * kLd + col] = col < row ? bet[row] * d * kk[j][r] : 0.f;
        X[row * kLd + col] = 0.f;
        pv[j][r] = lower ? a.scale * d * qk[j][r] : 0.f;
      }
    lds_barrier();
    // X = (I + A)^-1: the diagonal 16 x 16 blocks by substitution (a lane has one column), then joined in pairs
    if (wave == 0 && g < S::RT) {
      float x[16];
      const float* blk = A + (16 * g) * kLd + 16 * g;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float t = i == m ? 1.f : 0.f;
#pragma unroll
        for (int q = 0; q < (i + 3) / 4; ++q) {
          const f32x4 v = *reinterpret_cast<const f32x4*>(blk + i * kLd + 4 * q);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (4 * q + j < i) t = fmaf(-v[j], x[4 * q + j], t);
        }
        x[i] = t;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) X[(16 * g + i) * kLd + 16 * g + m] = x[i];
    }
    lds_barrier();
    if (wave < C / 32) {   // [X11 0; -X22 A21 X11  X22], 16 rows each
      const f32x4 y = mm16(A + (32 * wave + 16) * kLd + 32 * wave, kLd, X + 32 * wave * kLd + 32 * wave, kLd, 1, lane);
#pragma unroll
      for (int r = 0; r < 4; ++r) Y[(16 * wave + 4 * g + r) * kLdY + m] = y[r];
    }
    lds_barrier();
    if (wave < C / 32) {
      const f32x4 z = mm16(X + (32 * wave + 16) * kLd + 32 * wave + 16, kLd, Y + 16 * wave * kLdY, kLdY, 1, lane);
#pragma unroll
      for (int r = 0; r < 4; ++r) X[(32 * wave + 16 + 4 * g + r) * kLd + 32 * wave + m] = -z[r];
    }
    lds_barrier();
    if constexpr (C == 64) {   // the same of 32 rows each, a wave has one 16 x 16 tile
      const int ti = wave >> 1, tj = wave & 1;
      const f32x4 y = mm16(A + (32 + 16 * ti) * kLd, kLd, X + 16 * tj, kLd, 2, lane);
#pragma unroll
      for (int r = 0; r < 4; ++r) Y[(16 * ti + 4 * g + r) * kLdY + 16 * tj + m] = y[r];
      lds_barrier();
      const f32x4 z = mm16(X + (32 + 16 * ti) * kLd + 32, kLd, Y + 16 * tj, kLdY, 2, lane);
#pragma unroll
      for (int r = 0; r < 4; ++r) X[(32 + 16 * ti + 4 * g + r) * kLd + 16 * tj + m] = -z[r];
    }
    // P where A was (all of A has been read before the last barrier)
#pragma unroll
    for (int j = 0; j < S::RT; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) A[(16 * wave + 4 * g + r) * kLd + 16 * j + m] = pv[j][r];
    lds_barrier();
    char* dst = a.xp + ch * (int64_t)S::kXP + lane * 16;
    // a fragment's tile and inner step: rows (kind 0, 1: X, P) or columns (2, 3: X^T, P^T)
    auto cut = [&](auto np, auto transposed, const float* mat, int first, int f) {
      constexpr int N = decltype(np)::value;
      constexpr bool TR = decltype(transposed)::value;
      const int t = C == 32 ? f : TR ? (f >= 4 ? f - 2 : f >> 1) : (f < 2 ? f : 2 + ((f - 2) >> 1));
      const int s = C == 32 ? 0 : TR ? (f >= 4 ? 1 : f & 1) : (f < 2 ? 0 : (f - 2) & 1);
      bf16x8 v[N];
      tile_planes<N, TR>(mat, kLd, perm_row(t, m), 32 * s + 8 * g, v);
#pragma unroll
      for (int j = 0; j < N; ++j) *reinterpret_cast<bf16x8*>(dst + (first + f * N + j) * 1024) = v[j];
    };
    for (int f = wave; f < 2 * S::TRI; f += W) {
      if (f < S::TRI) cut(std::integral_constant<int, 3>(), std::false_type(), X, S::pX, f);
      else cut(std::integral_constant<int, S::NPP>(), std::false_type(), A, S::pP, f - S::TRI);
    }
    if constexpr (SAVE) {
      for (int f = wave; f < 2 * S::TRI; f += W) {
        if (f < S::TRI) cut(std::integral_constant<int, 3>(), std::true_type(), X, S::pXT, f);
        else cut(std::integral_constant<int, 3>(), std::true_type(), A, S::pPT, f - S::TRI);
      }
    }
    if (e + 1 < group) lds_barrier();   // before the next head's sums and tiles
  }
}

// --------------------------------------------------------------------------------------------- chunk after chunk

// A workgroup owns NC tiles of 16 columns, from the first chunk to the last.  C / 16 waves carry the state: each keeps TW tiles
// of S in registers and forms their share of K S for all rows; the shares are added up in LDS, where wave w takes rows
// perm_row(w, .) of R = beta (v - exp(G_i) K S) and of u.  R and u are handed on as planes in operand order: three barriers a
// chunk.  As many more waves form o (Q S and P u) beside them, a step behind.  The fragments of the next chunk are loaded as
// soon as those of this one are used.
//
// Bound by a chunk's chain of products and exchanges (few heads) or by loads and issue (many).  T 8192 of 128 x 128, bf16: one
// wave for all rows and products took 6.3 us a chunk, four waves 2.5 us, eight with all of S handed through LDS 2.0 us, with
// shares of K S instead 1.9 us (1.7 us, 222 us in all, at the clocks of a program that goes on).
template <int DT, int KP, int C, int NC, bool SAVE>
struct Scan {
  using S = DeltaShape<DT, KP, C, SAVE>;
  static constexpr int TW = S::KT >= 2 * S::RT ? S::KT / S::RT : 2, HW = S::KT / TW;   // HW waves have tiles of the state
  static constexpr int bS = 0, bK = S::KS * S::NO, bR = bK + HW * S::RT, bU = bR + S::CS * 3, bL = bU + S::CS * S::NO,
                       bEnd = bL + S::CS * 3;   // KB
  static constexpr int bad = NC * bEnd * 1024, bytes = bad + NC * 16 * S::RT * 4;
};

template <int DT, int KP, int C, int NC, bool SAVE>
__global__ __launch_bounds__(8 * C, 2) void k_delta_scan(DeltaArgs a) {
  using S = DeltaShape<DT, KP, C, SAVE>;
  using Sc = Scan<DT, KP, C, NC, SAVE>;
  using T = typename Elem<DT>::T;
  constexpr int NP = S::NP, NO = S::NO, TW = Sc::TW, HW = Sc::HW;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63, wave = wave_id(), w = wave % S::RT, x = lane & 15, g = lane >> 4;
  const int groups = (a.VP / 16 + NC - 1) / NC;
  int64_t n;
  int h, hk, group;
  if (!place_columns(a, groups, n, h, hk, group)) return;
  const int64_t head = n * a.Hv + h;
  const int col0 = group * NC * 16 + x;   // the lane's column in the first tile
  int64_t begin, len, c0;
  a.rows.range(n, begin, len, c0);
  begin = uniform(begin), len = uniform(len), c0 = uniform(c0);
  const int nc = (int)((len + C - 1) / C);
  const int row0 = perm_row(w, 4 * g);    // its rows of a chunk: row0..row0 + 3
  const float nan = __builtin_nanf("");
  const uint32_t at16 = lane * 16;

  const char* kq = a.kq + (c0 * a.Hk + hk) * (int64_t)S::kKQ;
  const char* xp = a.xp + (c0 * a.Hv + h) * (int64_t)S::kXP;
  const char* vec = a.vec + (c0 * a.Hv + h) * (int64_t)kVec;
  const int64_t kq_step = (int64_t)a.Hk * S::kKQ, xp_step = (int64_t)a.Hv * S::kXP, vec_step = (int64_t)a.Hv * kVec;
  bool in[NC];
#pragma unroll
  for (int i = 0; i < NC; ++i) in[i] = col0 + 16 * i < a.V;
  int* const bads = reinterpret_cast<int*>(lds + Sc::bad);
  auto part = [&](int i, int b) { return lds + (i * Sc::bEnd + b) * 1024; };
  // the first row of a lane's column that is not finite
  auto first_bad = [&](int i) {
    int b = C;
#pragma unroll
    for (int r = 0; r < S::RT; ++r) b = min(b, bads[(i * 16 + x) * S::RT + r]);
    return b;
  };

  if (wave < S::RT) {   // ---- the state
    const bool holds = w < HW;              // whether this wave has tiles of it
    f32x4 st[NC][TW];
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
      for (int t = 0; t < TW; ++t)
        st[i][t] = load_state(a.initial && holds ? a.initial + head * a.K * a.V : nullptr, a.K, a.V, col0 + 16 * i, w * TW + t, g);
    const T* vp[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i)
      vp[i] = static_cast<const T*>(a.v) + a.rows.batch(n) * a.vs[0] + begin * a.vs[1] + h * a.vs[2] + (in[i] ? col0 + 16 * i : a.V - 1);
    int64_t vrow[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) vrow[r] = (row0 + r) * a.vs[1];

    bf16x8 fk[S::RT][TW / 2][NP], fx[S::CS][3], ft[TW][S::CS][NP];
    struct { f32x4 into, left, beta; float all, bad; } f, fnext;   // of the wave's rows
    ColumnRows<T, C> v[NC];
    auto load_k = [&]() {
      if (!holds) return;
#pragma unroll
      for (int t = 0; t < S::RT; ++t)
#pragma unroll
        for (int s = 0; s < TW / 2; ++s) load_frag<NP>(kq, (S::fK + t * S::KS + w * (TW / 2) + s) * NP, at16, fk[t][s]);
    };
    auto load_x = [&]() {   // (rows of the upper half have no second inner step: theirs stays zero)
#pragma unroll
      for (int s = 0; s < S::CS; ++s)
        if (s <= w / 2) load_frag<3>(xp, S::pX + 3 * tri_frag(w, s), at16, fx[s]);
    };
#pragma unroll
    for (int s = 0; s < S::CS; ++s)
#pragma unroll
      for (int i = 0; i < 3; ++i) fx[s][i] = bf16x8{};
    auto load_t = [&]() {
      if (!holds) return;
#pragma unroll
      for (int t = 0; t < TW; ++t)
#pragma unroll
        for (int s = 0; s < S::CS; ++s) load_frag<NP>(kq, (S::fKT + (w * TW + t) * S::CS + s) * NP, at16, ft[t][s]);
    };
    auto load_v = [&](int ci) {
      const int64_t left_rows = len - (int64_t)ci * C;
#pragma unroll
      for (int i = 0; i < NC; ++i) v[i].load(vp[i] + (int64_t)ci * C * a.vs[1], vrow, a.vs[1], (int)(left_rows < C ? left_rows : C), row0);
    };
    auto load_vec = [&]() {
      const float* p = reinterpret_cast<const float*>(vec);
      fnext.into = *reinterpret_cast<const f32x4*>(p + row0);
      fnext.left = *reinterpret_cast<const f32x4*>(p + 64 + row0);
      fnext.beta = *reinterpret_cast<const f32x4*>(p + 128 + row0);
      fnext.all = p[192];
      fnext.bad = p[193];
    };
    // S as planes for Q S, and this wave's share of K S (where it has tiles of S)
    auto put_state = [&]() {
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        f32x4 ks[S::RT];
#pragma unroll
        for (int t = 0; t < S::RT; ++t) ks[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < TW / 2; ++s) {
          bf16x8 sp[3];
          planes8<3>(cat8(st[i][2 * s], st[i][2 * s + 1]), sp);
          mfma_rows<NP, 3, 3, S::RT>([&](int t) -> const bf16x8(&)[NP] { return fk[t][s]; }, sp, ks);
#pragma unroll
          for (int j = 0; j < NO; ++j)
            *reinterpret_cast<bf16x8*>(part(i, Sc::bS) + ((w * (TW / 2) + s) * NO + j) * 1024 + at16) = sp[j];
        }
#pragma unroll
        for (int t = 0; t < S::RT; ++t) *reinterpret_cast<f32x4*>(part(i, Sc::bK) + (t * HW + w) * 1024 + at16) = ks[t];
      }
    };
    if (nc > 0) {
      load_k();
      load_v(0);
      load_vec();
      load_x();
      load_t();
      if (holds) put_state();
    }
    for (int ci = 0; ci < nc; ++ci) {
      const bool more = ci + 1 < nc;   // behind the last chunk its own values are loaded again, and not used
      const int64_t ch = (c0 + ci) * a.Hv + h;
      lds_barrier();
      f32x4 ks[NC];
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        ks[i] = *reinterpret_cast<const f32x4*>(part(i, Sc::bK) + w * HW * 1024 + at16);
#pragma unroll
        for (int j = 1; j < HW; ++j) ks[i] += *reinterpret_cast<const f32x4*>(part(i, Sc::bK) + (w * HW + j) * 1024 + at16);
      }
      f = fnext;
      if (more) vec += vec_step;
      load_vec();
      // beta (v - exp(G_i) K S)
      int bad[NC];
      float odd = 0.f;
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        ks[i] = f.beta * (v[i].get(in[i], row0) - f.into * ks[i]);
        odd += zero_if_finite(ks[i]);
        bad[i] = (int)f.bad;
      }
      if (__ballot(odd != 0.f)) {
        rare_path();
#pragma unroll
        for (int i = 0; i < NC; ++i) {
#pragma unroll
          for (int r = 3; r >= 0; --r)
            if (ks[i][r] * 0.f != 0.f) {   // (not a - a, which may contract to the rounding error of a product)
              ks[i][r] = 0.f;
              bad[i] = row0 + r < bad[i] ? row0 + r : bad[i];
            }
          bad[i] = min(bad[i], __shfl_xor(bad[i], 16));
          bad[i] = min(bad[i], __shfl_xor(bad[i], 32));
        }
      }
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        put_half<3>(part(i, Sc::bR), w / 2, w & 1, lane, ks[i]);
        if (g == 0) bads[(i * 16 + x) * S::RT + w] = bad[i];
      }
      if (more) kq += kq_step;
      load_k();
      load_v(more ? ci + 1 : ci);
      if (SAVE && holds) {
        float* s0 = a.s0 + ch * (int64_t)KP * a.VP + col0;
#pragma unroll
        for (int i = 0; i < NC; ++i)
#pragma unroll
          for (int t = 0; t < TW; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (col0 + 16 * i < a.VP) s0[perm_row(w * TW + t, 4 * g + r) * a.VP + 16 * i] = st[i][t][r];
      }
      lds_barrier();
      // u = X of it
      f32x4 u[NC];
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        u[i] = product<3, 3, 3, S::CS>(fx, [&](int s, bf16x8(&b)[3]) { get_operand<3>(part(i, Sc::bR), s, lane, b); });
        put_half<3>(part(i, Sc::bL), w / 2, w & 1, lane, f.left * u[i]);
        put_half<NO>(part(i, Sc::bU), w / 2, w & 1, lane, u[i]);
        bad[i] = first_bad(i);
      }
      if (more) xp += xp_step;
      load_x();
      lds_barrier();
      // S <- exp(G) S + K^T (exp(G - G_i) u)
      if (holds) {
#pragma unroll
        for (int i = 0; i < NC; ++i) {
#pragma unroll
          for (int t = 0; t < TW; ++t) st[i][t] *= bad[i] < C ? nan : f.all;   // a column that is no longer finite
#pragma unroll
          for (int s = 0; s < S::CS; ++s) {
            bf16x8 up[3];
            get_operand<3>(part(i, Sc::bL), s, lane, up);
#pragma unroll
            for (int t = 0; t < TW; ++t) st[i][t] = mfma_planes<NP, 3, 3>(ft[t][s], up, st[i][t]);
          }
        }
        put_state();   // behind no branch: it reads the products' results first
      }
      load_t();
      if (SAVE) {
        float* us = a.u + (ch * C + row0) * (int64_t)a.VP + col0;
#pragma unroll
        for (int i = 0; i < NC; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (col0 + 16 * i < a.VP) us[r * a.VP + 16 * i] = row0 + r >= bad[i] ? nan : u[i][r];
      }
    }
    if (holds) {
#pragma unroll
      for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int t = 0; t < TW; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int kd = perm_row(w * TW + t, 4 * g + r);
            if (in[i] && kd < a.K) a.final[(head * a.K + kd) * a.V + col0 + 16 * i] = st[i][t][r];
          }
    }
  } else {   // ---- o
    T* op[NC];
    const int64_t orow = (int64_t)a.Hv * a.V;
#pragma unroll
    for (int i = 0; i < NC; ++i)
      op[i] = static_cast<T*>(a.o) + ((a.rows.batch(n) * a.rows.T + begin) * a.Hv + h) * (int64_t)a.V + col0 + 16 * i + row0 * orow;
    bf16x8 fq[S::KS][NP], fp[S::CS][NO];
    f32x4 into;
    auto load_q = [&]() {
#pragma unroll
      for (int s = 0; s < S::KS; ++s) load_frag<NP>(kq, (S::fQ + w * S::KS + s) * NP, at16, fq[s]);
      into = *reinterpret_cast<const f32x4*>(vec + row0 * 4);
    };
    auto load_p = [&]() {
#pragma unroll
      for (int s = 0; s < S::CS; ++s)
        if (s <= w / 2) load_frag<NO>(xp, S::pP + S::NPP * tri_frag(w, s), at16, fp[s]);
    };
#pragma unroll
    for (int s = 0; s < S::CS; ++s)
#pragma unroll
      for (int i = 0; i < NO; ++i) fp[s][i] = bf16x8{};
    f32x4 o[NC];
    int bad[NC];
    // o of chunk ci, of which only P u is missing
    auto finish = [&](int ci) {
      const int rows = (int)(len - (int64_t)ci * C < C ? len - (int64_t)ci * C : C);
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        o[i] += product<NO, NO, NO, S::CS>(fp, [&](int s, bf16x8(&b)[NO]) { get_operand<NO>(part(i, Sc::bU), s, lane, b); });
#pragma unroll
        for (int r = 0; r < 4; ++r) o[i][r] = row0 + r >= bad[i] ? nan : o[i][r];
        if (rows == C) {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (in[i]) op[i][r * orow] = (T)o[i][r];
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (in[i] && row0 + r < rows) op[i][r * orow] = (T)o[i][r];
        }
        op[i] += C * orow;
      }
    };
    if (nc > 0) load_q();
    for (int ci = 0; ci < nc; ++ci) {
      lds_barrier();
      if (ci > 0) finish(ci - 1);
      load_p();
      lds_barrier();
#pragma unroll
      for (int i = 0; i < NC; ++i)
        o[i] = product<NP, NO, NO, S::KS>(fq, [&](int s, bf16x8(&b)[NO]) { get_operand<NO>(part(i, Sc::bS), s, lane, b); });
#pragma unroll
      for (int i = 0; i < NC; ++i) o[i] *= a.scale * into;
      if (ci + 1 < nc) kq += kq_step, vec += vec_step, xp += xp_step;
      load_q();
      lds_barrier();
#pragma unroll
      for (int i = 0; i < NC; ++i) bad[i] = first_bad(i);
    }
    if (nc > 0) finish(nc - 1);
  }
}

// zeros in the rows of packed sequences that belong to none, before the first and behind the last, of up to five tensors
__global__ void k_delta_outside(DeltaRows rows, DeltaOutside t) {
  const int64_t first = rows.at(0), end = rows.at(rows.N), last = end > first ? end : first;
  const int64_t row = t.row[blockIdx.y], n = (first + rows.T - last) * row;   // row: bytes, even
  char* q = static_cast<char*>(t.p[blockIdx.y]);
  for (int64_t b = 2 * (blockIdx.x * (int64_t)blockDim.x + threadIdx.x); b < n; b += 2 * (int64_t)gridDim.x * blockDim.x)
    *reinterpret_cast<uint16_t*>(q + (b < first * row ? b : b + (last - first) * row)) = 0;
}

template <int DT, int KP, int C, int NC, bool SAVE>
hipError_t scan(const DeltaArgs& a, hipStream_t s) {
  using Sc = Scan<DT, KP, C, NC, SAVE>;
  const hipError_t e = allow_lds(k_delta_scan<DT, KP, C, NC, SAVE>, Sc::bytes);
  if (e != hipSuccess) return e;
  const int groups = (a.VP / 16 + NC - 1) / NC;
  k_delta_scan<DT, KP, C, NC, SAVE><<<column_blocks(a, groups), 8 * C, Sc::bytes, s>>>(a);
  return hipGetLastError();
}

template <int DT, int KP, int C, bool SAVE>
hipError_t forward(const DeltaArgs& a, hipStream_t s) {
  constexpr int bytes = PrepLds<DT, KP, C, SAVE>::bytes;
  const hipError_t e = allow_lds(k_delta_prep<DT, KP, C, SAVE>, bytes);
  if (e != hipSuccess) return e;
  if (a.chunks) k_delta_prep<DT, KP, C, SAVE><<<(unsigned)(a.chunks * a.Hk), 4 * C, bytes, s>>>(a);
  return a.wide_cols ? scan<DT, KP, C, 2, SAVE>(a, s) : scan<DT, KP, C, 1, SAVE>(a, s);
}

template <int DT, int KP>
hipError_t forward(const DeltaArgs& a, bool save, hipStream_t s) {
  if (a.rows.C == 32) return save ? forward<DT, KP, 32, true>(a, s) : forward<DT, KP, 32, false>(a, s);
  return save ? forward<DT, KP, 64, true>(a, s) : forward<DT, KP, 64, false>(a, s);
}

template <int DT>
hipError_t forward(const DeltaArgs& a, int KP, bool save, hipStream_t s) {
  return KP == 32 ? forward<DT, 32>(a, save, s) : KP == 64 ? forward<DT, 64>(a, save, s) : forward<DT, 128>(a, save, s);
}

}  // namespace

hipError_t delta_outside(const DeltaRows& rows, const DeltaOutside& t, hipStream_t s) {
  k_delta_outside<<<dim3(64, t.n), 256, 0, s>>>(rows, t);
  return hipGetLastError();
}

hipError_t delta_forward(const DeltaArgs& a, int dtype, int KP, bool save, hipStream_t s) {
  return dtype == SEQ_BF16 ? forward<SEQ_BF16>(a, KP, save, s)
         : dtype == SEQ_FP16 ? forward<SEQ_FP16>(a, KP, save, s) : forward<SEQ_FP32>(a, KP, save, s);
}

}  // namespace seq
