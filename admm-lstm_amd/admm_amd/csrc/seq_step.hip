// seq_step.hip -- one token of the gated delta rule per stream (serving), the state updated in place.
//
// Bound by the state: K V values of 32 bits read and written per stream and head, everything else is a few rows.  A
// workgroup takes COLS columns of one head's state, all rows of it in registers (a lane: 4 columns of some rows), so
// that one load and one store of the state are all the traffic, and S^T k and S^T q come out of one reduction: with
// S' = exp(g) S and u = beta (v - S'^T k), S = S' + k u^T and S^T q = S'^T q + (k . q) u.
#include "seq_delta.hpp"

namespace seq {
namespace {

// STREAM: the states are too many for the caches to hold them until the next token
template <int DT, int COLS, int R, bool STREAM>
__global__ __launch_bounds__(256) void k_delta_step(SeqDeltaStep d, bool wide) {
  using T = typename Elem<DT>::T;
  constexpr int L = COLS / 4, kRows = 256 / L;   // lanes side by side, rows at a time
  __shared__ float part[4][L][9];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c4 = tid % L, kr = tid / L;
  const int tiles = (d.V + COLS - 1) / COLS;
  const int64_t bh = blockIdx.x / tiles;
  const int64_t b = bh / d.Hv;
  const int h = (int)(bh % d.Hv), hk = h / (d.Hv / d.Hk);
  const int col = (int)(blockIdx.x % tiles) * COLS + 4 * c4;
  const int nc = d.V - col < 4 ? d.V - col : 4;   // columns of this lane inside the row (may be negative)
  auto slot_of = [&](int64_t i) {
    return d.slots_64 ? static_cast<const int64_t*>(d.slots)[i] : (int64_t) static_cast<const int32_t*>(d.slots)[i];
  };
  const int64_t slot = d.slots ? slot_of(b) : b;
  const bool idle = slot < 0;
  bool bad = slot >= d.pool;
  float* S = d.state + (idle || bad ? 0 : slot) * d.state_stride[0] + h * d.state_stride[1] + col;

  f32x4 st[R];
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int kd = kr + kRows * j;
    st[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (kd < d.K && !idle && !bad) {
      const float* p = S + (int64_t)kd * d.V;
      if (wide && nc == 4) {
        const f32x4* q = reinterpret_cast<const f32x4*>(p);
        st[j] = STREAM ? __builtin_nontemporal_load(q) : *q;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i < nc) st[j][i] = p[i];
      }
    }
  }
  if (d.slots) {   // the same slot in an earlier row: that row has it
    bool dup = false;
    if (!idle && !bad)
      for (int64_t i = tid; i < b; i += 256) dup |= slot_of(i) == slot;
    bad |= __syncthreads_or(dup) != 0;
  }
  const float a = expf(d.g[b * d.g_stride[0] + h * d.g_stride[1]]);
  const float beta = d.beta[b * d.beta_stride[0] + h * d.beta_stride[1]];
  const T* kp = static_cast<const T*>(d.k) + b * d.k_stride[0] + hk * d.k_stride[1];
  const T* qp = static_cast<const T*>(d.q) + b * d.q_stride[0] + hk * d.q_stride[1];
  const T* vp = static_cast<const T*>(d.v) + b * d.v_stride[0] + h * d.v_stride[1] + col;
  float k[R], sums[9] = {};
  float v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = i < nc ? (float)vp[i] : 0.f;
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int kd = kr + kRows * j;
    const bool in = kd < d.K;
    k[j] = in ? (float)kp[kd] : 0.f;
    const float q = in ? (float)qp[kd] : 0.f;
    st[j] *= a;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sums[i] = fmaf(st[j][i], k[j], sums[i]);
      sums[4 + i] = fmaf(st[j][i], q, sums[4 + i]);
    }
    sums[8] = fmaf(k[j], q, sums[8]);
  }
#pragma unroll
  for (int i = 0; i < 9; ++i) {
#pragma unroll
    for (int x = L; x < 64; x *= 2) sums[i] += __shfl_xor(sums[i], x);
  }
  if (lane < L) {
#pragma unroll
    for (int i = 0; i < 9; ++i) part[wave][c4][i] = sums[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 9; ++i) sums[i] = (part[0][c4][i] + part[1][c4][i]) + (part[2][c4][i] + part[3][c4][i]);
  f32x4 u;
#pragma unroll
  for (int i = 0; i < 4; ++i) u[i] = beta * (v[i] - sums[i]);
  if (tid < L) {
    T* o = static_cast<T*>(d.o) + (b * d.Hv + h) * (int64_t)d.V + col;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float y = d.scale * fmaf(sums[8], u[i], sums[4 + i]);
      if (i < nc) o[i] = (T)(idle ? 0.f : bad ? __builtin_nanf("") : y);
    }
  }
  if (idle || bad) return;
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int kd = kr + kRows * j;
    if (kd >= d.K) continue;
    float* p = S + (int64_t)kd * d.V;
    const f32x4 n = st[j] + k[j] * u;
    if (wide && nc == 4) {
      if (STREAM) __builtin_nontemporal_store(n, reinterpret_cast<f32x4*>(p));
      else *reinterpret_cast<f32x4*>(p) = n;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < nc) p[i] = n[i];
    }
  }
}

template <int DT, int COLS, bool STREAM>
void launch(const SeqDeltaStep& d, hipStream_t s) {
  constexpr int kRows = 1024 / COLS;
  const unsigned grid = (unsigned)(d.batch * d.Hv * ((d.V + COLS - 1) / COLS));
  const bool wide = d.V % 4 == 0 && d.state_stride[0] % 4 == 0 && d.state_stride[1] % 4 == 0 &&
                    reinterpret_cast<uintptr_t>(d.state) % 16 == 0;
  if (d.K <= 32) k_delta_step<DT, COLS, 32 / kRows, STREAM><<<grid, 256, 0, s>>>(d, wide);
  else if (d.K <= 64) k_delta_step<DT, COLS, 64 / kRows, STREAM><<<grid, 256, 0, s>>>(d, wide);
  else k_delta_step<DT, COLS, 128 / kRows, STREAM><<<grid, 256, 0, s>>>(d, wide);
}

// 32 columns: the most workgroups (one stream of 32 heads of 128 x 128: 128 of them, 6.6 us; with 128 columns 32).  128
// columns, whole rows of 512 bytes, where every compute unit has several of those, and past the caches where the states are
// more than half of the 256 MB that stay on the chip: 192 such streams, 402 MB of states read and written, take 227 us
// with 32 columns, 181 us with 128, 158 us (5.1 TB/s, what a copy reaches) past the caches.
template <int DT>
void launch(const SeqDeltaStep& d, hipStream_t s) {
  const int64_t heads = d.batch * d.Hv;
  if (step_cols(heads, d.V) == 32) launch<DT, 32, false>(d, s);
  else if (heads * d.K * d.V <= (32 << 20)) launch<DT, 128, false>(d, s);
  else launch<DT, 128, true>(d, s);
}

}  // namespace

hipError_t delta_step(const SeqDeltaStep& d, hipStream_t s) {
  if (d.dtype == SEQ_BF16) launch<SEQ_BF16>(d, s);
  else if (d.dtype == SEQ_FP16) launch<SEQ_FP16>(d, s);
  else launch<SEQ_FP32>(d, s);
  return hipGetLastError();
}

}  // namespace seq
