// seq_host.hip -- the C ABI of libseqops.so (include/seq_ops.h): checks, work-memory layout, dispatch.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>

#include "seq_delta.hpp"

namespace seq {
hipError_t delta_forward(const DeltaArgs& a, int dtype, int KP, bool save, hipStream_t s);
hipError_t delta_backward(const DeltaGradArgs& ga, int dtype, int KP, bool wide_v, bool wide_o, hipStream_t s);
hipError_t delta_outside(const DeltaRows& rows, void* p, int64_t row_bytes, hipStream_t s);
hipError_t delta_step(const SeqDeltaStep& d, hipStream_t s);
}  // namespace seq

using namespace seq;

namespace {

thread_local char g_error[512];   // a plain array: nothing here can throw across the C boundary

int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_error, sizeof g_error, fmt, ap);
  va_end(ap);
  return code;
}

int hip_result(hipError_t e, const char* what) {
  return e == hipSuccess ? SEQ_OK : fail(SEQ_EHIP, "%s: %s", what, hipGetErrorString(e));
}

// the tensors' device for the length of a call; the caller's device afterwards
struct OnDevice {
  int prev = -1;
  hipError_t err = hipSuccess;
  explicit OnDevice(int dev) {
    if (hipGetDevice(&prev) != hipSuccess) prev = -1;
    if (prev != dev) err = hipSetDevice(dev);
  }
  ~OnDevice() {
    int cur = -1;
    if (prev >= 0 && hipGetDevice(&cur) == hipSuccess && cur != prev) (void)hipSetDevice(prev);
  }
};

#define ON_DEVICE(dev)  \
  OnDevice on_(dev);    \
  if (on_.err != hipSuccess) return fail(SEQ_EHIP, "hipSetDevice(%d): %s", (int)(dev), hipGetErrorString(on_.err))

int elem_size(int dtype) { return dtype == SEQ_FP32 ? 4 : 2; }
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

constexpr int64_t kMaxBlocks = 0x7fffffff;

// ----------------------------------------------------------------------------------------------- gated delta rule

int check_heads(int Hk, int Hv, int K, int V, int dtype) {
  if (dtype < SEQ_BF16 || dtype > SEQ_FP32) return fail(SEQ_EINVAL, "unknown dtype %d", dtype);
  if (Hk < 1 || Hv < 1 || Hv % Hk) return fail(SEQ_EINVAL, "value heads (%d) must be a multiple of query/key heads (%d)", Hv, Hk);
  if (K < 1 || K > SEQ_DELTA_MAX_K) return fail(SEQ_EINVAL, "query/key rows of %d values: 1 to %d are supported", K, SEQ_DELTA_MAX_K);
  if (V < 1 || V > SEQ_DELTA_MAX_V) return fail(SEQ_EINVAL, "value rows of %d values: 1 to %d are supported", V, SEQ_DELTA_MAX_V);
  return SEQ_OK;
}

struct DeltaSizes {
  int KP, NP, NO;
  int64_t per, chunks, VP, kq, xp, vec, s0, u, heads, need;
};

int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }

int delta_sizes(const SeqDelta* d, bool saved, DeltaSizes& z) {
  if (!d) return fail(SEQ_EINVAL, "NULL argument");
  const int rc = check_heads(d->Hk, d->Hv, d->K, d->V, d->dtype);
  if (rc) return rc;
  if (d->batch < 0 || d->T < 0 || d->sequences < 0) return fail(SEQ_EINVAL, "negative size");
  if (d->offsets ? d->batch != 1 : d->sequences != d->batch)
    return fail(SEQ_EINVAL, d->offsets ? "packed sequences need batch 1 (got %lld)" : "sequences must equal batch (%lld)", (long long)d->batch);
  z.KP = d->K <= 32 ? 32 : d->K <= 64 ? 64 : 128;
  z.NP = d->dtype + 1;
  z.NO = d->dtype == SEQ_FP32 ? 3 : 2;
  z.per = (d->T + kC - 1) / kC;
  z.VP = (d->V + 15) / 16 * 16;
  z.chunks = d->offsets ? (d->sequences && d->T ? d->T / kC + d->sequences + 1 : 0) : z.per * d->batch;
  const int64_t blocks = (z.VP / 16 + 3) / 4;
  if (z.chunks > kMaxBlocks / d->Hv || (d->sequences + 8) > kMaxBlocks / (d->Hv * blocks))
    return fail(SEQ_EINVAL, "too many sequences, rows or heads for one launch");
  z.kq = up256(z.chunks * d->Hk * (4LL * z.NP * kC * z.KP));
  z.xp = up256(z.chunks * d->Hv * (2LL * (3 + (saved ? 3 : z.NO)) * kTri));
  z.vec = up256(z.chunks * d->Hv * (4LL * kC * 4));
  z.s0 = up256(z.chunks * d->Hv * 4 * z.KP * z.VP);
  z.u = up256(z.chunks * d->Hv * 4 * kC * z.VP);
  const int64_t rows = d->batch * d->T;
  z.heads = d->Hv > d->Hk ? up256(rows * d->Hv * d->K * 4) : 0;
  z.need = z.kq + z.xp + z.vec + (saved ? z.s0 + z.u : 0);
  return SEQ_OK;
}

int check_memory(const char* name, const void* p, int64_t bytes, int64_t need) {
  if (bytes < need) return fail(SEQ_EINVAL, "%s memory of %lld bytes: %lld are needed", name, (long long)bytes, (long long)need);
  if (need && (!p || !aligned16(p))) return fail(SEQ_EINVAL, "%s memory is NULL or not 16-byte aligned", name);
  return SEQ_OK;
}

// whether 16 bytes at a time may be read from rows of n values
template <class S>
bool wide_rows(const SeqDelta* d, int len, const void* p, const S& stride) {
  const int n = 16 / elem_size(d->dtype);
  return aligned16(p) && len % 8 == 0 && stride[0] % n == 0 && stride[1] % n == 0 && stride[2] % n == 0;
}

void delta_args(const SeqDelta* d, const DeltaSizes& z, void* work, DeltaArgs& a) {
  memset(&a, 0, sizeof a);
  a.rows.T = d->T;
  a.rows.N = d->sequences;
  a.rows.per = z.per;
  a.rows.off = d->offsets;
  a.rows.off64 = d->offsets_64;
  a.Hk = d->Hk, a.Hv = d->Hv, a.K = d->K, a.V = d->V, a.VP = (int)z.VP;
  a.scale = d->scale;
  a.q = d->q, a.k = d->k, a.v = d->v, a.g = d->g, a.beta = d->beta;
  memcpy(a.qs, d->q_stride, sizeof a.qs);
  memcpy(a.ks, d->k_stride, sizeof a.ks);
  memcpy(a.vs, d->v_stride, sizeof a.vs);
  memcpy(a.gs, d->g_stride, sizeof a.gs);
  memcpy(a.bs, d->beta_stride, sizeof a.bs);
  a.wide_q = wide_rows(d, d->K, d->q, d->q_stride);
  a.wide_k = wide_rows(d, d->K, d->k, d->k_stride);
  a.initial = d->initial;
  a.chunks = z.chunks;
  char* w = static_cast<char*>(work);
  a.kq = w;
  a.xp = w + z.kq;
  a.vec = a.xp + z.xp;
  a.s0 = reinterpret_cast<float*>(a.vec + z.vec);
  a.u = reinterpret_cast<float*>(a.vec + z.vec + z.s0);
}

bool delta_inputs(const SeqDelta* d) { return d->batch * d->T == 0 || (d->q && d->k && d->v && d->g && d->beta); }

}  // namespace

extern "C" {

int32_t seq_abi_version(void) { return SEQ_OPS_ABI_VERSION; }
const char* seq_last_error(void) { return g_error; }

int seq_delta_workspace(const SeqDelta* d, int32_t saved, int64_t* bytes) {
  DeltaSizes z;
  const int rc = delta_sizes(d, saved != 0, z);
  if (rc) return rc;
  if (!bytes) return fail(SEQ_EINVAL, "NULL argument");
  *bytes = z.need;
  return SEQ_OK;
}

int seq_delta_forward(const SeqDelta* d, int32_t saved, void* work, int64_t work_bytes, void* o, float* final_state,
                      void* stream) {
  DeltaSizes z;
  int rc = delta_sizes(d, saved != 0, z);
  if (!rc) rc = check_memory("work", work, work_bytes, z.need);
  if (rc) return rc;
  if (!delta_inputs(d) || (d->batch * d->T && !o) || (d->sequences && !final_state)) return fail(SEQ_EINVAL, "NULL buffer");
  ON_DEVICE(d->device);
  DeltaArgs a;
  delta_args(d, z, work, a);
  a.o = o;
  a.final = final_state;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (d->offsets && d->T) {
    const int e = hip_result(delta_outside(a.rows, o, (int64_t)d->Hv * d->V * elem_size(d->dtype), s), "delta_rule");
    if (e) return e;
  }
  if (!d->sequences) return SEQ_OK;
  return hip_result(delta_forward(a, d->dtype, z.KP, saved != 0, s), "delta_rule");
}

int seq_delta_backward_scratch(const SeqDelta* d, int64_t* bytes) {
  DeltaSizes z;
  const int rc = delta_sizes(d, true, z);
  if (rc) return rc;
  if (!bytes) return fail(SEQ_EINVAL, "NULL argument");
  *bytes = z.s0 + z.u + 2 * z.heads;
  return SEQ_OK;
}

int seq_delta_backward(const SeqDelta* d, const void* work, int64_t work_bytes, void* scratch, int64_t scratch_bytes,
                       const void* d_o, const float* d_final, void* dq, void* dk, void* dv, float* dg, float* dbeta,
                       float* d_initial, void* stream) {
  DeltaSizes z;
  int rc = delta_sizes(d, true, z);
  if (!rc) rc = check_memory("work", work, work_bytes, z.need);
  if (!rc) rc = check_memory("scratch", scratch, scratch_bytes, z.s0 + z.u + 2 * z.heads);
  if (rc) return rc;
  const bool some = d->batch * d->T != 0;
  if (!delta_inputs(d) || (some && (!d_o || !dq || !dk || !dv || !dg || !dbeta))) return fail(SEQ_EINVAL, "NULL buffer");
  ON_DEVICE(d->device);
  hipStream_t s = static_cast<hipStream_t>(stream);
  DeltaGradArgs ga;
  memset(&ga, 0, sizeof ga);
  delta_args(d, z, const_cast<void*>(work), ga.f);   // read only
  char* p = static_cast<char*>(scratch);
  ga.ds = reinterpret_cast<float*>(p);
  ga.dr = reinterpret_cast<float*>(p + z.s0);
  if (z.heads) {
    ga.dq32 = reinterpret_cast<float*>(p + z.s0 + z.u);
    ga.dk32 = reinterpret_cast<float*>(p + z.s0 + z.u + z.heads);
  }
  ga.d_o = d_o, ga.d_final = d_final;
  ga.dq = dq, ga.dk = dk, ga.dv = dv, ga.dg = dg, ga.dbeta = dbeta, ga.d_initial = d_initial;
  if (d->sequences) {
    const bool wide_o = aligned16(d_o) && d->V % 8 == 0;
    rc = hip_result(delta_backward(ga, d->dtype, z.KP, wide_rows(d, d->V, d->v, d->v_stride), wide_o, s), "delta_rule backward");
  }
  if (rc || !d->offsets || !some) return rc;
  const int64_t size = elem_size(d->dtype), kb = (int64_t)d->Hk * d->K * size, vb = (int64_t)d->Hv * d->V * size, hb = (int64_t)d->Hv * 4;
  void* const out[5] = {dq, dk, dv, dg, dbeta};
  const int64_t row[5] = {kb, kb, vb, hb, hb};
  for (int i = 0; i < 5 && !rc; ++i) rc = hip_result(delta_outside(ga.f.rows, out[i], row[i], s), "delta_rule backward");
  return rc;
}

int seq_delta_step(const SeqDeltaStep* d, void* stream) {
  if (!d) return fail(SEQ_EINVAL, "NULL argument");
  const int rc = check_heads(d->Hk, d->Hv, d->K, d->V, d->dtype);
  if (rc) return rc;
  if (d->batch < 0 || d->pool < 0) return fail(SEQ_EINVAL, "negative size");
  if (!d->slots && d->batch > d->pool) return fail(SEQ_EINVAL, "%lld rows and %lld states", (long long)d->batch, (long long)d->pool);
  if (d->batch > kMaxBlocks / d->Hv / ((d->V + 31) / 32)) return fail(SEQ_EINVAL, "too many rows for one launch");
  if (!d->batch) return SEQ_OK;
  if (!d->q || !d->k || !d->v || !d->g || !d->beta || !d->o || (d->pool && !d->state)) return fail(SEQ_EINVAL, "NULL buffer");
  ON_DEVICE(d->device);
  return hip_result(delta_step(*d, static_cast<hipStream_t>(stream)), "delta_step");
}

}  // extern "C"
