// seq_host.hip -- the C ABI of libseqops.so (include/seq_ops.h): checks, work-memory layout, dispatch.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>

#include "seq_delta.hpp"
#include "seq_unit.hpp"

namespace seq {
hipError_t delta_forward(const DeltaArgs& a, int dtype, int KP, bool save, hipStream_t s);
hipError_t delta_backward(const DeltaGradArgs& ga, int dtype, int KP, bool wide_v, bool wide_o, hipStream_t s);
hipError_t delta_heads(const DeltaGradArgs& ga, int dtype, hipStream_t s);
hipError_t delta_short_forward(const DeltaArgs& a, int dtype, int KP, hipStream_t s);
hipError_t delta_short_backward(const DeltaGradArgs& ga, int dtype, int KP, bool wide_s, hipStream_t s);
hipError_t delta_outside(const DeltaRows& rows, const DeltaOutside& t, hipStream_t s);
hipError_t delta_step(const SeqDeltaStep& d, hipStream_t s);
hipError_t dropout(int dtype, const void* x, const void* res, void* y, int64_t n, uint32_t below, uint64_t seed, uint64_t offset,
                   const int64_t* seed_dev, hipStream_t s);
hipError_t unit_forward_bf16(const UnitArgs& u, hipStream_t s);
hipError_t unit_forward_fp16(const UnitArgs& u, hipStream_t s);
hipError_t unit_forward_fp32(const UnitArgs& u, hipStream_t s);
hipError_t unit_backward_bf16(const UnitArgs& u, hipStream_t s);
hipError_t unit_backward_fp16(const UnitArgs& u, hipStream_t s);
hipError_t unit_backward_fp32(const UnitArgs& u, hipStream_t s);
int unit_few_splits(int M, int D, int F, int dtype);
hipError_t unit_few(const UnitArgs& u, int splits, float* sums, hipStream_t s);
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

constexpr int64_t kMaxThreads = 0xffffffff;   // of a launch, along an axis

// ----------------------------------------------------------------------------------------------- gated delta rule

int check_heads(int Hk, int Hv, int K, int V, int dtype) {
  if (dtype < SEQ_BF16 || dtype > SEQ_FP32) return fail(SEQ_EINVAL, "unknown dtype %d", dtype);
  if (Hk < 1 || Hv < 1 || Hv % Hk) return fail(SEQ_EINVAL, "value heads (%d) must be a multiple of query/key heads (%d)", Hv, Hk);
  if (K < 1 || K > SEQ_DELTA_MAX_K) return fail(SEQ_EINVAL, "query/key rows of %d values: 1 to %d are supported", K, SEQ_DELTA_MAX_K);
  if (V < 1 || V > SEQ_DELTA_MAX_V) return fail(SEQ_EINVAL, "value rows of %d values: 1 to %d are supported", V, SEQ_DELTA_MAX_V);
  return SEQ_OK;
}

struct DeltaSizes {
  int KP, C;
  bool brief, wide_cols;   // brief: one kernel for a whole sequence (at most 32 rows, not packed), without work memory
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
  // Chunks of 32 rows where sequences are so short that half of 64 would be empty, and where there are more column tiles than two
  // rounds of the chip's: less is done then in each chunk (X is formed in C^3, P u in C^2 a row), while with few tiles the number of
  // chunks counts.  With gradients these take more for the chunks' states than that saves, but in f32, heads of 32 and short
  // sequences.  In us, 32 and 64 rows, forward alone and with gradients, 1024 rows but for the last:
  //   32 heads of 128 x 128, bf16: 62, 214 and 47, 151;  128 such heads, bf16: 142, 710 and 143, 583, f32: 243, 928 and 298, 1006;
  //   512 heads of 64 x 64, bf16: 274, 1273 and 342, 1093, f32: 457, 1536 and 501, 1741;
  //   1024 heads of 64 x 64, 48 rows, bf16: 39, 151 and 63, 174, f32: 57, 220 and 79, 274.
  const int64_t tiles = d->sequences * d->Hv * ((d->V + 15) / 16);
  const bool many = tiles > 512 && (!saved || d->dtype == SEQ_FP32 || d->K <= 32 || d->T <= 64 || (d->offsets && d->T <= 64 * d->sequences));
  z.C = many || d->T <= 32 || (d->offsets && d->T <= 32 * d->sequences) ? 32 : 64;
  // (faster in every size tried, seq_delta_short.hip; it works with 32-bit offsets within a sequence)
  z.brief = !d->offsets && d->T > 0 && d->T <= 32 && std::max({d->v_stride[1], (int64_t)d->Hv * d->V, (int64_t)d->Hv * d->K}) < 1 << 25;
  const int NP = d->dtype + 1, NO = d->dtype == SEQ_FP32 ? 3 : 2, tri = z.C == 64 ? 6 : 2;
  z.per = (d->T + z.C - 1) / z.C;
  z.VP = (d->V + 15) / 16 * 16;
  // Two column tiles a workgroup, which share its loads, where one each would be more than a round.  In us, one and two, forward
  // alone and with gradients, 1024 rows of 128 x 128, bf16: 256 tiles 48, 159 and 65, 187; 512: 79, 355 and 69, 303; 768: 111, 530
  // and 117, 501; 1024: 162, 695 and 144, 583.  Packed sequences are of uneven length as a rule: the time is the longest one's, whose
  // chunks take longer with two, and the short ones' units are soon free for others.  8192 to 12288 rows cut at random, bf16: 320
  // tiles (10 sequences, 4 heads of 128 x 128) 73, 236 and 105, 306; 384 (12, 8 of 64 x 64) 96, 332 and 135, 391; 448 (14, 4 of 128 x
  // 128) 69, 227 and 85, 263; 512 (4, 16 of 128 x 128) 186, 775 and 196, 761; cut evenly, which the host cannot know: 64, 215 and 57,
  // 198; 80, 278 and 74, 250; 57, 200 and 51, 187; 163, 703 and 144, 597
  z.wide_cols = tiles > (d->offsets ? 512 : 256);
  z.chunks = d->offsets ? (d->sequences && d->T ? d->T / z.C + d->sequences + 1 : 0) : z.per * d->batch;
  // the largest launch of each kind: a sequence and head; a chunk and head; a sequence's column tiles (column_blocks)
  const int64_t groups = (z.VP / 16 + (z.wide_cols ? 1 : 0)) / (z.wide_cols ? 2 : 1);
  if (z.brief ? d->sequences > kMaxThreads / 256 / d->Hv
              : z.chunks > kMaxThreads / (4 * z.C) / d->Hv || d->sequences + 7 > kMaxThreads / (8 * z.C) / (d->Hv * groups))
    return fail(SEQ_EINVAL, "too many sequences, rows or heads for one launch");
  // sizes of DeltaShape: K, Q, K^T (saved: Q^T), each z.C x KP planes; X, P (saved: their transposes) as fragments
  z.kq = up256(z.chunks * d->Hk * ((saved ? 4LL : 3LL) * NP * z.C * z.KP * 2));
  z.xp = up256(z.chunks * d->Hv * ((saved ? 12LL : 3LL + NO) * tri * 1024));
  z.vec = up256(z.chunks * d->Hv * (int64_t)kVec);
  z.s0 = up256(z.chunks * d->Hv * 4 * z.KP * z.VP);
  z.u = up256(z.chunks * d->Hv * 4 * z.C * z.VP);
  const int64_t rows = d->batch * d->T;
  z.heads = d->Hv > d->Hk ? up256(rows * d->Hv * d->K * 4) : 0;
  if (z.brief) z.kq = z.xp = z.vec = z.s0 = z.u = 0;
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
  a.rows.C = z.C;
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
  a.wide_cols = z.wide_cols;
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

// ------------------------------------------------------------------------------------------------------ gated unit

struct UnitSizes {
  bool copy_x, copy_w;
  int few;   // the forward of a few rows: workgroups along the inner axis; 0: tiles
  int64_t D8, F8, x, w, da, sums, need;
};

int unit_sizes(const SeqUnit* u, bool backward, UnitSizes& z) {
  if (!u) return fail(SEQ_EINVAL, "NULL argument");
  if (u->dtype < SEQ_BF16 || u->dtype > SEQ_FP32) return fail(SEQ_EINVAL, "unknown dtype %d", u->dtype);
  if (u->act < SEQ_SILU || u->act > SEQ_SIGMOID) return fail(SEQ_EINVAL, "unknown activation %d", u->act);
  if (u->M < 0) return fail(SEQ_EINVAL, "negative number of rows");
  if (u->M > kUnitMaxRows) return fail(SEQ_EINVAL, "too many rows (%lld): up to %lld are supported", (long long)u->M, (long long)kUnitMaxRows);
  if (u->D < 1 || u->D > SEQ_UNIT_MAX || u->F < 1 || u->F > SEQ_UNIT_MAX)
    return fail(SEQ_EINVAL, "weights of %d x %d: 1 to %d are supported", u->D, u->F, SEQ_UNIT_MAX);
  const UnitParts way = backward ? unit_parts(u->M, u->D, u->F, u->dtype) : UnitParts{0, 1};
  const int64_t n = backward ? u->D : 2 * (int64_t)u->F;
  if (tile_threads(tile_for(u->M, n, true, 1, nullptr), u->M, n) > kMaxThreads || (backward && tile_threads(way.tile, u->D, 2 * (int64_t)u->F) > kMaxThreads))
    return fail(SEQ_EINVAL, "too many rows for one launch");
  const int np = u->dtype == SEQ_FP32 ? 3 : backward && u->dtype == SEQ_FP16 ? 2 : 1;   // planes of x and the weights
  z.D8 = (u->D + 7) / 8 * 8;
  z.F8 = (u->F + 7) / 8 * 8;
  // rows that loads of 16 bytes at 32-bit offsets do not fit
  z.copy_x = np > 1 || !aligned16(u->x) || u->x_ld % 8 || u->D % 8 || u->x_ld > 1 << 22;
  z.copy_w = np > 1 || !aligned16(u->wg) || !aligned16(u->wu) || u->wg_ld % 8 || u->wu_ld != u->wg_ld || u->F % 8 || u->wg_ld > 1 << 22;
  z.x = z.copy_x ? up256(u->M * z.D8 * 2 * np) : 0;
  z.w = z.copy_w ? up256(u->D * z.F8 * 2 * np) : 0;
  z.da = backward ? up256(u->M * z.F8 * 2 * np) : 0;
  z.sums = way.parts > 1 ? up256(way.parts * 8LL * u->D * u->F) : 0;
  z.need = z.x + 2 * z.w + 2 * z.da + z.sums;
  z.few = backward ? 0 : unit_few_splits(u->M, u->D, u->F, u->dtype);
  if (z.few) z.need = z.few > 1 ? up256(2LL * z.few * u->M * u->F * 4) : 0;
  return SEQ_OK;
}

void unit_args(const SeqUnit* u, const UnitSizes& z, void* work, UnitArgs& a) {
  memset(&a, 0, sizeof a);
  a.M = (int)u->M, a.D = u->D, a.F = u->F, a.act = u->act, a.dtype = u->dtype;
  a.x = u->x, a.wg = u->wg, a.wu = u->wu;
  a.x_ld = u->x_ld, a.w_ld = u->wg_ld, a.wu_ld = u->wu_ld;
  a.copy_x = z.copy_x, a.copy_w = z.copy_w, a.D8 = z.D8, a.F8 = z.F8;
  char* w = static_cast<char*>(work);
  a.xp = w;
  a.wgp = w + z.x;
  a.wup = a.wgp + z.w;
  a.dap = a.wup + z.w;
  a.dbp = a.dap + z.da;
  a.sums = reinterpret_cast<float*>(a.dbp + z.da);
}

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
    const DeltaOutside t = {1, {o}, {(int64_t)d->Hv * d->V * elem_size(d->dtype)}};
    const int e = hip_result(delta_outside(a.rows, t, s), "delta_rule");
    if (e) return e;
  }
  if (!d->sequences) return SEQ_OK;
  if (z.brief) return hip_result(delta_short_forward(a, d->dtype, z.KP, s), "delta_rule");
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
    hipError_t e;
    if (z.brief) {
      const bool wide_s = d->V % 4 == 0 && aligned16(d->initial) && aligned16(d_final);
      e = delta_short_backward(ga, d->dtype, z.KP, wide_s, s);
    } else {
      const bool wide_o = aligned16(d_o) && d->V % 8 == 0;
      e = delta_backward(ga, d->dtype, z.KP, wide_rows(d, d->V, d->v, d->v_stride), wide_o, s);
    }
    if (e == hipSuccess && z.heads) e = delta_heads(ga, d->dtype, s);
    rc = hip_result(e, "delta_rule backward");
  }
  if (rc || !d->offsets || !some) return rc;
  const int64_t size = elem_size(d->dtype), kb = (int64_t)d->Hk * d->K * size, vb = (int64_t)d->Hv * d->V * size, hb = (int64_t)d->Hv * 4;
  const DeltaOutside t = {5, {dq, dk, dv, dg, dbeta}, {kb, kb, vb, hb, hb}};
  return hip_result(delta_outside(ga.f.rows, t, s), "delta_rule backward");
}

int seq_delta_step(const SeqDeltaStep* d, void* stream) {
  if (!d) return fail(SEQ_EINVAL, "NULL argument");
  const int rc = check_heads(d->Hk, d->Hv, d->K, d->V, d->dtype);
  if (rc) return rc;
  if (d->batch < 0 || d->pool < 0) return fail(SEQ_EINVAL, "negative size");
  if (!d->slots && d->batch > d->pool) return fail(SEQ_EINVAL, "%lld rows and %lld states", (long long)d->batch, (long long)d->pool);
  if (d->batch > kMaxThreads / d->Hv) return fail(SEQ_EINVAL, "too many rows for one launch");
  const int64_t heads = d->batch * d->Hv, cols = step_cols(heads, d->V);
  if (heads > kMaxThreads / 256 / ((d->V + cols - 1) / cols)) return fail(SEQ_EINVAL, "too many rows for one launch");
  if (!d->batch) return SEQ_OK;
  if (!d->q || !d->k || !d->v || !d->g || !d->beta || !d->o || (d->pool && !d->state)) return fail(SEQ_EINVAL, "NULL buffer");
  ON_DEVICE(d->device);
  return hip_result(delta_step(*d, static_cast<hipStream_t>(stream)), "delta_step");
}

int seq_dropout(int32_t dtype, const void* x, const void* residual, void* y, int64_t n, int32_t below, uint64_t seed,
                uint64_t offset, const int64_t* seed_device, int32_t device, void* stream) {
  if (dtype < SEQ_BF16 || dtype > SEQ_FP32) return fail(SEQ_EINVAL, "unknown dtype %d", dtype);
  if (n < 0) return fail(SEQ_EINVAL, "negative size");
  if (below < 0 || below > 65536) return fail(SEQ_EINVAL, "below must be 0 to 65536 (got %d)", below);
  if (!n) return SEQ_OK;
  if (!x || !y) return fail(SEQ_EINVAL, "NULL buffer");
  ON_DEVICE(device);
  return hip_result(dropout(dtype, x, residual, y, n, (uint32_t)below, seed, offset, seed_device, static_cast<hipStream_t>(stream)),
                    "dropout");
}

int seq_unit_workspace(const SeqUnit* u, int32_t backward, int64_t* bytes) {
  UnitSizes z;
  const int rc = unit_sizes(u, backward != 0, z);
  if (rc) return rc;
  if (!bytes) return fail(SEQ_EINVAL, "NULL argument");
  *bytes = z.need;
  return SEQ_OK;
}

int seq_unit_forward(const SeqUnit* u, void* work, int64_t work_bytes, void* y, float* pre, void* stream) {
  UnitSizes z;
  int rc = unit_sizes(u, false, z);
  if (!rc) rc = check_memory("work", work, work_bytes, z.need);
  if (rc) return rc;
  if (!u->M) return SEQ_OK;
  if (!u->x || !u->wg || !u->wu || !y) return fail(SEQ_EINVAL, "NULL buffer");
  ON_DEVICE(u->device);
  UnitArgs a;
  unit_args(u, z, work, a);
  a.y = y, a.pre = pre;
  if (z.few) return hip_result(unit_few(a, z.few, static_cast<float*>(work), static_cast<hipStream_t>(stream)), "gated_unit");
  auto* f = a.dtype == SEQ_BF16 ? unit_forward_bf16 : a.dtype == SEQ_FP16 ? unit_forward_fp16 : unit_forward_fp32;
  return hip_result(f(a, static_cast<hipStream_t>(stream)), "gated_unit");
}

int seq_unit_backward(const SeqUnit* u, void* work, int64_t work_bytes, const float* pre, const void* dy, int64_t dy_ld,
                      void* dx, void* dwg, void* dwu, void* stream) {
  UnitSizes z;
  int rc = unit_sizes(u, true, z);
  if (!rc) rc = check_memory("work", work, work_bytes, z.need);
  if (rc) return rc;
  if (!u->wg || !u->wu || (u->M && (!u->x || !pre || !dy)) || !dwg != !dwu) return fail(SEQ_EINVAL, "NULL buffer");
  ON_DEVICE(u->device);
  UnitArgs a;
  unit_args(u, z, work, a);
  a.pre = const_cast<float*>(pre);   // read only
  a.dy = dy, a.dy_ld = dy_ld;
  a.dx = u->M ? dx : nullptr, a.dwg = dwg, a.dwu = dwu;
  auto* f = a.dtype == SEQ_BF16 ? unit_backward_bf16 : a.dtype == SEQ_FP16 ? unit_backward_fp16 : unit_backward_fp32;
  return hip_result(f(a, static_cast<hipStream_t>(stream)), "gated_unit backward");
}

}  // extern "C"
