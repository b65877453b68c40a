/*
 * seq_ops.h -- C ABI of libseqops.so: sequence-layer operators for MI355X (gfx950) beside the ADMM-LSTM step.
 *
 * They are what a recurrent model is built from next to the LSTM of blocks/lstm.py: the gated delta rule (a gated
 * recurrence with a matrix state), the gated unit (two projections, an activation and a product) and dropout whose
 * mask is recomputed from a counter instead of stored.  The Python entry points are blocks/delta_rule.py,
 * blocks/gated_unit.py and blocks/dropout.py, which call these through the extension _seq_torch (csrc/seq_torch.cpp);
 * admm_amd/_seq_native.py loads the library and declares the calls for ctypes.
 *
 * Conventions (those of admm_lstm.h)
 *  - Plain C types: device pointers, sizes, a hipStream_t passed as void*; strides are in elements.
 *  - 0 on success, a negative SEQ_E* code on failure; seq_last_error() has the thread's last message.
 *  - Enqueue-only on the given stream; nothing is allocated, nothing synchronises, nothing outlives the call.  Work
 *    memory is the caller's (seq_*_workspace gives its size); two calls that may overlap need two.
 *  - `device` is the HIP device that every pointer belongs to; the caller's current device is restored.
 *  - Every call may be captured into a HIP graph.
 *  - A call larger than a launch takes (2^32 threads along an axis) is refused before anything is enqueued.
 */
#ifndef SEQ_OPS_H
#define SEQ_OPS_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define SEQ_OPS_ABI_VERSION 1

enum { SEQ_OK = 0, SEQ_EINVAL = -1, SEQ_EHIP = -2 };
enum { SEQ_BF16 = 0, SEQ_FP16 = 1, SEQ_FP32 = 2 };
enum { SEQ_SILU = 0, SEQ_GELU = 1, SEQ_SIGMOID = 2 };

#define SEQ_DELTA_MAX_K 128      /* longest query/key row of the delta rule */
#define SEQ_DELTA_MAX_V 65536    /* longest value row */

int32_t seq_abi_version(void);
const char* seq_last_error(void);

/* The gated delta rule.  For each sequence n and value head h (query/key head h / (Hv / Hk)), with the state
 * S [K, V] starting at `initial` (NULL: zeros):
 *     S = exp(g_t) S;  u = beta_t (v_t - S^T k_t);  S = S + k_t u^T;  o_t = scale S^T q_t
 *
 * q, k [batch, T, Hk, K], v, o [batch, T, Hv, V] of `dtype`, g, beta [batch, T, Hv] float32; strides (batch, time, head)
 * in elements, the last axis contiguous (g, beta: stride of the head axis given too); o contiguous.
 * initial, final [sequences, Hv, K, V] float32, contiguous.
 * offsets (NULL: every batch row is a sequence): batch == 1 and sequence n is rows [offsets[n], offsets[n + 1]);
 * `sequences` + 1 non-decreasing int32 (offsets_64 = 0) or int64 values in [0, T] on the device.  Values outside are
 * taken as the nearest inside.  Rows of o that belong to no sequence are set to zero. */
typedef struct SeqDelta {
  int64_t batch, T, sequences;
  int32_t Hk, Hv, K, V;
  int32_t dtype, offsets_64;
  float scale;
  int32_t device;
  const void *q, *k, *v;
  const float *g, *beta;
  int64_t q_stride[3], k_stride[3], v_stride[3], g_stride[3], beta_stride[3];
  const void* offsets;
  const float* initial;
} SeqDelta;

/* Bytes of work memory: for the forward alone (saved = 0) or for a forward whose gradients follow (saved = 1; the same
 * memory is handed to the backward). */
int seq_delta_workspace(const SeqDelta* d, int32_t saved, int64_t* bytes);
int seq_delta_forward(const SeqDelta* d, int32_t saved, void* work, int64_t work_bytes, void* o, float* final_state,
                      void* stream);

/* Gradients.  `work` as the forward with saved = 1 left it; `scratch` is more work memory.  d_o contiguous like o, d_final
 * like final (NULL: zeros).  dq, dk, dv contiguous and of `dtype`, dg, dbeta contiguous float32, d_initial like
 * initial (NULL: not wanted).  Rows that belong to no sequence get zero gradients. */
int seq_delta_backward_scratch(const SeqDelta* d, int64_t* bytes);
int seq_delta_backward(const SeqDelta* d, const void* work, int64_t work_bytes, void* scratch, int64_t scratch_bytes,
                       const void* d_o, const float* d_final, void* dq, void* dk, void* dv, float* dg, float* dbeta,
                       float* d_initial, void* stream);

/* One token of each of `batch` streams; the state of row b is state[slots[b]] (slots NULL: state[b]) and is replaced.
 * q, k [batch, Hk, K], v, o [batch, Hv, V], g, beta [batch, Hv]; strides (batch, head) in elements, o contiguous.
 * state: `pool` states with the strides (slot, head) in elements, [K, V] contiguous.  A row whose slot is negative is idle: its
 * o is zero and no state changes.  A slot >= pool, or one that an earlier row names too, is refused in the kernel: o is NaN in
 * that row, and the row touches no state. */
typedef struct SeqDeltaStep {
  int64_t batch, pool;
  int32_t Hk, Hv, K, V;
  int32_t dtype, slots_64;
  float scale;
  int32_t device;
  const void *q, *k, *v;
  const float *g, *beta;
  int64_t q_stride[2], k_stride[2], v_stride[2], g_stride[2], beta_stride[2], state_stride[2];
  const void* slots;
  float* state;
  void* o;
} SeqDeltaStep;
int seq_delta_step(const SeqDeltaStep* d, void* stream);

/* Dropout: y_i = residual_i + (keep_i ? x_i * 65536 / (65536 - below) : 0) for n contiguous values, residual may be NULL, y may
 * be x or residual.  keep_i: 16 bits of Philox4x32-10 at counter (i / 8 in the low, offset in the high 64 bits) under the key
 * seed -- half (i % 2) of word (i % 8) / 2 -- are not below `below` (0..65536).  seed_device (NULL: `seed` counts): one
 * value on the device, read by the kernel. */
int seq_dropout(int32_t dtype, const void* x, const void* residual, void* y, int64_t n, int32_t below, uint64_t seed,
                uint64_t offset, const int64_t* seed_device, int32_t device, void* stream);

/* The gated unit y = act(x Wg) * (x Wu): x [M, D] with the row stride x_ld, Wg and Wu [D, F] with the row strides wg_ld and
 * wu_ld, y [M, F] contiguous, all of `dtype`; act: SEQ_SILU (z / (1 + exp(-z))), SEQ_GELU (the exact one, z Phi(z)) or
 * SEQ_SIGMOID. */
typedef struct SeqUnit {
  int64_t M;
  int32_t D, F, act, dtype, device;
  const void *x, *wg, *wu;
  int64_t x_ld, wg_ld, wu_ld;
} SeqUnit;

#define SEQ_UNIT_MAX 1048576     /* largest D and F (M: up to 2^31 - 256) */

/* Work memory of the forward (backward = 0) or the backward.  `pre` [2, M, F] float32 receives x Wg and x Wu for the
 * gradients, or is NULL.  dy [M, F] with the row stride dy_ld; dx [M, D], dwg and dwu [D, F] contiguous, dx and the pair dwg, dwu
 * may be NULL where they are not wanted. */
int seq_unit_workspace(const SeqUnit* u, int32_t backward, int64_t* bytes);
int seq_unit_forward(const SeqUnit* u, void* work, int64_t work_bytes, void* y, float* pre, void* stream);
int seq_unit_backward(const SeqUnit* u, void* work, int64_t work_bytes, const float* pre, const void* dy, int64_t dy_ld,
                      void* dx, void* dwg, void* dwu, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* SEQ_OPS_H */
