// seq_dropout.hip -- dropout whose mask is never stored: y = residual + x keep / P(keep), keep recomputed wherever needed.
//
// keep comes from Philox4x32-10 (J. Salmon et al., "Parallel random numbers: as easy as 1, 2, 3", 2011): a keyed bijection of
// a 128-bit counter, here (element / 8, offset) under the key seed.  Its 128 bits serve eight elements, 16 bits each:
// element 8 c + 2 w + h takes half h of word w and is dropped where those bits are below round(65536 p).
//
// Bound by memory: x (and the residual) read once, y written once, 16 bytes a lane where the tensors are aligned.  32 bits for
// each element would double the generator's multiplications (20 wide ones for a counter), which then take longer than the bytes.
// 16384 x 8191 bf16 with a residual: 155 us forward (5.2 TB/s), 88 us backward.
#include "seq_dev.hpp"

namespace seq {
namespace {

struct Drop {
  uint32_t key[2], offset[2];
  uint32_t below;   // 0..65536
  float factor;
};

__device__ __forceinline__ u32x4 philox(uint64_t c, const Drop& d) {
  u32x4 x = {(uint32_t)c, (uint32_t)(c >> 32), d.offset[0], d.offset[1]};
  uint32_t k0 = d.key[0], k1 = d.key[1];
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t a = (uint64_t)0xD2511F53u * x[0], b = (uint64_t)0xCD9E8D57u * x[2];
    x = u32x4{(uint32_t)(b >> 32) ^ x[1] ^ k0, (uint32_t)b, (uint32_t)(a >> 32) ^ x[3] ^ k1, (uint32_t)a};
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return x;
}

template <class T, bool RES>
__global__ __launch_bounds__(256) void k_dropout(const T* x, const T* res, T* y, int64_t n, Drop d, const int64_t* seed, bool wide) {
  if (seed) {   // the seed is on the device: a captured call draws a new mask when it changes
    const uint64_t s = (uint64_t)*seed;
    d.key[0] = (uint32_t)s;
    d.key[1] = (uint32_t)(s >> 32);
  }
  const int64_t groups = (n + 7) / 8;
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < groups; i += (int64_t)gridDim.x * 256) {
    const int left = n - 8 * i < 8 ? (int)(n - 8 * i) : 8;
    const f32x8 v = load8(x + 8 * i, left, wide);
    f32x8 r = {};
    if (RES) r = load8(res + 8 * i, left, wide);
    const u32x4 w = philox((uint64_t)i, d);
    typedef T T8 __attribute__((ext_vector_type(8)));
    T8 out;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t bits = j & 1 ? w[j >> 1] >> 16 : w[j >> 1] & 0xffffu;
      const float kept = bits >= d.below ? v[j] * d.factor : 0.f;
      out[j] = (T)(RES ? kept + r[j] : kept);
    }
    T* p = y + 8 * i;
    if (wide && left == 8) {
      if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<f32x4*>(p) = out.lo;
        *reinterpret_cast<f32x4*>(p + 4) = out.hi;
      } else {
        *reinterpret_cast<T8*>(p) = out;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < left) p[j] = out[j];
    }
  }
}

template <class T>
void launch(const void* x, const void* res, void* y, int64_t n, const Drop& d, const int64_t* seed, bool wide, hipStream_t s) {
  const int64_t want = (n + 2047) / 2048;
  const unsigned grid = (unsigned)(want < 256 * 64 ? want : 256 * 64);
  const T* xp = static_cast<const T*>(x);
  if (res) k_dropout<T, true><<<grid, 256, 0, s>>>(xp, static_cast<const T*>(res), static_cast<T*>(y), n, d, seed, wide);
  else k_dropout<T, false><<<grid, 256, 0, s>>>(xp, nullptr, static_cast<T*>(y), n, d, seed, wide);
}

}  // namespace

hipError_t dropout(int dtype, const void* x, const void* res, void* y, int64_t n, uint32_t below, uint64_t seed, uint64_t offset,
                   const int64_t* seed_dev, hipStream_t s) {
  const Drop d = {{(uint32_t)seed, (uint32_t)(seed >> 32)}, {(uint32_t)offset, (uint32_t)(offset >> 32)}, below,
                  below < 65536 ? 65536.f / (float)(65536 - below) : 0.f};
  const bool wide = (reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(res)) % 16 == 0;
  if (dtype == SEQ_BF16) launch<__bf16>(x, res, y, n, d, seed_dev, wide, s);
  else if (dtype == SEQ_FP16) launch<_Float16>(x, res, y, n, d, seed_dev, wide, s);
  else launch<float>(x, res, y, n, d, seed_dev, wide, s);
  return hipGetLastError();
}

}  // namespace seq
