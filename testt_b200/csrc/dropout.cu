// Dropout from a counter-based generator, with an optional residual add, for sm_100a:
//   y[i] = residual[i] + (w_i >= threshold ? x[i] * scale : 0)
// w_i is word i % 4 of Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as
// easy as 1, 2, 3", SC 2011) at counter offset + i / 4 under the key `seed`. The mask is a
// function of (seed, offset, i) alone, so it is never stored: the backward is the same kernel over
// dy, and the element type, the launch shape and the device do not change it. A dropped element is
// selected away, not multiplied by 0, so an infinity or NaN that is dropped leaves nothing.
//
// 33.6 M elements: fp16 x + fp32 residual -> fp32 50 us (336 MB, the memory's rate), the backward
// fp32 -> fp16 41 us (202 MB, 31 us at that rate): the generator's integer work then weighs as much
// as the bytes (issue 63 %, DRAM 48 %). Persistent CTAs with the next vector in flight took 55 / 46
// us. The seed from device memory costs nothing measurable (53 + 42 us against 52 + 41).
//
// Reference: solution/model.py:195-206 runs PyTorch's dropout, which stores a byte mask.
#include "dtypes.cuh"

namespace tb {
namespace {

constexpr int kThreads = 256;

// The four words of one counter. 10 rounds of two 32 x 32 -> 64 bit products.
__device__ __forceinline__ void philox(uint64_t counter, uint64_t seed, uint32_t *w) {
  uint32_t c0 = (uint32_t)counter, c1 = (uint32_t)(counter >> 32), c2 = 0, c3 = 0;
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c1 = (uint32_t)b;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  w[0] = c0; w[1] = c1; w[2] = c2; w[3] = c3;
}

// A thread draws for kAhead vectors of eight elements, two counters each.
template <int IN, int OUT, bool kRes, bool kVec, int kAhead>
__global__ void __launch_bounds__(kThreads)
    dropout_kernel(const void *__restrict__ x, const void *__restrict__ res, void *__restrict__ y,
                   int64_t n, const int64_t *__restrict__ state, int64_t *__restrict__ used,
                   uint64_t seed, uint64_t offset, uint32_t threshold, bool none, float scale) {
  pdl_wait();
  pdl_release();
  if (state != nullptr) {
    seed = (uint64_t)__ldg(state);
    offset += (uint64_t)__ldg(state + 1);
  }
  if (used != nullptr && blockIdx.x == 0 && threadIdx.x == 0) {
    used[0] = (int64_t)seed;
    used[1] = (int64_t)offset;
  }
  const int64_t nv = (n + 7) / 8, v0 = (int64_t)blockIdx.x * kThreads * kAhead + threadIdx.x;
  float f[kAhead][8], r[kAhead][8];
#pragma unroll
  for (int j = 0; j < kAhead; ++j) {
    const int64_t v = v0 + j * kThreads, i = v * 8;
    if (v >= nv) continue;
    if (kVec && i + 8 <= n) {
      load8<IN>(x, i, f[j]);
      if (kRes) load8<OUT>(res, i, r[j]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        f[j][e] = i + e < n ? load1<IN>(x, i + e) : 0.f;
        if (kRes) r[j][e] = i + e < n ? load1<OUT>(res, i + e) : 0.f;
      }
    }
  }
#pragma unroll
  for (int j = 0; j < kAhead; ++j) {
    const int64_t v = v0 + j * kThreads, i = v * 8;
    if (v >= nv) break;
    uint32_t w[8];
    philox(offset + (uint64_t)v * 2, seed, w);
    philox(offset + (uint64_t)v * 2 + 1, seed, w + 4);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float kept = w[e] >= threshold && !none ? f[j][e] * scale : 0.f;
      f[j][e] = kRes ? r[j][e] + kept : kept;
    }
    if (kVec && i + 8 <= n) {
      store8<OUT>(y, i, f[j]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (i + e < n) store1<OUT>(y, i + e, f[j][e]);
    }
  }
}

template <int IN, int OUT>
int run_dropout(const void *x, const void *res, void *y, int64_t n, const int64_t *state,
                int64_t *used, int64_t seed, int64_t offset, int64_t threshold, float scale,
                cudaStream_t st) {
  const bool none = threshold >= (1LL << 32);
  const uint32_t thr = none ? 0u : (uint32_t)threshold;
  const bool vec = aligned(x, 16) && aligned(y, 16) && (!res || aligned(res, 16));
  // two vectors a thread share the key schedule, which pays where there is no residual to read too
  // (33.6 M elements, fp32 -> fp16: 41 against 44 us; fp16 + fp32 residual: 56 against 50)
  const int64_t nv = (n + 7) / 8;
  const bool two = !res && nv > (int64_t)sm_count() * 4 * kThreads;
  const int64_t per = (int64_t)kThreads * (two ? 2 : 1), blocks = (nv + per - 1) / per;
  if (blocks > 0x7fffffffLL) return set_error(TB_EINVAL, "dropout: n %lld", (long long)n);
#define TB_DROPOUT(R, V, A)                                                                     \
  launch("dropout", dropout_kernel<IN, OUT, R, V, A>, dim3((unsigned)blocks), kThreads, 0, st,  \
         x, res, y, n, state, used, (uint64_t)seed, (uint64_t)offset, thr, none, scale)
  if (res) return vec ? TB_DROPOUT(true, true, 1) : TB_DROPOUT(true, false, 1);
  if (two) return vec ? TB_DROPOUT(false, true, 2) : TB_DROPOUT(false, false, 2);
  return vec ? TB_DROPOUT(false, true, 1) : TB_DROPOUT(false, false, 1);
#undef TB_DROPOUT
}

}  // namespace
}  // namespace tb

using namespace tb;

extern "C" int tb_dropout(const void *x, int32_t x_type, const void *residual, void *y,
                          int32_t y_type, int64_t n, int64_t threshold, float scale, int64_t seed,
                          int64_t offset, const int64_t *state, int64_t *used, void *stream) {
  if (!elem_type_ok(x_type) || !elem_type_ok(y_type) ||
      (x_type != y_type && x_type != TB_FP32 && y_type != TB_FP32))
    return set_error(TB_EINVAL, "dropout: types %d -> %d", x_type, y_type);
  if (n < 0 || threshold < 0 || threshold > (1LL << 32))
    return set_error(TB_EINVAL, "dropout: n %lld threshold %lld", (long long)n,
                     (long long)threshold);
  if (n == 0) return TB_OK;
  if (!x || !y) return set_error(TB_EINVAL, "dropout: x and y are required");
  const int ys = elem_size_of(y_type);
  if (!aligned(x, elem_size_of(x_type)) || !aligned(y, ys) || !aligned(residual, ys) ||
      !aligned(state, 8) || !aligned(used, 8))
    return set_error(TB_EALIGN, "dropout: a buffer is not aligned to its element");
  cudaStream_t st = as_stream(stream);
#define TB_RUN(A, B) \
  return run_dropout<A, B>(x, residual, y, n, state, used, seed, offset, threshold, scale, st)
  if (x_type == y_type) TB_WITH_TYPE(x_type, T, TB_RUN(T, T));
  if (y_type == TB_FP32) TB_WITH_TYPE(x_type, T, TB_RUN(T, TB_FP32));
  TB_WITH_TYPE(y_type, T, TB_RUN(TB_FP32, T));
#undef TB_RUN
}
