// Log-probabilities of given tokens with entropy and the top alternatives, from given logits, in
// one read of them, and their gradient in one read and one write; for sm_100a.
//   z = logits / T    lse = log sum e^z    p = e^(z - lse)
//   lp = z[id] - lse    H = lse - sum p z    top: the k largest (value descending, index ascending)
//   d logits = (1/T) (g_lp (1_id - p) + sum_j g_j (1_top_j - p) - g_H p (log p + H))
//
// Forward: an online softmax per thread over the raw logits x: a running maximum m, t = x - m,
// S = sum 2^(t c) with c = log2(e) / T, U = sum 2^(t c) t; lp = t_id / T - ln2 log2 S and
// H = ln2 log2 S - U / (S T). Differences, not products, are taken first, so logits of any size
// keep their precision. m counts as -FLT_MAX at least there, so t is never -inf - -inf: a -inf mask
// adds 2^-inf = 0 beside any finite logits, the type's lowest value included, and exponents are
// held at kFar where they are factors, so that 0 * t stays 0. A NaN makes the row's results NaN. A
// row of -inf only has S = 0, lp -inf, entropy 0 and no gradient.
//
// Top k without work per logit: every thread knows its own maximum (the softmax needs it anyway).
// The k-th largest of the threads' maxima is a lower bound of the row's k-th largest logit, and
// only threads whose maxima reach it (k of them, more with ties) own logits that do, so only their
// vectors are read again (from L2). Those logits become keys (ordered value << 32 | ~index), which
// all differ and settle ties by the lowest index, in descending lists over a warp's lanes.
//
// Measured (6.55 TB/s is a plain copy's rate):
//   2048 x 151936 bf16, top 5: forward 125 us (622 MB, 5.0 TB/s), backward 186 us (1245 MB, 6.7)
//   1531 x 50021 fp32, top 8: 70 us (306 MB, 4.3 TB/s) and 90 us (613 MB, 6.8)
//   621 x 151936 fp16: 44 us (189 MB, 4.3 TB/s; 4.2 rows an SM) and 55 us (377 MB, 6.9)
// The backward is bound by memory; no unit is full in the forward, whose CTAs wait for their
// vectors, then compute, then reduce (about 2 us a row an SM). Reading the next batch of vectors
// ahead costs registers or L1 and lost (57 against 48 us by registers; by a ring of copies 135
// against 125 at 2048 rows), and so did an eighth of the exponentials by a polynomial (129; their
// pipe is 63 % busy at 621 rows). What is not tried: the CTAs of a cluster sharing a row.
//
// Beside the head's statistics over given logits (solution/head.py:34-76, tb_head_stats_grad).
#include <math_constants.h>

#include "dtypes.cuh"

namespace tb {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
// 16-byte vectors in flight per thread of the forward, at five CTAs an SM (2048 x 151936 bf16:
// 124 us; 2 at eight CTAs 138, 3 at six 135, 6 at four 128, 8 at three 132).
constexpr int kUnroll = 4;
// Of the backward, and batches a CTA takes. 621 x 151936 fp16 / 2048 x 151936 bf16, in us: 2
// vectors by 4 batches 56 / 187, by 2 62 / 208, by 16 58 / 195; 4 by 4 59 / 193; 1 by 8 63 / 188.
constexpr int kBwdUnroll = 2, kBwdBatches = 4;
constexpr int kAgain = 2;        // vectors in flight per thread when they are read again
constexpr int kMaxTop = 32;      // one list entry per lane
// Logits are held at it where the sums' reference is known to be above -1e12: 2^.. is 0 for both.
constexpr float kLow = -1e20f;
constexpr float kFar = -1024.f;  // exponents are held at it where they are factors: 2^kFar is 0
constexpr float kLn2 = 0.693147180559945309f;
constexpr float kLog2e = 1.44269504088896341f;
constexpr uint32_t kAll = 0xffffffffu;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

template <int T>
constexpr int per_vec() {
  return 16 / elem_size<T>();
}

// A row as `head` columns up to a 16-byte boundary, nw whole vectors of E columns and `tail`
// columns. The (at most 2 E - 2) edge columns go one to a thread of the row's first split.
struct Row {
  const char *base;  // column 0
  int64_t nw;
  int head, edges;
};

template <int T>
__device__ __forceinline__ Row row_of(const void *logits, int64_t row, int64_t ld, int64_t vocab) {
  constexpr int E = per_vec<T>();
  Row r;
  r.base = static_cast<const char *>(logits) + row * ld * elem_size<T>();
  const int shift = (int)((reinterpret_cast<uintptr_t>(r.base) & 15) / elem_size<T>());
  r.head = (E - shift) % E;
  if (r.head > vocab) r.head = (int)vocab;
  r.nw = (vocab - r.head) / E;
  r.edges = (int)(vocab - r.nw * E);
  return r;
}

// Column of edge j.
template <int T>
__device__ __forceinline__ int64_t edge_col(const Row &r, int j) {
  return j < r.head ? j : r.nw * per_vec<T>() + j;
}

template <int T>
__device__ __forceinline__ void unpack_vec(const uint4 &v, float (&z)[per_vec<T>()]) {
  if constexpr (T == TB_FP32) {
    z[0] = __uint_as_float(v.x);
    z[1] = __uint_as_float(v.y);
    z[2] = __uint_as_float(v.z);
    z[3] = __uint_as_float(v.w);
  } else {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = Elem<T>::get2(w[i]);
      z[2 * i] = f.x;
      z[2 * i + 1] = f.y;
    }
  }
}

// Whole vector v of the row (columns head + v E + e).
template <int T>
__device__ __forceinline__ void load_vec(const Row &r, int64_t v, float (&z)[per_vec<T>()]) {
  const char *p = r.base + (int64_t)r.head * elem_size<T>() + v * 16;
  unpack_vec<T>(__ldg(reinterpret_cast<const uint4 *>(p)), z);
}

// A batch: the vectors p, p + kThreads, ..., N of them, in flight together.
template <int N>
__device__ __forceinline__ void load_batch(const uint4 *p, uint4 (&raw)[N]) {
#pragma unroll
  for (int b = 0; b < N; ++b) raw[b] = __ldg(p + b * kThreads);
}

// Monotone in (value, then lower index first); -0 counts as +0. 0: nothing.
__device__ __forceinline__ uint64_t make_key(float z, int64_t c) {
  const uint32_t b = __float_as_uint(z + 0.f);
  const uint32_t o = b & 0x80000000u ? ~b : b | 0x80000000u;
  return (uint64_t)o << 32 | (uint32_t)~(uint32_t)c;
}

__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t o = (uint32_t)(key >> 32);
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

__device__ __forceinline__ uint32_t key_index(uint64_t key) { return ~(uint32_t)key; }

// The warp's 32 values in descending order over the lanes.
__device__ __forceinline__ float warp_sort(float v, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size *= 2) {
#pragma unroll
    for (int stride = size / 2; stride > 0; stride /= 2) {
      const float other = __shfl_xor_sync(kAll, v, stride);
      const bool lower = (lane & stride) == 0, down = (lane & size) == 0 || size == 32;
      v = lower == down ? fmaxf(v, other) : fminf(v, other);
    }
  }
  return v;
}

// The 32 largest of two descending lists, descending.
template <typename K>
__device__ __forceinline__ K warp_merge(K a, K b, int lane) {
  const K r = __shfl_sync(kAll, b, 31 - lane);
  K key = a > r ? a : r;  // bitonic
#pragma unroll
  for (int stride = 16; stride > 0; stride /= 2) {
    const K other = __shfl_xor_sync(kAll, key, stride);
    key = ((lane & stride) == 0) == (key > other) ? key : other;
  }
  return key;
}

// The 32 largest of the warps' descending lists in warp 0, by pairs; `sh` [kWarps][32]. Ends with
// every warp's reads of sh done and warp 0's result its own (and in sh[0]).
template <typename K>
__device__ __forceinline__ K block_merge(K list, K (*sh)[32], int warp, int lane) {
  sh[warp][lane] = list;
  __syncthreads();
#pragma unroll
  for (int step = 1; step < kWarps; step *= 2) {
    if (warp % (2 * step) == 0) {
      list = warp_merge(list, sh[warp + step][lane], lane);
      sh[warp][lane] = list;
    }
    __syncthreads();
  }
  return list;
}

// Adds each lane's key (0: none) to the warp's descending list when it beats the k-th entry.
__device__ __forceinline__ void warp_insert(uint64_t &list, uint64_t key, int k, int lane) {
  const uint64_t kth = __shfl_sync(kAll, list, k - 1);
  uint32_t todo = __ballot_sync(kAll, key > kth);
  while (todo) {
    const int src = __ffs(todo) - 1;
    todo &= todo - 1;
    const uint64_t x = __shfl_sync(kAll, key, src);
    const int place = __popc(__ballot_sync(kAll, list > x));
    const uint64_t up = __shfl_up_sync(kAll, list, 1);
    list = lane < place ? list : lane == place ? x : up;
  }
}

struct State {  // max, and S and U about max(max, -FLT_MAX)
  float m, s, u;
};

__device__ __forceinline__ float reference(float m) { return fmaxf(m, -CUDART_MAX_NORMAL_F); }

// (s, u) about m moved to a reference m2 >= m.
__device__ __forceinline__ void move_to(float &s, float &u, float m, float m2, float c) {
  const float d = (m - m2) * c, f = ex2(d);
  u = f > 0.f ? f * (u + s * d) : 0.f;
  s *= f;
}

__device__ __forceinline__ State warp_merge_states(State a, float c) {
  float m = a.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kAll, m, o));
  move_to(a.s, a.u, reference(a.m), reference(m), c);
  a.m = m;
  a.s = warp_sum(a.s);
  a.u = warp_sum(a.u);
  return a;
}

// A thread's running sums. d is formed as fma(x, c, -M) with M = c ref rounded, which is one
// instruction less a logit than (x - ref) c; what M's rounding leaves, rho = c ref - M, is taken
// back batch by batch: 2^-rho s and 2^-rho (u - rho s). That holds for |M| below 1e8 (rho up to
// 4), and for fp16, whose -inf counts as -65504 there, while 2^((-65504 - ref) c) is 0; beyond,
// the difference is taken first.
template <int T>
struct Running {
  float m, s, u, ref, M, rho, back;
  bool small;

  __device__ __forceinline__ void set_ref(float c) {
    ref = reference(m);
    M = ref * c;
    rho = fmaf(ref, c, -M);
    small = fabsf(M) < 1e8f && (T != TB_FP16 || (ref + 65504.f) * c > 200.f);
    back = fabsf(rho) < 0x1p-10f ? fmaf(-rho, kLn2, 1.f) : ex2(-rho);
  }
  __device__ __forceinline__ void start(float c) {
    m = -CUDART_INF_F;
    s = u = 0.f;
    set_ref(c);
  }
  __device__ __forceinline__ void raise(float m2, float c) {
    move_to(s, u, ref, reference(m2), c);
    m = m2;
    set_ref(c);
  }
  __device__ __forceinline__ void add(float bs, float bu) {
    if (small) {
      bu = back * fmaf(-rho, bs, bu);
      bs *= back;
    }
    s += bs;
    u += bu;
  }
  __device__ __forceinline__ void one(float x, float c) {  // x below m already
    const float d = (x - ref) * c, p = ex2(d);
    s += p;
    u = fmaf(p, fmaxf(d, kFar), u);
  }
};

struct FwdArgs {
  const void *logits;
  const void *ids;  // int64 or int32
  float *logprob, *entropy, *top_lp, *stats;
  int64_t *top_ids;
  float4 *states;       // [rows, splits] partial states (splits > 1)
  uint64_t *lists;      // [rows, splits, k]
  int64_t rows, vocab, ld;
  int64_t split_vecs;   // vectors of a split
  int splits, k;
  bool ids64;
  float c, inv_t;
};

__device__ __forceinline__ int64_t id_of(const void *ids, bool ids64, int64_t row) {
  return ids64 ? static_cast<const int64_t *>(ids)[row]
               : (int64_t)static_cast<const int32_t *>(ids)[row];
}

// Log-probability of logit x in a row of state a, l = log2 S. The difference is halved where it may
// be past fp32 although its product with 1 / T is not.
__device__ __forceinline__ float logprob_of(float x, const State &a, float l, float inv_t) {
  if (a.m == -CUDART_INF_F) return l == l ? x : l;  // no logit above -inf, perhaps a NaN
  float d = (x - a.m) * inv_t;
  if (d == -CUDART_INF_F) d = 2.f * ((0.5f * x - 0.5f * a.m) * inv_t);
  return d - kLn2 * l;
}

// The row's given id and its logit (0 for an id outside).
template <int T>
__device__ __forceinline__ float logit_of(const FwdArgs &a, int64_t row, int64_t id) {
  return id >= 0 && id < a.vocab ? load1<T>(a.logits, row * a.ld + id) : 0.f;
}

// One warp writes a row's results. key: the row's list over the lanes; x: logit `id`.
__device__ __forceinline__ void finish_row(const FwdArgs &a, int64_t row, const State &st,
                                           uint64_t key, int64_t id, float x, int lane) {
  const float l = log2f(st.s);
  const bool empty = st.m == -CUDART_INF_F && st.s == st.s;
  if (lane == 0) {
    a.logprob[row] = id >= 0 && id < a.vocab ? logprob_of(x, st, l, a.inv_t) : 0.f;
    float h = kLn2 * (l - st.u / st.s);
    h = empty || h < 0.f ? 0.f : h;
    a.entropy[row] = h;
    a.stats[3 * row] = reference(st.m);
    a.stats[3 * row + 1] = empty ? CUDART_INF_F : l;
    a.stats[3 * row + 2] = h;
  }
  if (lane < a.k) {
    a.top_ids[row * a.k + lane] = key == 0 ? 0 : (int64_t)key_index(key);
    a.top_lp[row * a.k + lane] =
        key == 0 ? CUDART_NAN_F : logprob_of(key_value(key), st, l, a.inv_t);
  }
}

// The words of a vector held at kLow (fp16: at its lowest value) and above, and their maximum;
// 16-bit types two at a time.
template <int T>
struct Words;

template <>
struct Words<TB_FP16> {
  using type = __half2;
  static __device__ __forceinline__ type low() { return __float2half2_rn(-65504.f); }
};

template <>
struct Words<TB_BF16> {
  using type = __nv_bfloat162;
  static __device__ __forceinline__ type low() { return __float2bfloat162_rn(kLow); }
};

template <int T>
__device__ __forceinline__ uint32_t hold(uint32_t w) {
  if constexpr (T == TB_FP32) {
    return __float_as_uint(max_nan(__uint_as_float(w), kLow));
  } else {
    using W = typename Words<T>::type;
    const W v = __hmax2_nan(*reinterpret_cast<W *>(&w), Words<T>::low());
    return *reinterpret_cast<const uint32_t *>(&v);
  }
}

template <int T, int N>
__device__ __forceinline__ float batch_max(const uint4 (&raw)[N]) {
  if constexpr (T == TB_FP32) {
    float m = -CUDART_INF_F;
#pragma unroll
    for (int b = 0; b < N; ++b) {
      m = fmaxf(fmaxf(m, __uint_as_float(raw[b].x)), __uint_as_float(raw[b].y));
      m = fmaxf(fmaxf(m, __uint_as_float(raw[b].z)), __uint_as_float(raw[b].w));
    }
    return m;
  } else {
    using W = typename Words<T>::type;
    uint32_t none = T == TB_FP16 ? 0xfc00fc00u : 0xff80ff80u;  // two -inf
    W m = *reinterpret_cast<W *>(&none);
#pragma unroll
    for (int b = 0; b < N; ++b) {
      const uint32_t w[4] = {raw[b].x, raw[b].y, raw[b].z, raw[b].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) m = __hmax2(m, *reinterpret_cast<const W *>(&w[i]));
    }
    const float2 f = Elem<T>::get2(*reinterpret_cast<uint32_t *>(&m));
    return fmaxf(f.x, f.y);
  }
}

template <int T>
__device__ __forceinline__ void hold_vec(uint4 &v, float (&z)[per_vec<T>()]) {
  v.x = hold<T>(v.x);
  v.y = hold<T>(v.y);
  v.z = hold<T>(v.z);
  v.w = hold<T>(v.w);
  unpack_vec<T>(v, z);
}

template <int T, int N>
__device__ __forceinline__ void add_batch(Running<T> &r, uint4 (&raw)[N], float c) {
  constexpr int E = per_vec<T>();
  float s = 0.f, u = 0.f;
  if (r.small) {
#pragma unroll
    for (int b = 0; b < N; ++b) {
      float z[E];
      hold_vec<T>(raw[b], z);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float d = fmaf(z[e], c, -r.M), p = ex2(d);
        s += p;
        u = fmaf(p, d, u);
      }
    }
  } else {
#pragma unroll
    for (int b = 0; b < N; ++b) {
      float z[E];
      unpack_vec<T>(raw[b], z);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float d = (z[e] - r.ref) * c, p = ex2(d);
        s += p;
        u = fmaf(p, fmaxf(d, kFar), u);  // d may be past fp32: 0 times it is no NaN
      }
    }
  }
  r.add(s, u);
}

template <int T, bool kTop>
__global__ void __launch_bounds__(kThreads, T == TB_FP32 ? 6 : 5) logprobs_fwd(FwdArgs a) {
  pdl_wait();
  pdl_release();
  constexpr int E = per_vec<T>();
  __shared__ State sh_state[kWarps];
  __shared__ uint64_t sh_list[kWarps][32];
  __shared__ float sh_max[kWarps][32];
  __shared__ int sh_n;
  __shared__ uint16_t sh_who[kThreads];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = blockIdx.x / a.splits;
  const int split = (int)(blockIdx.x - row * a.splits);
  const Row r = row_of<T>(a.logits, row, a.ld, a.vocab);
  const int64_t v0 = split * a.split_vecs;
  const int64_t v1 = v0 + a.split_vecs < r.nw ? v0 + a.split_vecs : r.nw;
  const int edges = split == 0 ? r.edges : 0;
  Running<T> run;
  run.start(a.c);
  const uint4 *vecs = reinterpret_cast<const uint4 *>(r.base + r.head * elem_size<T>());
  int64_t v = v0 + threadIdx.x;
  for (; v + (kUnroll - 1) * kThreads < v1; v += kUnroll * kThreads) {
    uint4 raw[kUnroll];
    load_batch(vecs + v, raw);
    const float m = batch_max<T>(raw);
    if (m > run.m) run.raise(m, a.c);
    add_batch<T>(run, raw, a.c);
  }
  for (; v < v1; v += kThreads) {
    uint4 raw[1];
    load_batch(vecs + v, raw);
    const float m = batch_max<T>(raw);
    if (m > run.m) run.raise(m, a.c);
    add_batch<T>(run, raw, a.c);
  }
  const float own_max = run.m;  // of the whole vectors
  const int64_t id = id_of(a.ids, a.ids64, row);  // used at the end: in flight meanwhile
  uint64_t edge_key = 0;
  if ((int)threadIdx.x < edges) {
    const int64_t col = edge_col<T>(r, threadIdx.x);
    const float x = load1<T>(r.base, col);
    if (x == x) edge_key = make_key(x, col);
    if (x > run.m) run.raise(x, a.c);
    run.one(x, a.c);
  }
  State w = warp_merge_states(State{run.m, run.s, run.u}, a.c);
  if (lane == 0) sh_state[warp] = w;
  const float x_id = logit_of<T>(a, row, id);
  uint64_t list = 0;
  if constexpr (kTop) {
    // the k-th largest of the threads' maxima; their owners
    if (threadIdx.x == 0) sh_n = 0;
    const bool any_vec = v0 + threadIdx.x < v1;
    block_merge(warp_sort(any_vec ? own_max : -CUDART_INF_F, lane), sh_max, warp, lane);
    const float bar = sh_max[0][a.k - 1];
    if (any_vec && own_max >= bar) sh_who[atomicAdd(&sh_n, 1)] = (uint16_t)threadIdx.x;
    __syncthreads();
    // the owners' vectors once more, and the edges (the first warp holds them all)
    if (warp == 0) warp_insert(list, edge_key, a.k, lane);
    const int each = (int)((v1 - v0 + kThreads - 1) / kThreads), items = each * sh_n;
    const int span = (int)(v1 - v0);
    for (int i0 = warp * 32; i0 < items; i0 += kThreads * kAgain) {
      uint4 raw[kAgain];
      int at[kAgain];
#pragma unroll
      for (int b = 0; b < kAgain; ++b) {
        const int i = i0 + b * kThreads + lane, who = i / each;
        at[b] = i < items ? sh_who[who] + (i - who * each) * kThreads : span;
        if (at[b] < span) raw[b] = __ldg(vecs + v0 + at[b]);
      }
#pragma unroll
      for (int b = 0; b < kAgain; ++b) {
        float z[E];
        bool any = false;
        if (at[b] < span) {
          unpack_vec<T>(raw[b], z);
#pragma unroll
          for (int e = 0; e < E; ++e) any |= z[e] >= bar;
        }
        if (__ballot_sync(kAll, any) == 0) continue;
#pragma unroll
        for (int e = 0; e < E; ++e)
          warp_insert(list,
                      any && z[e] >= bar ? make_key(z[e], r.head + (v0 + at[b]) * E + e) : 0,
                      a.k, lane);
      }
    }
    list = block_merge(list, sh_list, warp, lane);
  } else {
    __syncthreads();  // sh_state
  }
  if (warp != 0) return;
  w = lane < kWarps ? sh_state[lane] : State{-CUDART_INF_F, 0.f, 0.f};
  w = warp_merge_states(w, a.c);
  if (a.splits == 1) {
    finish_row(a, row, w, list, id, x_id, lane);
  } else {
    if (lane == 0) a.states[blockIdx.x] = make_float4(w.m, w.s, w.u, 0.f);
    if (lane < a.k) a.lists[(int64_t)blockIdx.x * a.k + lane] = list;
  }
}

// A CTA per row over its splits' states and (descending) lists.
template <int T>
__global__ void __launch_bounds__(kThreads) logprobs_merge(FwdArgs a) {
  pdl_wait();
  pdl_release();
  __shared__ uint64_t sh_list[kWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = blockIdx.x;
  const int64_t id = id_of(a.ids, a.ids64, row);
  const float x_id = logit_of<T>(a, row, id);
  State w{-CUDART_INF_F, 0.f, 0.f};
  for (int i = lane; i < a.splits && warp == 0; i += 32) {
    const float4 q = a.states[row * a.splits + i];
    State o{q.x, q.y, q.z};
    const float m = fmaxf(w.m, o.m);
    move_to(w.s, w.u, reference(w.m), reference(m), a.c);
    move_to(o.s, o.u, reference(o.m), reference(m), a.c);
    w = State{m, w.s + o.s, w.u + o.u};
  }
  uint64_t list = 0;
  if (a.k > 0) {
    constexpr int kAhead = 8;
    const uint64_t *lists = a.lists + row * a.splits * a.k;
    for (int i0 = warp; i0 < a.splits; i0 += kWarps * kAhead) {
      uint64_t key[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int i = i0 + j * kWarps;
        key[j] = i < a.splits && lane < a.k ? lists[(int64_t)i * a.k + lane] : 0;
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
        if (i0 + j * kWarps < a.splits) list = warp_merge(list, key[j], lane);
    }
    list = block_merge(list, sh_list, warp, lane);
  }
  if (warp != 0) return;
  w = warp_merge_states(w, a.c);
  finish_row(a, row, w, list, id, x_id, lane);
}

struct BwdArgs {
  const void *logits;
  const void *ids;
  const int64_t *top_ids;
  const float *stats, *g_lp, *g_ent, *g_top;
  void *grad;
  int64_t rows, vocab, ld, ld_grad, split_vecs;
  int splits, k;
  bool ids64;
  float c, inv_t;
};

// p (G + g_H (log p + H)) of a logit: d = log2 p, A and B hold the factors.
__device__ __forceinline__ float slope(float x, float ref, float l, float c, float A, float B) {
  const float d = fmaf(x - ref, c, -l);
  return ex2(d) * fmaf(B, fmaxf(d, kFar), A);
}

template <int T>
__device__ __forceinline__ uint4 slopes(const uint4 &raw, float ref, float l, float c, float A,
                                        float B) {
  constexpr int E = per_vec<T>();
  float z[E];
  unpack_vec<T>(raw, z);
#pragma unroll
  for (int e = 0; e < E; ++e) z[e] = slope(z[e], ref, l, c, A, B);
  if constexpr (T == TB_FP32)
    return make_uint4(__float_as_uint(z[0]), __float_as_uint(z[1]), __float_as_uint(z[2]),
                      __float_as_uint(z[3]));
  else
    return make_uint4(Elem<T>::put2(z[0], z[1]), Elem<T>::put2(z[2], z[3]),
                      Elem<T>::put2(z[4 % E], z[5 % E]), Elem<T>::put2(z[6 % E], z[7 % E]));
}

template <int T>
__global__ void __launch_bounds__(kThreads) logprobs_bwd(BwdArgs a) {
  pdl_wait();
  pdl_release();
  constexpr int E = per_vec<T>();
  __shared__ int64_t sh_col[kMaxTop + 1];
  __shared__ float sh_g[kMaxTop + 1];
  const int64_t row = blockIdx.x / a.splits;
  const int split = (int)(blockIdx.x - row * a.splits);
  const Row r = row_of<T>(a.logits, row, a.ld, a.vocab);
  char *out = static_cast<char *>(a.grad) + row * a.ld_grad * elem_size<T>();
  const int64_t v0 = split * a.split_vecs;
  const int64_t v1 = v0 + a.split_vecs < r.nw ? v0 + a.split_vecs : r.nw;
  const int edges = split == 0 ? r.edges : 0;
  if ((int)threadIdx.x <= a.k) {
    const int j = threadIdx.x;
    int64_t col = j == 0 ? id_of(a.ids, a.ids64, row) : a.top_ids[row * a.k + j - 1];
    float g = j == 0 ? (a.g_lp ? a.g_lp[row] : 0.f) : (a.g_top ? a.g_top[row * a.k + j - 1] : 0.f);
    if (col < 0 || col >= a.vocab) {
      col = -1;
      g = 0.f;
    }
    sh_col[j] = col;
    sh_g[j] = g;
  }
  __syncthreads();
  float G = 0.f;
  for (int j = 0; j <= a.k; ++j) G += sh_g[j];
  const float ref = a.stats[3 * row];
  const bool empty = a.stats[3 * row + 1] == CUDART_INF_F;
  const float l = empty ? 0.f : a.stats[3 * row + 1];
  const float gh = a.g_ent ? a.g_ent[row] : 0.f;
  const float A = empty ? 0.f : -a.inv_t * (G + gh * a.stats[3 * row + 2]);
  const float B = empty ? 0.f : -a.inv_t * gh * kLn2;
  const uint4 *vecs = reinterpret_cast<const uint4 *>(r.base + r.head * elem_size<T>());
  uint4 *out_vecs = reinterpret_cast<uint4 *>(out + r.head * elem_size<T>());
  int64_t v = v0 + threadIdx.x;
  for (; v + (kBwdUnroll - 1) * kThreads < v1; v += kBwdUnroll * kThreads) {
    uint4 raw[kBwdUnroll];
    load_batch(vecs + v, raw);
#pragma unroll
    for (int b = 0; b < kBwdUnroll; ++b)
      out_vecs[v + b * kThreads] = slopes<T>(raw[b], ref, l, a.c, A, B);
  }
  for (; v < v1; v += kThreads) out_vecs[v] = slopes<T>(__ldg(vecs + v), ref, l, a.c, A, B);
  if ((int)threadIdx.x < edges) {
    const int64_t col = edge_col<T>(r, threadIdx.x);
    store1<T>(out, col, slope(load1<T>(r.base, col), ref, l, a.c, A, B));
  }
  if (empty) return;
  __syncthreads();  // the given and top columns are written again, with their one-hot terms
  if ((int)threadIdx.x <= a.k && sh_col[threadIdx.x] >= 0) {
    const int64_t col = sh_col[threadIdx.x], v = (col - r.head) / E;
    const bool edge = col < r.head || v >= r.nw;
    if (edge ? split == 0 : v >= v0 && v < v1) {
      float g = 0.f;
      for (int j = 0; j <= a.k; ++j) g += sh_col[j] == col ? sh_g[j] : 0.f;
      store1<T>(out, col, fmaf(g, a.inv_t, slope(load1<T>(r.base, col), ref, l, a.c, A, B)));
    }
  }
}

// Splits of a row: four CTAs an SM when there are few rows (621 rows of 151936 fp16: 44 us unsplit,
// 46 + 3 us for the merge in two, 45 + 3 in four).
int64_t splits_of(int64_t rows, int64_t vecs, int64_t target) {
  int64_t s = (target + rows - 1) / rows;
  const int64_t most = (vecs + kThreads - 1) / kThreads;
  if (s > most) s = most;
  return s < 1 ? 1 : s;
}

int64_t most_vecs(int64_t vocab, int es) { return (vocab * es + 15) / 16; }

int check(const char *what, int64_t rows, int64_t vocab, int64_t ld, int type, int k, float t) {
  if (rows < 0 || vocab <= 0 || vocab > 0x7fffffffLL || rows > 0x7fffffffLL / 1024 ||
      (rows > 1 && ld < vocab))
    return set_error(TB_EINVAL, "%s: rows %lld vocab %lld row stride %lld", what, (long long)rows,
                     (long long)vocab, (long long)ld);
  if (!elem_type_ok(type)) return set_error(TB_EINVAL, "%s: type %d", what, type);
  if (k < 0 || k > kMaxTop || k > vocab)
    return set_error(TB_EINVAL, "%s: top %d (0 to %d, at most the vocabulary)", what, k, kMaxTop);
  if (!(t >= 1e-4f && t <= 1e4f))
    return set_error(TB_EINVAL, "%s: temperature %g outside [1e-4, 1e4]", what, (double)t);
  return TB_OK;
}

int64_t fwd_splits(int64_t rows, int64_t vocab, int type) {
  return splits_of(rows, most_vecs(vocab, elem_size_of(type)), (int64_t)sm_count() * 4);
}

}  // namespace
}  // namespace tb

using namespace tb;

extern "C" int64_t tb_token_logprobs_workspace(int64_t rows, int64_t vocab, int32_t type,
                                               int32_t top_k) {
  if (rows <= 0 || vocab <= 0 || top_k < 0 || !elem_type_ok(type)) return 0;
  const int64_t s = fwd_splits(rows, vocab, type);
  return s > 1 ? rows * s * (16 + 8 * (int64_t)top_k) : 0;
}

extern "C" int tb_token_logprobs_fwd(const void *logits, int32_t type, int64_t ld, const void *ids,
                                     int32_t ids_int64, float temperature, int32_t top_k,
                                     float *logprob, float *entropy, float *top_logprobs,
                                     int64_t *top_ids, float *stats, int64_t rows, int64_t vocab,
                                     void *workspace, int64_t workspace_bytes, void *stream) {
  int rc = check("token_logprobs_fwd", rows, vocab, ld, type, top_k, temperature);
  if (rc != TB_OK) return rc;
  if (rows == 0) return TB_OK;
  if (!logits || !ids || !logprob || !entropy || !stats ||
      (top_k > 0 && (!top_logprobs || !top_ids)))
    return set_error(TB_EINVAL, "token_logprobs_fwd: a buffer is missing");
  if (!aligned(logits, elem_size_of(type)) || !aligned(ids, ids_int64 ? 8 : 4) ||
      !aligned(logprob, 4) || !aligned(entropy, 4) || !aligned(stats, 4) ||
      !aligned(top_logprobs, 4) || !aligned(top_ids, 8) || !aligned(workspace, 16))
    return set_error(TB_EALIGN, "token_logprobs_fwd: a buffer is not aligned to its element");
  const int64_t need = tb_token_logprobs_workspace(rows, vocab, type, top_k);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return set_error(TB_EINVAL, "token_logprobs_fwd: workspace of %lld bytes, %lld needed",
                     (long long)workspace_bytes, (long long)need);
  const int64_t splits = fwd_splits(rows, vocab, type);
  const int64_t nv = most_vecs(vocab, elem_size_of(type));
  char *ws = static_cast<char *>(workspace);
  const FwdArgs a{logits, ids, logprob, entropy, top_logprobs, stats, top_ids,
                  reinterpret_cast<float4 *>(ws),
                  reinterpret_cast<uint64_t *>(ws + rows * splits * 16), rows, vocab, ld,
                  (nv + splits - 1) / splits, (int)splits, top_k, ids_int64 != 0,
                  kLog2e / temperature, 1.f / temperature};
  cudaStream_t st = as_stream(stream);
  const dim3 grid((unsigned)(rows * splits));
  TB_WITH_TYPE(type, T,
               rc = top_k > 0 ? launch("token_logprobs_fwd", logprobs_fwd<T, true>, grid, kThreads,
                                       0, st, a)
                              : launch("token_logprobs_fwd", logprobs_fwd<T, false>, grid,
                                       kThreads, 0, st, a);
               if (rc == TB_OK && splits > 1) rc =
                   launch("token_logprobs_fwd", logprobs_merge<T>, dim3((unsigned)rows), kThreads,
                          0, st, a));
  return rc;
}

extern "C" int tb_token_logprobs_bwd(const void *logits, int32_t type, int64_t ld, const void *ids,
                                     int32_t ids_int64, float temperature, int32_t top_k,
                                     const int64_t *top_ids, const float *stats,
                                     const float *g_logprob, const float *g_entropy,
                                     const float *g_top, void *grad, int64_t ld_grad, int64_t rows,
                                     int64_t vocab, void *stream) {
  int rc = check("token_logprobs_bwd", rows, vocab, ld, type, top_k, temperature);
  if (rc != TB_OK) return rc;
  if (rows == 0) return TB_OK;
  if (!logits || !ids || !stats || !grad || (top_k > 0 && !top_ids))
    return set_error(TB_EINVAL, "token_logprobs_bwd: a buffer is missing");
  if (rows > 1 && ld_grad < vocab)
    return set_error(TB_EINVAL, "token_logprobs_bwd: gradient row stride %lld", (long long)ld_grad);
  const int es = elem_size_of(type);
  if (!aligned(logits, es) || !aligned(ids, ids_int64 ? 8 : 4) || !aligned(top_ids, 8) ||
      !aligned(stats, 4) || !aligned(g_logprob, 4) || !aligned(g_entropy, 4) ||
      !aligned(g_top, 4))
    return set_error(TB_EALIGN, "token_logprobs_bwd: a buffer is not aligned to its element");
  // each gradient row lies in its 16-byte words as the logits' row does
  if (((reinterpret_cast<uintptr_t>(logits) ^ reinterpret_cast<uintptr_t>(grad)) & 15) != 0 ||
      (rows > 1 && (ld - ld_grad) * es % 16 != 0))
    return set_error(TB_EALIGN, "token_logprobs_bwd: the gradient's rows must lie modulo 16 bytes "
                                "as the logits' rows do");
  if (grad == logits)  // the columns with a one-hot term are read again after the row is written
    return set_error(TB_EINVAL, "token_logprobs_bwd: grad is the logits themselves");
  const int64_t nv = most_vecs(vocab, es);
  const int64_t per = (int64_t)kThreads * kBwdUnroll * kBwdBatches;
  int64_t splits = (nv + per - 1) / per;
  if (splits > 1024) splits = 1024;
  const BwdArgs a{logits, ids, top_ids, stats, g_logprob, g_entropy, g_top, grad, rows,
                  vocab, ld, ld_grad, (nv + splits - 1) / splits, (int)splits, top_k,
                  ids_int64 != 0, kLog2e / temperature, 1.f / temperature};
  cudaStream_t st = as_stream(stream);
  TB_WITH_TYPE(type, T,
               return launch("token_logprobs_bwd", logprobs_bwd<T>,
                             dim3((unsigned)(rows * splits)), kThreads, 0, st, a));
}
