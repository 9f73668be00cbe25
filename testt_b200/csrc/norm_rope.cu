// Per-head RMS norms of queries and keys with the rotation (and the LoRA add) in the same pass,
// token-major, forward and backward, for sm_100a. For each token and each q / k head, in fp32:
//   x = qkv + lora     r = rsqrt(mean(x^2) + eps)     n = x r (w0 + w)
//   y_i = n_i cos_i - n_{i+h} sin_i,  y_{i+h} = n_{i+h} cos_{i+h} + n_i sin_{i+h},  h = rot / 2
// dims past rot are not turned; v = qkv + lora. Rounded once, on the store. Backward:
//   dn = the transposed rotation of dy     g = dn (w0 + w)     dx = r (g - x r^2 mean(g x))
//   dw = sum over tokens and heads of dn x r
// x is read again and both means come out of one set of shuffles, so the forward stores nothing
// for the backward. dw: each lane keeps its sums over its warp's tokens; they are added in order of
// the lanes, then (a second kernel) of the CTAs, so results do not depend on timing.
//
// 16411 tokens of 32 + 8 + 8 heads of 128, half of each turned, bf16: forward 82 us (403 MB, 4.9
// TB/s), backward 131 + 3 us (571 MB, 4.4 TB/s); a plain copy runs at 6.55 TB/s. No unit is full:
// the time goes into fixed and shared-memory latencies at 24 and 16 warps an SM. One CTA a token
// with everything in registers took 259 / 291 us (one CTA an SM), deeper rings change nothing; bulk
// copies of a token's whole rows are not tried. Packed fp32 pairs halve
// the arithmetic's issue slots; the rotation's factors lie in shared memory once a warp and token,
// as 32 registers less a lane allow half as many warps again.
//
// Beside tb_rope_tokens_* (solution/rope.py:24-176), which has no norm; positions and tables as
// there. The reference's model has no head norms.
#include <initializer_list>
#include <type_traits>

#include "dtypes.cuh"

namespace tb {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kFwdPerSm = 3, kBwdPerSm = 2;  // resident CTAs of the vector kernels
constexpr uint32_t kAll = 0xffffffffu;

struct NormDims {
  int64_t rows, ld, slots;  // tokens, elements between qkv rows, batch * seq
  int nh, nkv, d, rot;
  float eps, w0, inv_d;
};

// V neighbouring values as loaded (16 bytes, or 8 for four 16-bit values) and as fp32 pairs.
template <int T, int V>
struct Vec {
  using type = typename std::conditional<V == 8, uint4, uint2>::type;
  static __device__ __forceinline__ void get(const type &v, F2 (&f)[V / 2]) {
    const uint32_t *w = reinterpret_cast<const uint32_t *>(&v);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const float2 a = Elem<T>::get2(w[i]);
      f[i] = make_f2(a.x, a.y);
    }
  }
  static __device__ __forceinline__ type put(const F2 (&f)[V / 2]) {
    type v;
    uint32_t *w = reinterpret_cast<uint32_t *>(&v);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const float2 a = parts(f[i]);
      w[i] = Elem<T>::put2(a.x, a.y);
    }
    return v;
  }
};

template <int V>
struct Vec<TB_FP32, V> {
  struct type {
    float4 q[V / 4];
  };
  static __device__ __forceinline__ void get(const type &v, F2 (&f)[V / 2]) {
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      f[2 * i] = make_f2(v.q[i].x, v.q[i].y);
      f[2 * i + 1] = make_f2(v.q[i].z, v.q[i].w);
    }
  }
  static __device__ __forceinline__ type put(const F2 (&f)[V / 2]) {
    type v;
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      const float2 a = parts(f[2 * i]), b = parts(f[2 * i + 1]);
      v.q[i] = make_float4(a.x, a.y, b.x, b.y);
    }
    return v;
  }
};

template <int T, int V>
__device__ __forceinline__ typename Vec<T, V>::type load_raw(const void *p, int64_t i) {
  const typename Elem<T>::type *q = static_cast<const typename Elem<T>::type *>(p) + i;
  if constexpr (T == TB_FP32) {
    typename Vec<T, V>::type v;
#pragma unroll
    for (int j = 0; j < V / 4; ++j) v.q[j] = __ldg(reinterpret_cast<const float4 *>(q) + j);
    return v;
  } else {
    return __ldg(reinterpret_cast<const typename Vec<T, V>::type *>(q));
  }
}

template <int V>
__device__ __forceinline__ void fill(F2 (&f)[V], float v) {
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = both(v);
}

// Sum over groups of `lanes` (a power of two) neighbouring lanes; every lane gets the total.
__device__ __forceinline__ float group_sum(float v, int lanes) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (o < lanes) v += __shfl_xor_sync(kAll, v, o);
  return v;
}

// Output (or gradient) row of head row hr: q [rows, nh, d], k and v [rows, nkv, d].
template <typename P>
__device__ __forceinline__ P pick(P q, P k, P v, const NormDims &dm, int64_t tok, int hr,
                                  int64_t &at) {
  if (hr < dm.nh) {
    at = (tok * dm.nh + hr) * (int64_t)dm.d;
    return q;
  }
  const bool key = hr < dm.nh + dm.nkv;
  at = (tok * dm.nkv + hr - dm.nh - (key ? 0 : dm.nkv)) * (int64_t)dm.d;
  return key ? k : v;
}

// How the vector kernels spread head rows: `lanes` lanes to a head row, each with two chunks of V
// dims (lanes below rot / 2V a rotation's pair, one chunk of each half; the others two neighbouring
// chunks of the rest), 32 / lanes head rows of one kind (q, k or v) to a group, a group to a warp
// at a time. `parts` warps share a token's groups (one, when there are many tokens).
struct Spread {
  int lanes, at_once, gq, gk, groups, parts;  // groups of q, of k (and of v), all of them
};

template <int V>
struct Lane {
  int a, b, slot;  // first dims of the two chunks; the head row in the group
  bool live, turn;
  __device__ __forceinline__ Lane(const NormDims &dm, const Spread &sp) {
    const int lane = threadIdx.x & (sp.lanes - 1), pairs = dm.rot / (2 * V);
    slot = (threadIdx.x & 31) / sp.lanes;
    turn = lane < pairs;
    a = turn ? lane * V : dm.rot + (lane - pairs) * 2 * V;
    b = turn ? dm.rot / 2 + lane * V : a + V;
    live = lane < dm.d / (2 * V);
  }
};

// w0 + weight of q and of k in fp32, in shared memory ([2][d]); 1 without a weight.
template <int W>
__device__ __forceinline__ void stage_weights(float *ws, const void *qw, const void *kw, float w0,
                                              int d) {
  for (int i = threadIdx.x; i < 2 * d; i += kThreads) {
    const void *w = i < d ? qw : kw;
    ws[i] = w == nullptr ? 1.f : w0 + load1<W>(w, i < d ? i : i - d);
  }
}

// ---- the walk of the vector kernels ----------------------------------------------------------
// The rows of the next stages - 1 groups of a warp's walk are on their way into the lane's own
// slots of shared memory (cp.async: no registers held, and no barrier, since a lane reads only what
// it copied).

constexpr int kFwdStages = 3, kBwdStages = 3;

template <int B>
__device__ __forceinline__ void copy_async(void *dst, const void *src) {
  if constexpr (B == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src)
                 : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(dst)), "l"(src),
                 "n"(B)
                 : "memory");
}

__device__ __forceinline__ void copies_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}

template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A warp's walk: groups part, part + parts, ... of tokens tok, + stride, ...
struct Walk {
  int part;
  int64_t tok, stride;
  __device__ __forceinline__ Walk(const NormDims &dm, const Spread &sp) {
    const int wid = blockIdx.x * kWarps + (threadIdx.x >> 5);
    part = wid % sp.parts;
    stride = (int)gridDim.x * kWarps / sp.parts;
    tok = wid / sp.parts < stride ? wid / sp.parts : dm.rows;  // leftover warps do nothing
  }
};

// Where the walk's copies are, stages - 1 groups ahead of the work: the lane's place in the qkv row
// and in the kind's gradient or LoRA-shaped rows, moved on by constants within a kind.
struct Ahead {
  int64_t tok;
  int g, end, left;  // group, first of the next kind, head rows from the lane's to the kind's end
  int kind;
  const char *x, *y;

  // bases: of q-, k- and v-shaped rows (may be NULL); es: bytes of an element
  __device__ __forceinline__ void locate(const NormDims &dm, const Spread &sp, const Walk &wk,
                                         int slot, const char *qkv, const char *bq,
                                         const char *bk, const char *bv, int es) {
    if (g >= sp.groups) {
      g = wk.part;
      tok += wk.stride;
    }
    kind = g < sp.gq ? 0 : g < sp.gq + sp.gk ? 1 : 2;
    const int start = kind == 0 ? 0 : kind == 1 ? sp.gq : sp.gq + sp.gk;
    end = kind == 0 ? sp.gq : kind == 1 ? sp.gq + sp.gk : sp.groups;
    const int n = kind == 0 ? dm.nh : dm.nkv, head = (g - start) * sp.at_once + slot;
    const int first = kind == 0 ? 0 : kind == 1 ? dm.nh : dm.nh + dm.nkv;
    left = tok < dm.rows ? n - head : 0;
    x = qkv + (tok * dm.ld + (first + head) * dm.d) * es;
    y = kind == 0 ? bq : kind == 1 ? bk : bv;
    if (y != nullptr) y += (tok * n + head) * (int64_t)dm.d * es;
  }
  __device__ __forceinline__ bool next(const Spread &sp, int step, int bytes) {
    g += sp.parts;
    left -= step;
    x += bytes;
    y += bytes;
    return g < end;
  }
};

// A warp's table of a token's rotation in shared memory, four rows of fp32 quads laid out
// [row][quad][lane]: all its head rows use the same factors, so a lane reads them where it needs
// them instead of holding 4 V registers. Forward rows: y1 = r (x1 A + x2 B), y2 = r (x2 C + x1 D)
// with the weights inside (A = w1 c1, B = -w2 s1, C = w2 c2, D = w1 s2); backward rows: c1, -s1,
// c2, s2. Lanes past rot turn by cosine 1, sine 0. The head rows' lanes share the work.
template <int V, bool kWeights>
__device__ __forceinline__ void make_table(float4 *tab, const float *cosv, const float *sinv,
                                           int64_t row, const float *w, const Lane<V> &ln,
                                           const Spread &sp) {
  const int lane = threadIdx.x & (sp.lanes - 1);
  __syncwarp();
  for (int i = ln.slot; i < V / 4 && ln.live; i += sp.at_once) {
    float4 c1 = make_float4(1.f, 1.f, 1.f, 1.f), c2 = c1;
    float4 s1 = make_float4(0.f, 0.f, 0.f, 0.f), s2 = s1;
    if (ln.turn) {
      c1 = __ldg(reinterpret_cast<const float4 *>(cosv + row + ln.a) + i);
      c2 = __ldg(reinterpret_cast<const float4 *>(cosv + row + ln.b) + i);
      s1 = __ldg(reinterpret_cast<const float4 *>(sinv + row + ln.a) + i);
      s2 = __ldg(reinterpret_cast<const float4 *>(sinv + row + ln.b) + i);
    }
    float4 w1 = make_float4(1.f, 1.f, 1.f, 1.f), w2 = w1;
    if (kWeights) {
      w1 = reinterpret_cast<const float4 *>(w + ln.a)[i];
      w2 = reinterpret_cast<const float4 *>(w + ln.b)[i];
    }
    float4 *t = tab + i * sp.lanes + lane;
    const int next = (V / 4) * sp.lanes;
    t[0] = make_float4(w1.x * c1.x, w1.y * c1.y, w1.z * c1.z, w1.w * c1.w);
    const float4 m = kWeights ? w2 : w1;
    t[next] = make_float4(-m.x * s1.x, -m.y * s1.y, -m.z * s1.z, -m.w * s1.w);
    t[2 * next] = make_float4(w2.x * c2.x, w2.y * c2.y, w2.z * c2.z, w2.w * c2.w);
    t[3 * next] = make_float4(w1.x * s2.x, w1.y * s2.y, w1.z * s2.z, w1.w * s2.w);
  }
  __syncwarp();
}

struct Quad2 {
  F2 lo, hi;
};

__device__ __forceinline__ Quad2 quad_at(const float4 *p) {
  const float4 q = *p;
  return Quad2{make_f2(q.x, q.y), make_f2(q.z, q.w)};
}

template <int V>
__device__ __forceinline__ float square_sum(const F2 (&x1)[V], const F2 (&x2)[V]) {
  F2 s = both(0.f), t = s;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    s = fma2(x1[i], x1[i], s);
    t = fma2(x2[i], x2[i], t);
  }
  const float2 p = parts(add2(s, t));
  return p.x + p.y;
}

// W: the weights' type, L: the LoRA rows'. The weights are folded into a token's factors, so that a
// pair costs four multiply-adds and two products with r.
template <int T, int V, int L, int W>
__global__ void __launch_bounds__(kThreads, kFwdPerSm)
    norm_rope_fwd(const void *__restrict__ qkv, const void *__restrict__ lq,
                  const void *__restrict__ lv, const void *__restrict__ qw,
                  const void *__restrict__ kw, const float *__restrict__ cosv,
                  const float *__restrict__ sinv, const int64_t *__restrict__ pos_idx, void *q,
                  void *k, void *v, NormDims dm, Spread sp, FastDiv seq_div) {
  pdl_wait();
  pdl_release();
  using Raw = typename Vec<T, V>::type;
  constexpr int kB = V * elem_size<T>(), es = elem_size<T>();
  extern __shared__ uint4 shared[];
  Raw(*ring)[2][kThreads] = reinterpret_cast<Raw(*)[2][kThreads]>(shared);
  float *ws = reinterpret_cast<float *>(ring + kFwdStages);
  float4 *tab = reinterpret_cast<float4 *>(ws + 2 * dm.d) + (threadIdx.x >> 5) * V * sp.lanes;
  const float4 *mine = tab + (threadIdx.x & (sp.lanes - 1));
  const Lane<V> ln(dm, sp);
  const Walk wk(dm, sp);
  const int step = sp.parts * sp.at_once, bytes = step * dm.d * es;
  Ahead ahead;
  ahead.tok = wk.tok;
  ahead.g = wk.part;
  auto locate = [&]() {
    ahead.locate(dm, sp, wk, ln.slot, static_cast<const char *>(qkv), nullptr, nullptr, nullptr,
                 es);
  };
  locate();
  auto fetch = [&](int stage) {
    if (ln.live && ahead.left > 0) {
      copy_async<kB>(&ring[stage][0][threadIdx.x], ahead.x + ln.a * es);
      copy_async<kB>(&ring[stage][1][threadIdx.x], ahead.x + ln.b * es);
    }
    copies_commit();
    if (!ahead.next(sp, step, bytes)) locate();
  };
  int64_t pos = wk.tok < dm.rows ? __ldg(pos_idx + wk.tok) : -1;
#pragma unroll
  for (int i = 0; i < kFwdStages - 1; ++i) fetch(i);
  stage_weights<W>(ws, qw, kw, dm.w0, dm.d);
  __syncthreads();
  int stage = 0;
  for (int64_t tok = wk.tok; tok < dm.rows; tok += wk.stride) {
    const bool inside = pos >= 0 && pos < dm.slots;
    uint32_t b32, t32 = 0;
    if (inside) seq_div.divmod((uint32_t)pos, b32, t32);
    if (tok + wk.stride < dm.rows) pos = __ldg(pos_idx + tok + wk.stride);
    int g = wk.part;
#pragma unroll
    for (int kind = 0; kind < 3; ++kind) {
      const int g0 = kind == 0 ? 0 : kind == 1 ? sp.gq : sp.gq + sp.gk;
      const int g1 = kind == 0 ? sp.gq : kind == 1 ? sp.gq + sp.gk : sp.groups;
      if (g >= g1) continue;
      const int n = kind == 0 ? dm.nh : dm.nkv;
      if (kind < 2)
        make_table<V, true>(tab, cosv, sinv, (int64_t)t32 * dm.rot, ws + kind * dm.d, ln, sp);
      int left = n - (g - g0) * sp.at_once - ln.slot;
      const int64_t at = (tok * n + (n - left)) * (int64_t)dm.d;
      char *out = static_cast<char *>(kind == 0 ? q : kind == 1 ? k : v) + at * es;
      const void *l = kind == 0 ? lq : kind == 1 ? nullptr : lv;
      const char *lora = static_cast<const char *>(l) + at * elem_size<L>();
      for (; g < g1; g += sp.parts) {
        const bool live = ln.live && left > 0;
        typename Vec<L, V>::type l1, l2;
        if (kind != 1 && l != nullptr && live) {
          l1 = load_raw<L, V>(lora, ln.a);
          l2 = load_raw<L, V>(lora, ln.b);
        }
        copies_wait<kFwdStages - 2>();
        F2 x1[V / 2], x2[V / 2];
        if (live && inside) {
          Vec<T, V>::get(ring[stage][0][threadIdx.x], x1);
          Vec<T, V>::get(ring[stage][1][threadIdx.x], x2);
          if (kind != 1 && l != nullptr) {
            F2 y1[V / 2], y2[V / 2];
            Vec<L, V>::get(l1, y1);
            Vec<L, V>::get(l2, y2);
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
              x1[i] = add2(x1[i], y1[i]);
              x2[i] = add2(x2[i], y2[i]);
            }
          }
        } else {
          fill(x1, 0.f);
          fill(x2, 0.f);
        }
        fetch((stage + kFwdStages - 1) % kFwdStages);
        stage = (stage + 1) % kFwdStages;
        if (kind < 2) {
          const float ss = group_sum(square_sum(x1, x2), sp.lanes);
          const F2 r = both(rsqrtf(fmaf(ss, dm.inv_d, dm.eps)));
          if (live && inside) {
            const int next = (V / 4) * sp.lanes;
#pragma unroll
            for (int i = 0; i < V / 4; ++i) {
              const float4 *p = mine + i * sp.lanes;
              const Quad2 A = quad_at(p), B = quad_at(p + next), C = quad_at(p + 2 * next),
                          D = quad_at(p + 3 * next);
              const F2 y = fma2(x1[2 * i], A.lo, mul2(x2[2 * i], B.lo));
              const F2 z = fma2(x1[2 * i + 1], A.hi, mul2(x2[2 * i + 1], B.hi));
              x2[2 * i] = mul2(r, fma2(x2[2 * i], C.lo, mul2(x1[2 * i], D.lo)));
              x2[2 * i + 1] = mul2(r, fma2(x2[2 * i + 1], C.hi, mul2(x1[2 * i + 1], D.hi)));
              x1[2 * i] = mul2(r, y);
              x1[2 * i + 1] = mul2(r, z);
            }
          }
        }
        if (live) {
          *reinterpret_cast<Raw *>(out + ln.a * es) = Vec<T, V>::put(x1);
          *reinterpret_cast<Raw *>(out + ln.b * es) = Vec<T, V>::put(x2);
        }
        left -= step;
        out += bytes;
        lora += (int64_t)step * dm.d * elem_size<L>();
      }
    }
  }
  copies_wait<0>();
}

// Backward. A lane's weight sums of the kind at hand are in registers, those of the walk in its own
// place of shared memory. part (may be NULL): fp32 [gridDim, 2, d], this CTA's sums of dqw and dkw.
template <int T, int V, int L, int W>
__global__ void __launch_bounds__(kThreads, kBwdPerSm)
    norm_rope_bwd(const void *__restrict__ dq, const void *__restrict__ dk,
                  const void *__restrict__ dv, const void *__restrict__ qkv,
                  const void *__restrict__ lq, const void *__restrict__ qw,
                  const void *__restrict__ kw, const float *__restrict__ cosv,
                  const float *__restrict__ sinv, const int64_t *__restrict__ pos_idx,
                  void *__restrict__ dqkv, float *__restrict__ part, NormDims dm, Spread sp,
                  FastDiv seq_div) {
  pdl_wait();
  pdl_release();
  using Raw = typename Vec<T, V>::type;
  constexpr int kB = V * elem_size<T>(), es = elem_size<T>();
  extern __shared__ uint4 shared[];
  Raw(*ring)[4][kThreads] = reinterpret_cast<Raw(*)[4][kThreads]>(shared);
  F2(*sums)[V][kThreads] = reinterpret_cast<F2(*)[V][kThreads]>(ring + kBwdStages);
  float *ws = reinterpret_cast<float *>(sums + 2);
  float4 *tab = reinterpret_cast<float4 *>(ws + 2 * dm.d) + (threadIdx.x >> 5) * V * sp.lanes;
  const float4 *mine = tab + (threadIdx.x & (sp.lanes - 1));
  const Lane<V> ln(dm, sp);
  const Walk wk(dm, sp);
  const int total = dm.nh + 2 * dm.nkv;
  const int step = sp.parts * sp.at_once, bytes = step * dm.d * es;
#pragma unroll
  for (int i = 0; i < V; ++i) sums[0][i][threadIdx.x] = sums[1][i][threadIdx.x] = both(0.f);
  Ahead ahead;
  ahead.tok = wk.tok;
  ahead.g = wk.part;
  auto locate = [&]() {
    ahead.locate(dm, sp, wk, ln.slot, static_cast<const char *>(qkv),
                 static_cast<const char *>(dq), static_cast<const char *>(dk),
                 static_cast<const char *>(dv), es);
  };
  locate();
  const bool has[3] = {dq != nullptr, dk != nullptr, dv != nullptr};
  auto fetch = [&](int stage) {
    if (ln.live && ahead.left > 0) {
      if (ahead.kind == 0 ? has[0] : ahead.kind == 1 ? has[1] : has[2]) {
        copy_async<kB>(&ring[stage][0][threadIdx.x], ahead.y + ln.a * es);
        copy_async<kB>(&ring[stage][1][threadIdx.x], ahead.y + ln.b * es);
      }
      if (ahead.kind < 2) {
        copy_async<kB>(&ring[stage][2][threadIdx.x], ahead.x + ln.a * es);
        copy_async<kB>(&ring[stage][3][threadIdx.x], ahead.x + ln.b * es);
      }
    }
    copies_commit();
    if (!ahead.next(sp, step, bytes)) locate();
  };
  int64_t pos = wk.tok < dm.rows ? __ldg(pos_idx + wk.tok) : -1;
#pragma unroll
  for (int i = 0; i < kBwdStages - 1; ++i) fetch(i);
  stage_weights<W>(ws, qw, kw, dm.w0, dm.d);
  __syncthreads();
  int stage = 0;
  for (int64_t tok = wk.tok; tok < dm.rows; tok += wk.stride) {
    const bool inside = pos >= 0 && pos < dm.slots;
    uint32_t b32, t32 = 0;
    if (inside) seq_div.divmod((uint32_t)pos, b32, t32);
    make_table<V, false>(tab, cosv, sinv, (int64_t)t32 * dm.rot, nullptr, ln, sp);
    if (tok + wk.stride < dm.rows) pos = __ldg(pos_idx + tok + wk.stride);
    int g = wk.part;
#pragma unroll
    for (int kind = 0; kind < 3; ++kind) {
      const int g0 = kind == 0 ? 0 : kind == 1 ? sp.gq : sp.gq + sp.gk;
      const int g1 = kind == 0 ? sp.gq : kind == 1 ? sp.gq + sp.gk : sp.groups;
      if (g >= g1) continue;
      const int n = kind == 0 ? dm.nh : dm.nkv;
      const int first = kind == 0 ? 0 : kind == 1 ? dm.nh : dm.nh + dm.nkv;
      const float *w = ws + kind * dm.d;
      F2 a1[V / 2], a2[V / 2];
      Quad2 w1[V / 4], w2[V / 4];
      if (kind < 2) {
        fill(a1, 0.f);
        fill(a2, 0.f);
        if (ln.live) {
#pragma unroll
          for (int i = 0; i < V / 4; ++i) {
            w1[i] = quad_at(reinterpret_cast<const float4 *>(w + ln.a) + i);
            w2[i] = quad_at(reinterpret_cast<const float4 *>(w + ln.b) + i);
          }
        }
      }
      int left = n - (g - g0) * sp.at_once - ln.slot;
      char *out =
          static_cast<char *>(dqkv) + (tok * total + first + (n - left)) * (int64_t)dm.d * es;
      const char *lora =
          static_cast<const char *>(lq) + (tok * n + (n - left)) * (int64_t)dm.d * elem_size<L>();
      for (; g < g1; g += sp.parts) {
        const bool live = ln.live && left > 0;
        typename Vec<L, V>::type l1, l2;
        if (kind == 0 && lq != nullptr && live) {
          l1 = load_raw<L, V>(lora, ln.a);
          l2 = load_raw<L, V>(lora, ln.b);
        }
        copies_wait<kBwdStages - 2>();
        F2 f1[V / 2], f2[V / 2];
        if (live && inside && has[kind]) {
          Vec<T, V>::get(ring[stage][0][threadIdx.x], f1);
          Vec<T, V>::get(ring[stage][1][threadIdx.x], f2);
        } else {
          fill(f1, 0.f);
          fill(f2, 0.f);
        }
        if (kind < 2) {
          F2 y1[V / 2], y2[V / 2], dot = both(0.f);
          float ss = 0.f, gx = 0.f;
          if (live && inside) {
            Vec<T, V>::get(ring[stage][2][threadIdx.x], y1);
            Vec<T, V>::get(ring[stage][3][threadIdx.x], y2);
            if (kind == 0 && lq != nullptr) {
              F2 z1[V / 2], z2[V / 2];
              Vec<L, V>::get(l1, z1);
              Vec<L, V>::get(l2, z2);
#pragma unroll
              for (int i = 0; i < V / 2; ++i) {
                y1[i] = add2(y1[i], z1[i]);
                y2[i] = add2(y2[i], z2[i]);
              }
            }
            ss = square_sum(y1, y2);
            const int next = (V / 4) * sp.lanes;
#pragma unroll
            for (int i = 0; i < V / 4; ++i) {
              const float4 *p = mine + i * sp.lanes;
              const Quad2 c1 = quad_at(p), s1 = quad_at(p + next), c2 = quad_at(p + 2 * next),
                          s2 = quad_at(p + 3 * next);
              const F2 d1 = fma2(f1[2 * i], c1.lo, mul2(f2[2 * i], s2.lo));
              const F2 e1 = fma2(f1[2 * i + 1], c1.hi, mul2(f2[2 * i + 1], s2.hi));
              f2[2 * i] = fma2(f2[2 * i], c2.lo, mul2(f1[2 * i], s1.lo));
              f2[2 * i + 1] = fma2(f2[2 * i + 1], c2.hi, mul2(f1[2 * i + 1], s1.hi));
              f1[2 * i] = d1;
              f1[2 * i + 1] = e1;
              dot = fma2(mul2(d1, y1[2 * i]), w1[i].lo, dot);
              dot = fma2(mul2(e1, y1[2 * i + 1]), w1[i].hi, dot);
              dot = fma2(mul2(f2[2 * i], y2[2 * i]), w2[i].lo, dot);
              dot = fma2(mul2(f2[2 * i + 1], y2[2 * i + 1]), w2[i].hi, dot);
            }
            const float2 p = parts(dot);
            gx = p.x + p.y;
          }
          ss = group_sum(ss, sp.lanes);
          gx = group_sum(gx, sp.lanes);
          const float r = rsqrtf(fmaf(ss, dm.inv_d, dm.eps));
          if (live && inside) {
            // r gx first: r^3 alone may be past fp32
            const F2 rr = both(r), rk = both(-(r * gx * dm.inv_d) * r * r);
#pragma unroll
            for (int i = 0; i < V / 4; ++i) {
#pragma unroll
              for (int j = 2 * i; j < 2 * i + 2; ++j) {
                f1[j] = mul2(f1[j], rr);
                f2[j] = mul2(f2[j], rr);
                a1[j] = fma2(f1[j], y1[j], a1[j]);
                a2[j] = fma2(f2[j], y2[j], a2[j]);
                f1[j] = fma2(f1[j], j == 2 * i ? w1[i].lo : w1[i].hi, mul2(y1[j], rk));
                f2[j] = fma2(f2[j], j == 2 * i ? w2[i].lo : w2[i].hi, mul2(y2[j], rk));
              }
            }
          }
        }
        fetch((stage + kBwdStages - 1) % kBwdStages);
        stage = (stage + 1) % kBwdStages;
        if (live) {
          *reinterpret_cast<Raw *>(out + ln.a * es) = Vec<T, V>::put(f1);
          *reinterpret_cast<Raw *>(out + ln.b * es) = Vec<T, V>::put(f2);
        }
        left -= step;
        out += bytes;
        lora += (int64_t)step * dm.d * elem_size<L>();
      }
      if (kind < 2 && ln.live && part != nullptr) {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
          sums[kind][i][threadIdx.x] = add2(sums[kind][i][threadIdx.x], a1[i]);
          sums[kind][V / 2 + i][threadIdx.x] = add2(sums[kind][V / 2 + i][threadIdx.x], a2[i]);
        }
      }
    }
  }
  copies_wait<0>();
  if (part == nullptr) return;
  // the lanes' sums, added in order of the warps and their head rows
  __syncthreads();
  const int pairs = dm.rot / (2 * V), h = dm.rot / 2;
  for (int i = threadIdx.x; i < 2 * dm.d; i += kThreads) {
    const int dim = i < dm.d ? i : i - dm.d, rest = dim - dm.rot, kind = i < dm.d ? 0 : 1;
    const int at = dim < dm.rot ? (dim % h) / V : pairs + rest / (2 * V);
    const int e = dim < dm.rot ? (dim >= h ? V : 0) + dim % V : rest % (2 * V);
    float s = 0.f;
    for (int j = 0; j < kThreads / sp.lanes; ++j)
      s += reinterpret_cast<const float *>(&sums[kind][e / 2][j * sp.lanes + at])[e % 2];
    part[(int64_t)blockIdx.x * 2 * dm.d + i] = s;
  }
}

// Any even head size and alignment: a warp per head row, a lane per pair of dims at a time (4096
// tokens of 12 + 2 + 2 heads of 100, bf16: 41 us, issue 65 %, against 4 for its bytes).
template <int T>
__device__ __forceinline__ float load_x(const void *qkv, const void *l, int l_type, int64_t at,
                                        int64_t li, int i) {
  float x = load1<T>(qkv, at + i);
  if (l != nullptr)
    x += l_type == TB_FP16   ? load1<TB_FP16>(l, li + i)
         : l_type == TB_BF16 ? load1<TB_BF16>(l, li + i)
                             : load1<TB_FP32>(l, li + i);
  return x;
}

__device__ __forceinline__ float weight_at(const void *w, int w_type, float w0, int i) {
  if (w == nullptr) return 1.f;
  return w0 + (w_type == TB_FP16   ? load1<TB_FP16>(w, i)
               : w_type == TB_BF16 ? load1<TB_BF16>(w, i)
                                   : load1<TB_FP32>(w, i));
}

// Pair j of a head: dims (j, j + rot/2) below rot/2, else two neighbours of the rest.
__device__ __forceinline__ void pair_of(int j, int rot, int &a, int &b) {
  const int h = rot / 2;
  a = j < h ? j : rot + 2 * (j - h);
  b = j < h ? j + h : a + 1;
}

template <int T>
__global__ void __launch_bounds__(256)
    norm_rope_fwd_any(const void *qkv, const void *lq, const void *lv, int l_type, const void *qw,
                      const void *kw, int w_type, const float *cosv, const float *sinv,
                      const int64_t *pos_idx, void *q, void *k, void *v, NormDims dm, int64_t seq) {
  pdl_wait();
  pdl_release();
  const int lane = threadIdx.x & 31, total = dm.nh + 2 * dm.nkv;
  const int64_t n = dm.rows * total;
  for (int64_t u = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); u < n;
       u += (int64_t)gridDim.x * 8) {
    const int64_t tok = u / total;
    const int hr = (int)(u - tok * total);
    const int64_t pos = pos_idx[tok];
    const bool inside = pos >= 0 && pos < dm.slots;
    const int64_t t = inside ? pos % seq : 0;
    const int64_t at = tok * dm.ld + (int64_t)hr * dm.d;
    const bool normed = hr < dm.nh + dm.nkv;
    const void *l = hr < dm.nh ? lq : normed ? nullptr : lv;
    int64_t out;
    void *dst = pick(q, k, v, dm, tok, hr, out);
    float ss = 0.f;
    if (inside && normed)
      for (int i = lane; i < dm.d; i += 32) {
        const float x = load_x<T>(qkv, l, l_type, at, out, i);
        ss += x * x;
      }
    const float r = rsqrtf(warp_sum(ss) * dm.inv_d + dm.eps);
    const void *w = hr < dm.nh ? qw : kw;
    for (int j = lane; j < dm.d / 2; j += 32) {
      int a, b;
      pair_of(j, dm.rot, a, b);
      float x1 = 0.f, x2 = 0.f;
      if (inside) {
        x1 = load_x<T>(qkv, l, l_type, at, out, a);
        x2 = load_x<T>(qkv, l, l_type, at, out, b);
        if (normed) {
          const float n1 = x1 * r * weight_at(w, w_type, dm.w0, a);
          const float n2 = x2 * r * weight_at(w, w_type, dm.w0, b);
          const bool turn = j < dm.rot / 2;
          x1 = turn ? n1 * cosv[t * dm.rot + a] - n2 * sinv[t * dm.rot + a] : n1;
          x2 = turn ? n2 * cosv[t * dm.rot + b] + n1 * sinv[t * dm.rot + b] : n2;
        }
      }
      store1<T>(dst, out + a, x1);
      store1<T>(dst, out + b, x2);
    }
  }
}

// A CTA of one warp per token range; its dw sums live in shared memory, each element touched by
// one lane only. The same tokens: 174 us (6 for the bytes), waiting for each load with 8 warps an
// SM (issue 16 %, DRAM 2 %): for sizes and alignments that a training step does not have.
template <int T>
__global__ void __launch_bounds__(32)
    norm_rope_bwd_any(const void *dq, const void *dk, const void *dv, const void *qkv,
                      const void *lq, int l_type, const void *qw, const void *kw, int w_type,
                      const float *cosv, const float *sinv, const int64_t *pos_idx, void *dqkv,
                      float *part, NormDims dm, int64_t seq) {
  pdl_wait();
  pdl_release();
  extern __shared__ float sums[];  // [2 d]
  const int lane = threadIdx.x, total = dm.nh + 2 * dm.nkv;
  const int64_t width = (int64_t)total * dm.d;
  for (int j = lane; j < dm.d / 2; j += 32) {
    int a, b;
    pair_of(j, dm.rot, a, b);
    sums[a] = sums[b] = sums[dm.d + a] = sums[dm.d + b] = 0.f;
  }
  for (int64_t tok = blockIdx.x; tok < dm.rows; tok += gridDim.x) {
    const int64_t pos = pos_idx[tok];
    const bool inside = pos >= 0 && pos < dm.slots;
    const int64_t t = inside ? pos % seq : 0;
    for (int hr = 0; hr < total; ++hr) {
      const int64_t at = tok * dm.ld + (int64_t)hr * dm.d;
      const bool normed = hr < dm.nh + dm.nkv;
      const void *l = hr < dm.nh ? lq : nullptr;
      const void *w = hr < dm.nh ? qw : kw;
      int64_t in;
      const void *src = pick(dq, dk, dv, dm, tok, hr, in);
      if (!inside) src = nullptr;
      float ss = 0.f, gx = 0.f;
      for (int phase = normed && inside ? 0 : 1; phase < 2; ++phase) {
        float r = 0.f, k2 = 0.f;
        if (phase == 1) {
          r = rsqrtf(warp_sum(ss) * dm.inv_d + dm.eps);
          k2 = r * r * (warp_sum(gx) * dm.inv_d);
        }
        for (int j = lane; j < dm.d / 2; j += 32) {
          int a, b;
          pair_of(j, dm.rot, a, b);
          float g1 = src ? load1<T>(src, in + a) : 0.f, g2 = src ? load1<T>(src, in + b) : 0.f;
          float o1 = g1, o2 = g2;
          if (normed && inside) {
            if (j < dm.rot / 2) {
              const float *c = cosv + t * dm.rot, *s = sinv + t * dm.rot;
              o1 = g1 * c[a] + g2 * s[b];
              o2 = g2 * c[b] - g1 * s[a];
            }
            const float x1 = load_x<T>(qkv, l, l_type, at, in, a);
            const float x2 = load_x<T>(qkv, l, l_type, at, in, b);
            const float w1 = weight_at(w, w_type, dm.w0, a), w2 = weight_at(w, w_type, dm.w0, b);
            if (phase == 0) {
              ss += x1 * x1 + x2 * x2;
              gx += o1 * w1 * x1 + o2 * w2 * x2;
              continue;
            }
            float *acc = sums + (hr < dm.nh ? 0 : dm.d);
            acc[a] += o1 * x1 * r;
            acc[b] += o2 * x2 * r;
            o1 = r * (o1 * w1 - x1 * k2);
            o2 = r * (o2 * w2 - x2 * k2);
          }
          const int64_t to = tok * width + (int64_t)hr * dm.d;
          store1<T>(dqkv, to + a, o1);
          store1<T>(dqkv, to + b, o2);
        }
      }
    }
  }
  if (part == nullptr) return;
  for (int j = lane; j < dm.d / 2; j += 32) {
    int a, b;
    pair_of(j, dm.rot, a, b);
    float *out = part + (int64_t)blockIdx.x * 2 * dm.d;
    out[a] = sums[a];
    out[b] = sums[b];
    out[dm.d + a] = sums[dm.d + a];
    out[dm.d + b] = sums[dm.d + b];
  }
}

// dqw / dkw from the CTAs' sums: 32 columns a block, 32 groups of CTAs each in order, then the
// groups in order.
__global__ void __launch_bounds__(1024)
    norm_rope_dw(const float *__restrict__ part, int ctas, int d, void *dqw, void *dkw,
                 int w_type) {
  pdl_wait();
  pdl_release();
  __shared__ float sh[32][33];
  const int lane = threadIdx.x & 31, grp = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
  const int per = (ctas + 31) / 32;
  float s = 0.f;
  if (col < 2 * d) {
#pragma unroll 8
    for (int c = grp * per; c < (grp + 1) * per; ++c)
      s += c < ctas ? part[(int64_t)c * 2 * d + col] : 0.f;
  }
  sh[grp][lane] = s;
  __syncthreads();
  if (grp != 0 || col >= 2 * d) return;
  for (int g = 1; g < 32; ++g) s += sh[g][lane];
  void *dst = col < d ? dqw : dkw;
  if (dst == nullptr) return;
  TB_WITH_TYPE(w_type, T, store1<T>(dst, col < d ? col : col - d, s));
}

int pow2_at_least(int n) {
  int p = 1;
  while (p < n) p *= 2;
  return p;
}

// Dims of a chunk on the vector path (0: not taken): 16 bytes, or 8 where the head size or rot of a
// 16-bit type ask for it.
int chunk_of(const NormDims &dm, int type) {
  if (type != TB_FP32 && dm.d % 16 == 0 && dm.rot % 16 == 0 && dm.d <= 512) return 8;
  return dm.d % 8 == 0 && dm.rot % 8 == 0 && dm.d <= 256 ? 4 : 0;
}

// CTAs of a walk: `per_sm` resident ones at most, at least a warp for each group of head rows.
int walk_ctas(const NormDims &dm, int chunk, int per_sm) {
  const int64_t at_once = 32 / pow2_at_least(dm.d / (2 * chunk));
  const int64_t groups = (dm.nh + at_once - 1) / at_once + 2 * ((dm.nkv + at_once - 1) / at_once);
  int64_t cap = (int64_t)sm_count() * per_sm;
  if (cap < (groups + kWarps - 1) / kWarps) cap = (groups + kWarps - 1) / kWarps;
  const int64_t want = (dm.rows * groups + kWarps - 1) / kWarps;
  return (int)(want < cap ? want : cap);
}

// A token's groups over as many warps as `ctas` CTAs have for them.
Spread spread_of(const NormDims &dm, int chunk, int ctas) {
  Spread sp;
  sp.lanes = pow2_at_least(dm.d / (2 * chunk));
  sp.at_once = 32 / sp.lanes;
  sp.gq = (dm.nh + sp.at_once - 1) / sp.at_once;
  sp.gk = (dm.nkv + sp.at_once - 1) / sp.at_once;
  sp.groups = sp.gq + 2 * sp.gk;
  const int64_t parts = dm.rows > 0 ? (int64_t)ctas * kWarps / dm.rows : 1;
  sp.parts = (int)(parts < 1 ? 1 : parts < sp.groups ? parts : sp.groups);
  return sp;
}

// CTAs of the backward for any size, one warp each.
int any_ctas(int64_t rows) {
  const int64_t cap = (int64_t)sm_count() * 8;
  return (int)(rows < cap ? rows : cap);
}

int check(const char *what, const NormDims &dm, int64_t batch, int64_t seq, int type, int l_type,
          int w_type) {
  if (dm.rows < 0 || batch < 0 || seq <= 0 || dm.nh <= 0 || dm.nkv < 0 || dm.d <= 0 || dm.d % 2 ||
      dm.rot < 0 || dm.rot % 2 || dm.rot > dm.d)
    return set_error(TB_EINVAL,
                     "%s: bad dims rows=%lld batch=%lld seq=%lld nh=%d nkv=%d d=%d rot=%d", what,
                     (long long)dm.rows, (long long)batch, (long long)seq, dm.nh, dm.nkv,
                     dm.d, dm.rot);
  if (dm.d > 4096 || dm.nh > 65536 || dm.nkv > 65536)
    return set_error(TB_EINVAL, "%s: head_dim %d (at most 4096), heads %d / %d (at most 65536)",
                     what, dm.d, dm.nh, dm.nkv);
  if (dm.rows > 0x7fffffffLL || batch > 0x7fffffffLL || seq > 0x7fffffffLL ||
      batch * seq > 0x7fffffffLL)
    return set_error(TB_EINVAL, "%s: too many rows or slots", what);
  if (dm.ld < (int64_t)(dm.nh + 2 * dm.nkv) * dm.d)
    return set_error(TB_EINVAL, "%s: row stride %lld below the row", what, (long long)dm.ld);
  if (!elem_type_ok(type) || !elem_type_ok(l_type) || !elem_type_ok(w_type))
    return set_error(TB_EINVAL, "%s: types %d %d %d", what, type, l_type, w_type);
  return TB_OK;
}

// Shared memory beyond 48 KB has to be asked for, on every device.
template <typename Kernel>
int allow_smem(const char *what, Kernel kernel, size_t bytes) {
  if (bytes <= 48 * 1024 ||
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) ==
          cudaSuccess)
    return TB_OK;
  (void)cudaGetLastError();
  return set_error(TB_ELAUNCH, "%s: %d bytes of shared memory", what, (int)bytes);
}

// Runs RUN(T, V, L, W) for the element type, the chunk and the LoRA rows' and weights' types.
#define TB_WITH_CHUNK(RUN)                                     \
  do {                                                         \
    if (type == TB_FP32) {                                     \
      RUN(TB_FP32, 4, TB_FP32, TB_FP32);                       \
    } else if (type == TB_FP16) {                              \
      TB_WITH_PARTS(RUN, TB_FP16);                             \
    } else {                                                   \
      TB_WITH_PARTS(RUN, TB_BF16);                             \
    }                                                          \
  } while (0)
#define TB_WITH_PARTS(RUN, T)                                  \
  do {                                                         \
    if (chunk == 8) {                                          \
      if (l_own && w_own) RUN(T, 8, T, T);                     \
      else if (l_own) RUN(T, 8, T, TB_FP32);                   \
      else if (w_own) RUN(T, 8, TB_FP32, T);                   \
      else RUN(T, 8, TB_FP32, TB_FP32);                        \
    } else {                                                   \
      if (l_own && w_own) RUN(T, 4, T, T);                     \
      else if (l_own) RUN(T, 4, T, TB_FP32);                   \
      else if (w_own) RUN(T, 4, TB_FP32, T);                   \
      else RUN(T, 4, TB_FP32, TB_FP32);                        \
    }                                                          \
  } while (0)

bool all_aligned(std::initializer_list<const void *> ps, uintptr_t a) {
  for (const void *p : ps)
    if (!aligned(p, a)) return false;
  return true;
}

}  // namespace
}  // namespace tb

using namespace tb;

extern "C" int tb_norm_rope_fwd(const void *qkv, int32_t type, int64_t ld, const void *lora_q,
                                const void *lora_v, int32_t lora_type, const void *q_weight,
                                const void *k_weight, int32_t weight_type, float weight_offset,
                                float eps, const float *cos, const float *sin, int32_t rot,
                                const int64_t *pos_idx, void *q, void *k, void *v, int64_t rows,
                                int64_t batch, int64_t seq, int32_t n_heads, int32_t n_kv,
                                int32_t head_dim, void *stream) {
  NormDims dm{rows, ld, batch * seq, n_heads, n_kv, head_dim, rot, eps, weight_offset,
              1.f / (float)(head_dim > 0 ? head_dim : 1)};
  int rc = check("norm_rope_fwd", dm, batch, seq, type, lora_type, weight_type);
  if (rc != TB_OK) return rc;
  if (rows == 0) return TB_OK;
  if (!qkv || !pos_idx || !q || (n_kv > 0 && (!k || !v)) || (rot > 0 && (!cos || !sin)))
    return set_error(TB_EINVAL, "norm_rope_fwd: qkv, pos_idx, q, k, v and the tables are required");
  const int es = elem_size_of(type), ls = elem_size_of(lora_type), ws = elem_size_of(weight_type);
  if (!all_aligned({qkv, q, k, v}, es) || !all_aligned({lora_q, lora_v}, ls) ||
      !all_aligned({q_weight, k_weight}, ws) || !all_aligned({cos, sin}, 4) || !aligned(pos_idx, 8))
    return set_error(TB_EALIGN, "norm_rope_fwd: a buffer is not aligned to its element");
  const int chunk = chunk_of(dm, type);
  const bool vec = chunk > 0 && ld % chunk == 0 && all_aligned({qkv, q, k, v}, chunk * es) &&
                   all_aligned({lora_q, lora_v, q_weight, k_weight, cos, sin}, 16);
  cudaStream_t st = as_stream(stream);
  // the LoRA rows and the weights in qkv's type or fp32 on the vector path
  const bool l_own = lora_type == type || (!lora_q && !lora_v);
  const bool w_own = weight_type == type || (!q_weight && !k_weight);
  if (vec && (l_own || lora_type == TB_FP32) && (w_own || weight_type == TB_FP32)) {
    const FastDiv sd((uint32_t)seq);
    const int ctas = walk_ctas(dm, chunk, kFwdPerSm);
    const Spread sp = spread_of(dm, chunk, ctas);
#define TB_FWD(T, V, L, W)                                                                       \
  do {                                                                                           \
    const size_t kSmem = (size_t)kThreads * kFwdStages * 2 * V * elem_size<T>() +                \
                         2 * head_dim * 4 + (size_t)kWarps * V * sp.lanes * 16;                  \
    rc = allow_smem("norm_rope_fwd", norm_rope_fwd<T, V, L, W>, kSmem);                          \
    if (rc != TB_OK) return rc;                                                                  \
    return launch("norm_rope_fwd", norm_rope_fwd<T, V, L, W>, dim3((unsigned)ctas), kThreads,    \
                  kSmem, st, qkv, lora_q, lora_v, q_weight, k_weight, cos, sin, pos_idx, q, k,   \
                  v, dm, sp, sd);                                                                \
  } while (0)
    TB_WITH_CHUNK(TB_FWD);
#undef TB_FWD
  }
  int64_t blocks = (rows * (n_heads + 2 * (int64_t)n_kv) + 7) / 8;
  const int64_t cap = (int64_t)sm_count() * 16;
  if (blocks > cap) blocks = cap;
  TB_WITH_TYPE(type, T,
               return launch("norm_rope_fwd", norm_rope_fwd_any<T>, dim3((unsigned)blocks), 256, 0,
                             st, qkv, lora_q, lora_v, lora_type, q_weight, k_weight, weight_type,
                             cos, sin, pos_idx, q, k, v, dm, seq));
}

extern "C" int64_t tb_norm_rope_bwd_workspace(int64_t rows, int32_t n_heads, int32_t n_kv,
                                              int32_t head_dim) {
  if (rows <= 0 || n_heads <= 0 || n_kv < 0 || head_dim <= 0) return 0;
  const NormDims dm{rows, 0, 0, n_heads, n_kv, head_dim, 0, 0.f, 0.f, 0.f};
  // the most of the paths that the type, rot and alignment choose from
  int most = any_ctas(rows);
  for (int chunk = 4; chunk <= 8; chunk += 4) {
    if (head_dim % (2 * chunk) || head_dim > 64 * chunk) continue;
    const int ctas = walk_ctas(dm, chunk, kBwdPerSm);
    if (ctas > most) most = ctas;
  }
  return (int64_t)most * 2 * head_dim * 4;
}

extern "C" int tb_norm_rope_bwd(const void *dq, const void *dk, const void *dv, const void *qkv,
                                int32_t type, int64_t ld, const void *lora_q, int32_t lora_type,
                                const void *q_weight, const void *k_weight, int32_t weight_type,
                                float weight_offset, float eps, const float *cos, const float *sin,
                                int32_t rot, const int64_t *pos_idx, void *dqkv, void *dq_weight,
                                void *dk_weight, void *workspace, int64_t workspace_bytes,
                                int64_t rows, int64_t batch, int64_t seq, int32_t n_heads,
                                int32_t n_kv, int32_t head_dim, void *stream) {
  NormDims dm{rows, ld, batch * seq, n_heads, n_kv, head_dim, rot, eps, weight_offset,
              1.f / (float)(head_dim > 0 ? head_dim : 1)};
  int rc = check("norm_rope_bwd", dm, batch, seq, type, lora_type, weight_type);
  if (rc != TB_OK) return rc;
  const bool want_dw = dq_weight || dk_weight;
  if (rows == 0 && !want_dw) return TB_OK;
  if (rows > 0 && (!qkv || !pos_idx || !dqkv || (rot > 0 && (!cos || !sin))))
    return set_error(TB_EINVAL, "norm_rope_bwd: qkv, pos_idx, dqkv and the tables are required");
  const int es = elem_size_of(type), ls = elem_size_of(lora_type), ws = elem_size_of(weight_type);
  if (!all_aligned({qkv, dq, dk, dv, dqkv}, es) || !aligned(lora_q, ls) ||
      !all_aligned({q_weight, k_weight, dq_weight, dk_weight}, ws) ||
      !all_aligned({cos, sin, workspace}, 4) || !aligned(pos_idx, 8))
    return set_error(TB_EALIGN, "norm_rope_bwd: a buffer is not aligned to its element");
  if (want_dw && rows > 0 &&
      (!workspace || workspace_bytes < tb_norm_rope_bwd_workspace(rows, n_heads, n_kv, head_dim)))
    return set_error(TB_EINVAL, "norm_rope_bwd: workspace of %lld bytes, %lld needed",
                     (long long)workspace_bytes,
                     (long long)tb_norm_rope_bwd_workspace(rows, n_heads, n_kv, head_dim));
  float *part = want_dw ? static_cast<float *>(workspace) : nullptr;
  cudaStream_t st = as_stream(stream);
  int ctas = 0;
  if (rows > 0) {
    const int chunk = chunk_of(dm, type);
    const bool vec = chunk > 0 && ld % chunk == 0 &&
                     all_aligned({qkv, dq, dk, dv, dqkv}, chunk * es) &&
                     all_aligned({lora_q, q_weight, k_weight, cos, sin}, 16);
    const bool l_own = lora_type == type || !lora_q;
    const bool w_own = weight_type == type || (!q_weight && !k_weight);
    if (vec && (l_own || lora_type == TB_FP32) && (w_own || weight_type == TB_FP32)) {
      const FastDiv sd((uint32_t)seq);
      ctas = walk_ctas(dm, chunk, kBwdPerSm);
      const Spread sp = spread_of(dm, chunk, ctas);
#define TB_BWD(T, V, L, W)                                                                       \
  do {                                                                                           \
    const size_t kSmem = (size_t)kThreads * (kBwdStages * 4 * V * elem_size<T>() + 2 * V * 8) +  \
                         2 * head_dim * 4 + (size_t)kWarps * V * sp.lanes * 16;                  \
    rc = allow_smem("norm_rope_bwd", norm_rope_bwd<T, V, L, W>, kSmem);                          \
    if (rc != TB_OK) return rc;                                                                  \
    rc = launch("norm_rope_bwd", norm_rope_bwd<T, V, L, W>, dim3((unsigned)ctas), kThreads,      \
                kSmem, st, dq, dk, dv, qkv, lora_q, q_weight, k_weight, cos, sin, pos_idx, dqkv, \
                part, dm, sp, sd);                                                               \
  } while (0)
      TB_WITH_CHUNK(TB_BWD);
#undef TB_BWD
    } else {
      ctas = any_ctas(rows);
      TB_WITH_TYPE(type, T,
                   rc = launch("norm_rope_bwd", norm_rope_bwd_any<T>, dim3((unsigned)ctas), 32,
                               (size_t)2 * head_dim * 4, st, dq, dk, dv, qkv, lora_q, lora_type,
                               q_weight, k_weight, weight_type, cos, sin, pos_idx, dqkv, part, dm,
                               seq));
    }
    if (rc != TB_OK) return rc;
  }
  if (!want_dw) return TB_OK;
  return launch("norm_rope_dw", norm_rope_dw, dim3((unsigned)((2 * head_dim + 31) / 32)), 1024, 0,
                st, part, ctas, head_dim, dq_weight, dk_weight, weight_type);
}
