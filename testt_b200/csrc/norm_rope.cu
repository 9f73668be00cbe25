// Per-head RMS norms of queries and keys with the rotation (and the LoRA add) in the same pass,
// token-major, forward and backward, for sm_100a. For each token and each q / k head, in fp32:
//   x = qkv + lora     r = rsqrt(mean(x^2) + eps)     n = x r (w0 + w)
//   y_i = n_i cos_i - n_{i+h} sin_i,  y_{i+h} = n_{i+h} cos_{i+h} + n_i sin_{i+h},  h = rot / 2
// dims past rot are not turned; v = qkv + lora. Rounded once, on the store. Backward:
//   dn = the transposed rotation of dy     g = dn (w0 + w)     dx = r (g - x r^2 mean(g x))
//   dw = sum over tokens and heads of dn x r
// x is read again and both means come out of one set of shuffles, so the forward stores nothing
// for the backward. dw: each CTA walks tokens blockIdx, + gridDim, ... and keeps its sums in
// registers; a second kernel adds the CTAs' sums in order, so results do not depend on timing.
//
// Beside tb_rope_tokens_* (solution/rope.py:24-176), which has no norm; positions and tables as
// there. The reference's model has no head norms.
#include <initializer_list>

#include "dtypes.cuh"

namespace tb {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr uint32_t kAll = 0xffffffffu;

struct NormDims {
  int64_t rows, ld, slots;  // tokens, elements between qkv rows, batch * seq
  int nh, nkv, d, rot;
  float eps, w0, inv_d;
};

// Four neighbouring values as loaded: 8 bytes of a 16-bit type, 16 of fp32.
template <int T>
struct Quad {
  using type = uint2;
  static __device__ __forceinline__ void get(const type &v, float (&f)[4]) {
    const float2 a = Elem<T>::get2(v.x), b = Elem<T>::get2(v.y);
    f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
  }
  static __device__ __forceinline__ type put(const float (&f)[4]) {
    return make_uint2(Elem<T>::put2(f[0], f[1]), Elem<T>::put2(f[2], f[3]));
  }
  static __device__ __forceinline__ type zero() { return make_uint2(0, 0); }
};

template <>
struct Quad<TB_FP32> {
  using type = float4;
  static __device__ __forceinline__ void get(const type &v, float (&f)[4]) {
    f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
  }
  static __device__ __forceinline__ type put(const float (&f)[4]) {
    return make_float4(f[0], f[1], f[2], f[3]);
  }
  static __device__ __forceinline__ type zero() { return make_float4(0.f, 0.f, 0.f, 0.f); }
};

template <int T>
__device__ __forceinline__ typename Quad<T>::type load4(const void *p, int64_t i) {
  return __ldg(reinterpret_cast<const typename Quad<T>::type *>(
      static_cast<const typename Elem<T>::type *>(p) + i));
}

template <int T>
__device__ __forceinline__ void store4(void *p, int64_t i, const float (&f)[4]) {
  *reinterpret_cast<typename Quad<T>::type *>(static_cast<typename Elem<T>::type *>(p) + i) =
      Quad<T>::put(f);
}

// Sum over groups of `lanes` (a power of two) neighbouring lanes; every lane gets the total.
__device__ __forceinline__ float group_sum(float v, int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}

// The two quads of a lane: lanes below rot / 8 hold a rotation's pair (four dims of each half),
// the others two neighbouring quads of the rest.
struct Chunks {
  int a, b;
  bool live, turn;
};

__device__ __forceinline__ Chunks chunks_of(int lane, int d, int rot) {
  const int pairs = rot / 8;
  Chunks c;
  c.turn = lane < pairs;
  c.a = c.turn ? lane * 4 : rot + (lane - pairs) * 8;
  c.b = c.turn ? rot / 2 + lane * 4 : c.a + 4;
  c.live = lane < d / 8;
  return c;
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

template <int T>
__device__ __forceinline__ void load_weight(const void *w, float w0, int i, float (&f)[4]) {
  if (w == nullptr) {
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = 1.f;
  } else {
    Quad<T>::get(load4<T>(w, i), f);
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] += w0;
  }
}

template <int L>
__device__ __forceinline__ void add4(const void *p, int64_t i, float (&f)[4]) {
  float a[4];
  Quad<L>::get(load4<L>(p, i), a);
#pragma unroll
  for (int e = 0; e < 4; ++e) f[e] += a[e];
}

// The rotation's factors of a token at a lane's quads.
struct Turn {
  float c1[4], c2[4], s1[4], s2[4];
  __device__ __forceinline__ void load(const float *cosv, const float *sinv, int64_t row, int rot,
                                       const Chunks &ch) {
    Quad<TB_FP32>::get(load4<TB_FP32>(cosv, row * rot + ch.a), c1);
    Quad<TB_FP32>::get(load4<TB_FP32>(cosv, row * rot + ch.b), c2);
    Quad<TB_FP32>::get(load4<TB_FP32>(sinv, row * rot + ch.a), s1);
    Quad<TB_FP32>::get(load4<TB_FP32>(sinv, row * rot + ch.b), s2);
  }
};

// `lanes` lanes per head row, so 32 / lanes head rows at a time to a warp. A warp takes a token
// and every `parts`-th such group of its head rows, two groups in flight; the rotation's factors
// are loaded once for them. W: the weights' type, L: the LoRA rows'.
template <int T, int L, int W>
__global__ void __launch_bounds__(kThreads, 4)
    norm_rope_fwd(const void *__restrict__ qkv, const void *__restrict__ lq,
                  const void *__restrict__ lv, const void *__restrict__ qw,
                  const void *__restrict__ kw, const float *__restrict__ cosv,
                  const float *__restrict__ sinv, const int64_t *__restrict__ pos_idx, void *q,
                  void *k, void *v, NormDims dm, FastDiv seq_div, FastDiv parts, int lanes) {
  pdl_wait();
  pdl_release();
  constexpr int kGroups = 2;
  const uint32_t unit = blockIdx.x * kWarps + (threadIdx.x >> 5);
  uint32_t tok32, part;
  parts.divmod(unit, tok32, part);
  const int64_t tok = tok32;
  if (tok >= dm.rows) return;
  const int lane = threadIdx.x & (lanes - 1), slot = (threadIdx.x & 31) / lanes;
  const int rows_at_once = 32 / lanes, total = dm.nh + 2 * dm.nkv;
  const Chunks ch = chunks_of(lane, dm.d, dm.rot);
  const int64_t pos = __ldg(pos_idx + tok);
  const bool inside = pos >= 0 && pos < dm.slots;
  Turn t;
  bool turned = false;
  for (int hr0 = part * rows_at_once; hr0 < total; hr0 += kGroups * (int)parts.d * rows_at_once) {
    float x1[kGroups][4], x2[kGroups][4], r[kGroups];
    typename Quad<T>::type r1[kGroups], r2[kGroups];
    int hr[kGroups];
#pragma unroll
    for (int j = 0; j < kGroups; ++j) {
      hr[j] = hr0 + j * (int)parts.d * rows_at_once + slot;
      r1[j] = r2[j] = Quad<T>::zero();
      if (ch.live && hr[j] < total && inside) {
        const int64_t at = tok * dm.ld + (int64_t)hr[j] * dm.d;
        r1[j] = load4<T>(qkv, at + ch.a);
        r2[j] = load4<T>(qkv, at + ch.b);
      }
    }
    if (!turned && ch.live && ch.turn && inside) {
      uint32_t b32, t32;
      seq_div.divmod((uint32_t)pos, b32, t32);
      t.load(cosv, sinv, t32, dm.rot, ch);
      turned = true;
    }
#pragma unroll
    for (int j = 0; j < kGroups; ++j) {
      Quad<T>::get(r1[j], x1[j]);
      Quad<T>::get(r2[j], x2[j]);
      const bool isq = hr[j] < dm.nh, isv = hr[j] >= dm.nh + dm.nkv && hr[j] < total;
      const void *l = isq ? lq : isv ? lv : nullptr;
      if (l != nullptr && ch.live && inside) {
        const int64_t li = isq ? (tok * dm.nh + hr[j]) * (int64_t)dm.d
                               : (tok * dm.nkv + hr[j] - dm.nh - dm.nkv) * (int64_t)dm.d;
        add4<L>(l, li + ch.a, x1[j]);
        add4<L>(l, li + ch.b, x2[j]);
      }
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) ss += x1[j][e] * x1[j][e] + x2[j][e] * x2[j][e];
      r[j] = rsqrtf(group_sum(ss, lanes) * dm.inv_d + dm.eps);
    }
#pragma unroll
    for (int j = 0; j < kGroups; ++j) {
      if (!ch.live || hr[j] >= total) continue;
      if (hr[j] < dm.nh + dm.nkv && inside) {
        const void *w = hr[j] < dm.nh ? qw : kw;
        float w1[4], w2[4];
        load_weight<W>(w, dm.w0, ch.a, w1);
        load_weight<W>(w, dm.w0, ch.b, w2);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float n1 = x1[j][e] * r[j] * w1[e], n2 = x2[j][e] * r[j] * w2[e];
          x1[j][e] = ch.turn ? n1 * t.c1[e] - n2 * t.s1[e] : n1;
          x2[j][e] = ch.turn ? n2 * t.c2[e] + n1 * t.s2[e] : n2;
        }
      }
      int64_t at;
      void *dst = pick(q, k, v, dm, tok, hr[j], at);
      store4<T>(dst, at + ch.a, x1[j]);
      store4<T>(dst, at + ch.b, x2[j]);
    }
  }
}

// Backward. Each warp keeps one group of head rows and walks tokens warp / groups, + stride, ...,
// the next token's rows in flight while this one's are worked on; so a lane's head row, weights
// and weight sums stay the same. part (may be NULL): fp32 [gridDim, 2, d], this CTA's sums of dqw
// and dkw.
template <int T, int L, int W>
__global__ void __launch_bounds__(kThreads, 3)
    norm_rope_bwd(const void *__restrict__ dq, const void *__restrict__ dk,
                  const void *__restrict__ dv, const void *__restrict__ qkv,
                  const void *__restrict__ lq, const void *__restrict__ qw,
                  const void *__restrict__ kw, const float *__restrict__ cosv,
                  const float *__restrict__ sinv, const int64_t *__restrict__ pos_idx,
                  void *__restrict__ dqkv, float *__restrict__ part, NormDims dm, FastDiv seq_div,
                  int lanes, int groups) {
  pdl_wait();
  pdl_release();
  using Raw = typename Quad<T>::type;
  const int wid = blockIdx.x * kWarps + (threadIdx.x >> 5);
  const int stride = (int)gridDim.x * kWarps / groups;  // tokens between a warp's
  const int lane = threadIdx.x & (lanes - 1), slot = (threadIdx.x & 31) / lanes;
  const int rows_at_once = 32 / lanes, total = dm.nh + 2 * dm.nkv;
  const int hr = (wid % groups) * rows_at_once + slot;
  const Chunks ch = chunks_of(lane, dm.d, dm.rot);
  const bool live = ch.live && hr < total, normed = live && hr < dm.nh + dm.nkv;
  const int64_t width = (int64_t)total * dm.d;
  float a1[4] = {0.f, 0.f, 0.f, 0.f}, a2[4] = {0.f, 0.f, 0.f, 0.f};
  float w1[4], w2[4];
  if (normed) {
    load_weight<W>(hr < dm.nh ? qw : kw, dm.w0, ch.a, w1);
    load_weight<W>(hr < dm.nh ? qw : kw, dm.w0, ch.b, w2);
  }
  int64_t tok = wid / groups < stride ? wid / groups : dm.rows;  // warps left over do nothing
  Raw g1 = Quad<T>::zero(), g2 = g1, x1 = g1, x2 = g1;
  int64_t pos = -1;
  auto load = [&](int64_t at_tok) {
    g1 = g2 = x1 = x2 = Quad<T>::zero();
    if (at_tok < dm.rows) {
      pos = __ldg(pos_idx + at_tok);
      if (live) {
        int64_t at;
        const void *src = pick(dq, dk, dv, dm, at_tok, hr, at);
        if (src != nullptr) {
          g1 = load4<T>(src, at + ch.a);
          g2 = load4<T>(src, at + ch.b);
        }
      }
      if (normed) {
        const int64_t at = at_tok * dm.ld + (int64_t)hr * dm.d;
        x1 = load4<T>(qkv, at + ch.a);
        x2 = load4<T>(qkv, at + ch.b);
      }
    }
  };
  load(tok);
  for (; tok < dm.rows; tok += stride) {
    const bool inside = pos >= 0 && pos < dm.slots;
    uint32_t b32 = 0, t32 = 0;
    if (inside) seq_div.divmod((uint32_t)pos, b32, t32);
    Turn t;
    if (normed && ch.turn) t.load(cosv, sinv, t32, dm.rot, ch);
    float f1[4], f2[4], y1[4], y2[4];
    Quad<T>::get(g1, f1);
    Quad<T>::get(g2, f2);
    Quad<T>::get(x1, y1);
    Quad<T>::get(x2, y2);
    if (lq != nullptr && live && hr < dm.nh) {
      const int64_t li = (tok * dm.nh + hr) * (int64_t)dm.d;
      add4<L>(lq, li + ch.a, y1);
      add4<L>(lq, li + ch.b, y2);
    }
    load(tok + stride);
    float ss = 0.f, gx = 0.f;
    if (normed) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (ch.turn) {
          const float d1 = f1[e] * t.c1[e] + f2[e] * t.s2[e];
          const float d2 = f2[e] * t.c2[e] - f1[e] * t.s1[e];
          f1[e] = d1;
          f2[e] = d2;
        }
        ss += y1[e] * y1[e] + y2[e] * y2[e];
        gx += f1[e] * w1[e] * y1[e] + f2[e] * w2[e] * y2[e];
      }
    }
    ss = group_sum(ss, lanes);
    gx = group_sum(gx, lanes);
    if (!live) continue;
    if (!inside) {
#pragma unroll
      for (int e = 0; e < 4; ++e) f1[e] = f2[e] = 0.f;
    } else if (normed) {
      const float r = rsqrtf(ss * dm.inv_d + dm.eps);
      const float k2 = r * r * (gx * dm.inv_d);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        a1[e] += f1[e] * y1[e] * r;
        a2[e] += f2[e] * y2[e] * r;
        f1[e] = r * (f1[e] * w1[e] - y1[e] * k2);
        f2[e] = r * (f2[e] * w2[e] - y2[e] * k2);
      }
    }
    const int64_t at = tok * width + (int64_t)hr * dm.d;
    store4<T>(dqkv, at + ch.a, f1);
    store4<T>(dqkv, at + ch.b, f2);
  }
  if (part == nullptr) return;
  // the lanes' sums, added in order of the warps and their head rows
  __shared__ float sums[kThreads][8];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    sums[threadIdx.x][e] = a1[e];
    sums[threadIdx.x][4 + e] = a2[e];
  }
  __syncthreads();
  const int pairs = dm.rot / 8;
  for (int i = threadIdx.x; i < 2 * dm.d; i += kThreads) {
    const int dim = i < dm.d ? i : i - dm.d, h = dm.rot / 2;
    const int rest = dim - dm.rot;
    const int at = dim < dm.rot ? (dim % h) / 4 : pairs + rest / 8;
    const int e = dim < dm.rot ? (dim >= h ? 4 : 0) + dim % 4 : rest % 8;
    float s = 0.f;
    for (int w = 0; w < kWarps; ++w) {
      const int first = ((blockIdx.x * kWarps + w) % groups) * rows_at_once;
      for (int j = 0; j < rows_at_once; ++j) {
        const bool isq = first + j < dm.nh, isk = !isq && first + j < dm.nh + dm.nkv;
        if (i < dm.d ? isq : isk) s += sums[w * 32 + j * lanes + at][e];
      }
    }
    part[(int64_t)blockIdx.x * 2 * dm.d + i] = s;
  }
}

// Any even head size and alignment: a warp per head row, a lane per pair of dims at a time.
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
  for (int64_t u = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); u < n; u += (int64_t)gridDim.x * 8) {
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
// one lane only.
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

// Lanes of a head row on the vector path (0: not taken).
int lanes_of(const NormDims &dm) {
  if (dm.d % 8 || dm.rot % 8 || dm.d > 256) return 0;
  return pow2_at_least(dm.d / 8);
}

int groups_of(const NormDims &dm, int lanes) {
  const int at_once = 32 / lanes;
  return (dm.nh + 2 * dm.nkv + at_once - 1) / at_once;
}

// Warps a token's head rows are spread over in the forward: one when there are many tokens.
int parts_of(const NormDims &dm, int groups) {
  const int64_t want = ((int64_t)sm_count() * 32 + dm.rows - 1) / dm.rows;
  return (int)(want < groups ? want : groups);
}

// CTAs of the backward: at most the resident ones, whose warps walk the tokens (the vector kernel:
// at least a warp for each group of head rows; the other: one warp a CTA).
int bwd_ctas(int64_t rows, int groups) {
  if (groups == 0) {
    const int64_t cap = (int64_t)sm_count() * 8;
    return (int)(rows < cap ? rows : cap);
  }
  int64_t cap = (int64_t)sm_count() * 3;
  if (cap < (groups + kWarps - 1) / kWarps) cap = (groups + kWarps - 1) / kWarps;
  const int64_t want = (rows * groups + kWarps - 1) / kWarps;
  return (int)(want < cap ? want : cap);
}

int check(const char *what, const NormDims &dm, int64_t batch, int64_t seq, int type, int l_type,
          int w_type) {
  if (dm.rows < 0 || batch < 0 || seq <= 0 || dm.nh <= 0 || dm.nkv < 0 || dm.d <= 0 || dm.d % 2 ||
      dm.rot < 0 || dm.rot % 2 || dm.rot > dm.d)
    return set_error(TB_EINVAL, "%s: bad dims rows=%lld batch=%lld seq=%lld nh=%d nkv=%d d=%d rot=%d",
                     what, (long long)dm.rows, (long long)batch, (long long)seq, dm.nh, dm.nkv,
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
  const int lanes = lanes_of(dm);
  const bool vec = lanes > 0 && ld % 4 == 0 && all_aligned({qkv, q, k, v}, 4 * es) &&
                   all_aligned({lora_q, lora_v}, 4 * ls) &&
                   all_aligned({q_weight, k_weight}, 4 * ws) && all_aligned({cos, sin}, 16);
  cudaStream_t st = as_stream(stream);
  // the LoRA rows and the weights in qkv's type or fp32 on the vector path
  const bool l_own = lora_type == type || (!lora_q && !lora_v);
  const bool w_own = weight_type == type || (!q_weight && !k_weight);
  if (vec && (l_own || lora_type == TB_FP32) && (w_own || weight_type == TB_FP32)) {
    const FastDiv sd((uint32_t)seq);
    const int parts = parts_of(dm, groups_of(dm, lanes));
    const int64_t ctas = (rows * parts + kWarps - 1) / kWarps;
#define TB_FWD(T, L, W)                                                                          \
  return launch("norm_rope_fwd", norm_rope_fwd<T, L, W>, dim3((unsigned)ctas),                   \
                kThreads, 0, st, qkv, lora_q, lora_v, q_weight, k_weight, cos, sin, pos_idx, q,  \
                k, v, dm, sd, FastDiv((uint32_t)parts), lanes)
    if (l_own && w_own) TB_WITH_TYPE(type, T, TB_FWD(T, T, T));
    if (l_own) TB_WITH_TYPE(type, T, TB_FWD(T, T, TB_FP32));
    if (w_own) TB_WITH_TYPE(type, T, TB_FWD(T, TB_FP32, T));
    TB_WITH_TYPE(type, T, TB_FWD(T, TB_FP32, TB_FP32));
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
  const int lanes = lanes_of(dm);
  const int vec = lanes > 0 ? bwd_ctas(rows, groups_of(dm, lanes)) : 0, any = bwd_ctas(rows, 0);
  return (int64_t)(vec > any ? vec : any) * 2 * head_dim * 4;
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
    const int lanes = lanes_of(dm);
    const bool vec = lanes > 0 && ld % 4 == 0 && all_aligned({qkv, dq, dk, dv, dqkv}, 4 * es) &&
                     aligned(lora_q, 4 * ls) && all_aligned({q_weight, k_weight}, 4 * ws) &&
                     all_aligned({cos, sin}, 16);
    const bool l_own = lora_type == type || !lora_q;
    const bool w_own = weight_type == type || (!q_weight && !k_weight);
    if (vec && (l_own || lora_type == TB_FP32) && (w_own || weight_type == TB_FP32)) {
      const FastDiv sd((uint32_t)seq);
      const int groups = groups_of(dm, lanes);
      ctas = bwd_ctas(rows, groups);
#define TB_BWD(T, L, W)                                                                          \
  rc = launch("norm_rope_bwd", norm_rope_bwd<T, L, W>, dim3((unsigned)ctas), kThreads, 0, st, dq, \
              dk, dv, qkv, lora_q, q_weight, k_weight, cos, sin, pos_idx, dqkv, part, dm, sd,     \
              lanes, groups)
      if (l_own && w_own) TB_WITH_TYPE(type, T, TB_BWD(T, T, T));
      else if (l_own) TB_WITH_TYPE(type, T, TB_BWD(T, T, TB_FP32));
      else if (w_own) TB_WITH_TYPE(type, T, TB_BWD(T, TB_FP32, T));
      else TB_WITH_TYPE(type, T, TB_BWD(T, TB_FP32, TB_FP32));
#undef TB_BWD
    } else {
      ctas = bwd_ctas(rows, 0);
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
