// The scaled token embedding and its gradient by sorted tokens, for sm_100a.
//
//   forward    y[t] = scale * W[id_t]
//   gradient   dW[v] = scale * sum over the tokens t with id_t = v of dy[t]   (0 without tokens)
//
// The gradient sorts the keys (id << 32 | t), all different, so the order does not depend on
// timing: tiles of kTile keys by a bitonic network in shared memory, then groups of kWays sorted
// runs are merged by ranks (a key's place in the merged run is its place in its own run plus the
// number of smaller keys in each other run, found by bisection). The tokens of one id are then
// neighbours. A CTA of the sum kernel takes kChunk places of the sorted order and all columns of
// a slice, adds rows in fp32 while the id stays, and writes an id's row when it ends. An id that
// crosses chunks leaves one fp32 partial row per chunk, which the join kernel adds in the order of
// the chunks. So each dy row is read once, each dW row is rounded once and no float atomics run.
// Rows of ids without tokens are zeros, written by the CTAs of the sort launches that do not
// sort (the dense gradient's zeros are most of its bytes: [151936, 1536] fp16 is 467 MB, against
// 621 tokens' 2 MB), so the sort costs no time of its own. With accumulate set nothing is zeroed
// and the sums are added to what dW holds.
//
// Reference: solution/model.py:220-225 embeds the real tokens with a frozen table.
#include "dtypes.cuh"

namespace tb {
namespace {

constexpr int kTile = 2048;         // keys of one shared-memory sort
constexpr int kSortThreads = 512;
constexpr int kWays = 16;           // runs merged per launch
constexpr int kSumThreads = 256;
constexpr uint64_t kNoKey = ~0ull;  // padding of the last tile

__device__ unsigned int g_invalid = 0;

struct Fill {  // the share of the zero fill of one launch: 16-byte words [lo, hi) and byte edges
  uint8_t *base;
  int64_t bytes, lo, hi;
};

// Zeros by the CTAs [first, gridDim): words of 16 bytes from the first aligned address; the
// unaligned edges by the launch that has lo == 0.
__device__ __forceinline__ void zero_fill(const Fill &f, int first) {
  if (f.base == nullptr) return;
  const int64_t head = (16 - (int64_t)(reinterpret_cast<uintptr_t>(f.base) & 15)) & 15;
  uint4 *words = reinterpret_cast<uint4 *>(f.base + head);
  const int64_t nw = f.bytes > head ? (f.bytes - head) / 16 : 0;
  const int64_t me = (int64_t)(blockIdx.x - first) * blockDim.x + threadIdx.x;
  const int64_t all = (int64_t)(gridDim.x - first) * blockDim.x;
  const uint4 z = make_uint4(0, 0, 0, 0);
  for (int64_t i = f.lo + me; i < f.hi && i < nw; i += all) words[i] = z;
  if (f.lo == 0 && me < 16) {
    if (me < head && me < f.bytes) f.base[me] = 0;
    const int64_t tail = head + nw * 16 + me;
    if (tail < f.bytes) f.base[tail] = 0;
  }
}

template <typename I>
__device__ __forceinline__ uint64_t key_of(const I *ids, int64_t t, int64_t vocab, int64_t pad) {
  const int64_t id = (int64_t)ids[t];
  // ids without a gradient sort behind all others, as id `vocab`
  const uint64_t v = id < 0 || id >= vocab || id == pad ? (uint64_t)vocab : (uint64_t)id;
  return v << 32 | (uint64_t)t;
}

// CTAs [0, tiles) sort a tile each; the others fill zeros.
template <typename I>
__global__ void __launch_bounds__(kSortThreads)
    sort_tiles(const I *__restrict__ ids, int64_t n, int64_t vocab, int64_t pad,
               uint64_t *__restrict__ keys, int tiles, Fill fill) {
  pdl_wait();
  pdl_release();
  if ((int)blockIdx.x >= tiles) {
    zero_fill(fill, tiles);
    return;
  }
  __shared__ uint64_t s[kTile];
  const int64_t base = (int64_t)blockIdx.x * kTile;
  for (int i = threadIdx.x; i < kTile; i += kSortThreads)
    s[i] = base + i < n ? key_of(ids, base + i, vocab, pad) : kNoKey;
  __syncthreads();
  for (int size = 2; size <= kTile; size *= 2) {
    for (int stride = size / 2; stride > 0; stride /= 2) {
      for (int p = threadIdx.x; p < kTile / 2; p += kSortThreads) {
        const int i = 2 * p - (p & (stride - 1)), j = i + stride;
        const bool up = (i & size) == 0;
        const uint64_t a = s[i], b = s[j];
        if ((a > b) == up) {
          s[i] = b;
          s[j] = a;
        }
      }
      __syncthreads();
    }
  }
  for (int i = threadIdx.x; i < kTile && base + i < n; i += kSortThreads) keys[base + i] = s[i];
}

// Sorted runs of `run` keys of `in` -> runs of run * kWays keys in `out`. The first `blocks` CTAs
// merge, the others fill zeros.
__global__ void __launch_bounds__(256)
    merge_runs(const uint64_t *__restrict__ in, uint64_t *__restrict__ out, int64_t n, int64_t run,
               int blocks, Fill fill) {
  pdl_wait();
  pdl_release();
  if ((int)blockIdx.x >= blocks) {
    zero_fill(fill, blocks);
    return;
  }
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)blocks * 256) {
    const uint64_t key = in[i];
    const int64_t mine = i / run, first = mine / kWays * kWays;
    int64_t place = first * run + (i - mine * run);
#pragma unroll 4
    for (int64_t r = first; r < first + kWays; ++r) {
      const int64_t lo0 = r * run;
      if (r == mine || lo0 >= n) continue;
      int64_t lo = lo0, hi = lo0 + run < n ? lo0 + run : n;
      while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (in[mid] < key) lo = mid + 1;
        else hi = mid;
      }
      place += lo - lo0;
    }
    out[place] = key;
  }
}

struct SumArgs {
  const uint64_t *keys;
  const void *dy;
  void *dw;
  float *part;  // [chunks, 2, hidden]: a chunk's first id (begun before), its last (going on)
  int64_t n, hidden, vocab;
  int chunk;
  float scale;
  bool accumulate;
};

__device__ __forceinline__ int64_t id_at(const uint64_t *keys, int64_t i, int64_t n) {
  return i >= 0 && i < n ? (int64_t)(__ldg(keys + i) >> 32) : -1;
}

// Writes an id's finished sum (V columns at c).
template <int T, int V>
__device__ __forceinline__ void write_row(const SumArgs &a, int64_t id, int64_t c, float (&f)[8]) {
  const int64_t at = id * a.hidden + c;
  if constexpr (V == 8) {
    float old[8];
    if (a.accumulate) load8<T>(a.dw, at, old);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = a.accumulate ? old[e] + a.scale * f[e] : a.scale * f[e];
    store8<T>(a.dw, at, f);
  } else {
    const float s = a.scale * f[0];
    store1<T>(a.dw, at, a.accumulate ? load1<T>(a.dw, at) + s : s);
  }
}

// G: dy's type, T: dW's. V columns a thread (8 on 16-byte aligned rows, else 1).
template <int G, int T, int V>
__global__ void __launch_bounds__(kSumThreads) sum_chunks(SumArgs a) {
  pdl_wait();
  pdl_release();
  const int64_t p0 = (int64_t)blockIdx.x * a.chunk;
  const int64_t p1 = p0 + a.chunk < a.n ? p0 + a.chunk : a.n;
  const int64_t c = ((int64_t)blockIdx.y * blockDim.x + threadIdx.x) * V;
  if (c >= a.hidden) return;
  const int64_t before = id_at(a.keys, p0 - 1, a.n), after = id_at(a.keys, p1, a.n);
  const int64_t first = id_at(a.keys, p0, a.n);
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  int64_t id = first;
  bool earlier = before == first;  // the running id began in an earlier chunk
  for (int64_t p = p0; p < p1; ++p) {
    const uint64_t key = __ldg(a.keys + p);
    const int64_t next = p + 1 < p1 ? id_at(a.keys, p + 1, a.n) : after;
    if (id < a.vocab) {
      const int64_t at = (int64_t)(key & 0xffffffffu) * a.hidden + c;
      float f[8];
      if constexpr (V == 8) load8<G>(a.dy, at, f);
      else f[0] = load1<G>(a.dy, at);
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] += f[e];
    }
    const bool ends = next != id;
    if (ends || p + 1 == p1) {
      if (id < a.vocab) {
        if (ends && !earlier) {
          write_row<T, V>(a, id, c, acc);
        } else {
          float *dst = a.part + ((int64_t)blockIdx.x * 2 + (earlier ? 0 : 1)) * a.hidden + c;
#pragma unroll
          for (int e = 0; e < V; ++e) dst[e] = acc[e];
        }
      }
      earlier = false;
      id = next;
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = 0.f;
    }
  }
}

// The ids that cross chunks: the CTA of the chunk an id begins in adds its partial rows in order.
template <int T>
__global__ void __launch_bounds__(kSumThreads) join_chunks(SumArgs a) {
  pdl_wait();
  pdl_release();
  const int64_t chunk = blockIdx.x, p1 = (chunk + 1) * a.chunk;
  if (p1 >= a.n) return;
  const int64_t id = id_at(a.keys, p1 - 1, a.n);
  if (id >= a.vocab || id_at(a.keys, p1, a.n) != id) return;
  const int64_t p0 = chunk * a.chunk;
  if (id_at(a.keys, p0, a.n) == id && id_at(a.keys, p0 - 1, a.n) == id) return;  // began earlier
  // the first place behind the id's
  int64_t lo = p1, hi = a.n;
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if ((int64_t)(__ldg(a.keys + mid) >> 32) <= id) lo = mid + 1;
    else hi = mid;
  }
  const int64_t last = (lo - 1) / a.chunk;
  const int64_t c = (int64_t)blockIdx.y * blockDim.x + threadIdx.x;
  if (c >= a.hidden) return;
  float s = a.part[(chunk * 2 + 1) * a.hidden + c];
  for (int64_t k = chunk + 1; k <= last; ++k) s += a.part[k * 2 * a.hidden + c];
  float f[8] = {s};
  write_row<T, 1>(a, id, c, f);
}

// A group of blockDim.x threads per token over its columns, V at a time.
template <int T, int O, int V, typename I>
__global__ void __launch_bounds__(256)
    embedding_fwd(const I *__restrict__ ids, const void *__restrict__ table, int64_t ld,
                  void *__restrict__ out, int64_t n, int64_t hidden, int64_t vocab, float scale) {
  pdl_wait();
  pdl_release();
  for (int64_t t = (int64_t)blockIdx.x * blockDim.y + threadIdx.y; t < n;
       t += (int64_t)gridDim.x * blockDim.y) {
    const int64_t id = (int64_t)ids[t];
    const bool ok = id >= 0 && id < vocab;
    if (!ok && threadIdx.x == 0) atomicAdd(&g_invalid, 1u);
    for (int64_t c = (int64_t)threadIdx.x * V; c < hidden; c += (int64_t)blockDim.x * V) {
      float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if constexpr (V == 8) {
        if (ok) load8<T>(table, id * ld + c, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] *= scale;
        store8<O>(out, t * hidden + c, f);
      } else {
        store1<O>(out, t * hidden + c, ok ? load1<T>(table, id * ld + c) * scale : 0.f);
      }
    }
  }
}

template <int T, int O, typename I>
int run_fwd(const I *ids, const void *table, int64_t ld, void *out, int64_t n, int64_t hidden,
            int64_t vocab, float scale, cudaStream_t st) {
  const bool vec = hidden % 8 == 0 && aligned(table, 16) && aligned(out, 16) &&
                   ld * elem_size<T>() % 16 == 0;
  const int64_t cols = vec ? hidden / 8 : hidden;
  const int64_t passes = (cols + 255) / 256;
  const int tx = (int)((cols + passes - 1) / passes), ty = 256 / tx;
  int64_t blocks = (n + ty - 1) / ty;
  const int64_t cap = (int64_t)sm_count() * 32;
  if (blocks > cap) blocks = cap;
  const dim3 grid((unsigned)blocks), block(tx, ty);
  if (vec)
    return launch("embedding_fwd", embedding_fwd<T, O, 8, I>, grid, block, 0, st, ids, table, ld,
                  out, n, hidden, vocab, scale);
  return launch("embedding_fwd", embedding_fwd<T, O, 1, I>, grid, block, 0, st, ids, table, ld,
                out, n, hidden, vocab, scale);
}

// Places of the sorted order a CTA sums: enough CTAs for the device, 32 places at most.
int chunk_of(int64_t n) { return n >= 32768 ? 32 : n >= 8192 ? 16 : 8; }

struct GradPlan {
  int64_t tiles, chunks, keys_bytes, part_bytes;
  int chunk, merges;
};

GradPlan grad_plan(int64_t n, int64_t hidden) {
  GradPlan p;
  p.tiles = (n + kTile - 1) / kTile;
  p.chunk = chunk_of(n);
  p.chunks = (n + p.chunk - 1) / p.chunk;
  p.merges = 0;
  for (int64_t run = kTile; run < n; run *= kWays) ++p.merges;
  p.keys_bytes = (n * 8 + 15) / 16 * 16;
  p.part_bytes = p.chunks * 2 * hidden * 4;
  return p;
}

template <int G, int T>
int run_sums(const SumArgs &a, int64_t chunks, cudaStream_t st) {
  const bool vec = a.hidden % 8 == 0 && aligned(a.dy, 16) && aligned(a.dw, 16);
  const int64_t cols = vec ? a.hidden / 8 : a.hidden;
  const int64_t slices = (cols + kSumThreads - 1) / kSumThreads;
  int threads = (int)((cols + slices - 1) / slices);
  threads = (threads + 31) / 32 * 32;
  const dim3 grid((unsigned)chunks, (unsigned)slices);
  int rc = vec ? launch("embedding_grad", sum_chunks<G, T, 8>, grid, threads, 0, st, a)
               : launch("embedding_grad", sum_chunks<G, T, 1>, grid, threads, 0, st, a);
  if (rc != TB_OK || chunks == 1) return rc;
  const dim3 jgrid((unsigned)chunks, (unsigned)((a.hidden + kSumThreads - 1) / kSumThreads));
  return launch("embedding_grad", join_chunks<T>, jgrid, kSumThreads, 0, st, a);
}

int check_sizes(const char *what, int64_t n, int64_t hidden, int64_t vocab) {
  if (n < 0 || hidden <= 0 || vocab <= 0 || n > 0x7fffffffLL || vocab > 0x7fffffffLL ||
      hidden > (1 << 20))
    return set_error(TB_EINVAL, "%s: n %lld hidden %lld vocab %lld", what, (long long)n,
                     (long long)hidden, (long long)vocab);
  return TB_OK;
}

}  // namespace

unsigned int embedding_invalid_ids(bool &ok) {
  unsigned int v = 0;
  ok = cudaMemcpyFromSymbol(&v, g_invalid, sizeof(v)) == cudaSuccess;
  return v;
}

}  // namespace tb

using namespace tb;

extern "C" int tb_embedding_fwd(const void *ids, int32_t ids_int64, const void *table, int32_t type,
                                int64_t ld, void *out, int32_t out_type, float scale, int64_t n,
                                int64_t hidden, int64_t vocab, void *stream) {
  int rc = check_sizes("embedding_fwd", n, hidden, vocab);
  if (rc != TB_OK) return rc;
  if (!elem_type_ok(type) || !elem_type_ok(out_type) || (out_type != type && out_type != TB_FP32))
    return set_error(TB_EINVAL, "embedding_fwd: types %d -> %d", type, out_type);
  if (n == 0) return TB_OK;
  if (!ids || !table || !out)
    return set_error(TB_EINVAL, "embedding_fwd: ids, table and out are required");
  if (ld < hidden) return set_error(TB_EINVAL, "embedding_fwd: row stride %lld", (long long)ld);
  if (!aligned(ids, ids_int64 ? 8 : 4) || !aligned(table, elem_size_of(type)) ||
      !aligned(out, elem_size_of(out_type)))
    return set_error(TB_EALIGN, "embedding_fwd: a buffer is not aligned to its element");
  cudaStream_t st = as_stream(stream);
#define TB_FWD(T, O)                                                                             \
  return ids_int64 ? run_fwd<T, O>(static_cast<const int64_t *>(ids), table, ld, out, n, hidden, \
                                   vocab, scale, st)                                             \
                   : run_fwd<T, O>(static_cast<const int32_t *>(ids), table, ld, out, n, hidden, \
                                   vocab, scale, st)
  if (out_type == type) TB_WITH_TYPE(type, T, TB_FWD(T, T));
  TB_WITH_TYPE(type, T, TB_FWD(T, TB_FP32));
#undef TB_FWD
}

extern "C" int64_t tb_embedding_grad_workspace(int64_t n, int64_t hidden) {
  if (n <= 0 || hidden <= 0) return 0;
  const GradPlan p = grad_plan(n, hidden);
  return 2 * p.keys_bytes + p.part_bytes;
}

extern "C" int tb_embedding_grad(const void *ids, int32_t ids_int64, const void *dy,
                                 int32_t dy_type, void *dw, int32_t type, float scale,
                                 int64_t padding_idx, int32_t accumulate, int64_t n,
                                 int64_t hidden, int64_t vocab, void *workspace,
                                 int64_t workspace_bytes, void *stream) {
  int rc = check_sizes("embedding_grad", n, hidden, vocab);
  if (rc != TB_OK) return rc;
  if (!elem_type_ok(type) || !elem_type_ok(dy_type) ||
      (dy_type != type && dy_type != TB_FP32 && type != TB_FP32))
    return set_error(TB_EINVAL, "embedding_grad: types %d -> %d", dy_type, type);
  if (n == 0 && accumulate) return TB_OK;
  if (!dw || (n > 0 && (!ids || !dy)))
    return set_error(TB_EINVAL, "embedding_grad: ids, dy and dw are required");
  const int es = elem_size_of(type);
  if (!aligned(dw, es) || !aligned(dy, elem_size_of(dy_type)) || !aligned(ids, ids_int64 ? 8 : 4) ||
      !aligned(workspace, 16))
    return set_error(TB_EALIGN, "embedding_grad: a buffer is not aligned to its element");
  if (n > 0 && (!workspace || workspace_bytes < tb_embedding_grad_workspace(n, hidden)))
    return set_error(TB_EINVAL, "embedding_grad: workspace of %lld bytes, %lld needed",
                     (long long)workspace_bytes,
                     (long long)tb_embedding_grad_workspace(n, hidden));
  cudaStream_t st = as_stream(stream);
  const GradPlan p = grad_plan(n, hidden);
  uint8_t *ws = static_cast<uint8_t *>(workspace);
  uint64_t *keys = reinterpret_cast<uint64_t *>(ws);
  uint64_t *other = reinterpret_cast<uint64_t *>(ws + p.keys_bytes);
  Fill fill{accumulate ? nullptr : static_cast<uint8_t *>(dw), vocab * hidden * es, 0, 0};
  const int64_t words = fill.bytes / 16 + 1;
  const int fill_ctas = accumulate ? 0 : sm_count() * 4;
  // the zero fill in equal shares over the sort's launches
  const int launches = 1 + p.merges;
  int64_t share = 0;
  auto next_share = [&]() {
    fill.lo = words * share / launches;
    fill.hi = words * ++share / launches;
  };
  next_share();
  const dim3 grid((unsigned)(p.tiles + fill_ctas));
  if (grid.x == 0) return TB_OK;
  if (ids_int64)
    rc = launch("embedding_grad", sort_tiles<int64_t>, grid, kSortThreads, 0, st,
                static_cast<const int64_t *>(ids), n, vocab, padding_idx, keys, (int)p.tiles, fill);
  else
    rc = launch("embedding_grad", sort_tiles<int32_t>, grid, kSortThreads, 0, st,
                static_cast<const int32_t *>(ids), n, vocab, padding_idx, keys, (int)p.tiles, fill);
  if (rc != TB_OK || n == 0) return rc;
  for (int64_t run = kTile; run < n; run *= kWays) {
    next_share();
    int64_t blocks = (n + 255) / 256;
    const int64_t cap = (int64_t)sm_count() * 8;
    if (blocks > cap) blocks = cap;
    rc = launch("embedding_grad", merge_runs, dim3((unsigned)(blocks + fill_ctas)), 256, 0, st,
                keys, other, n, run, (int)blocks, fill);
    if (rc != TB_OK) return rc;
    uint64_t *t = keys;
    keys = other;
    other = t;
  }
  const SumArgs a{keys,  dy,    dw,      reinterpret_cast<float *>(ws + 2 * p.keys_bytes),
                  n,     hidden, vocab, p.chunk, scale, accumulate != 0};
#define TB_SUM(G, T) return run_sums<G, T>(a, p.chunks, st)
  if (dy_type == type) TB_WITH_TYPE(type, T, TB_SUM(T, T));
  if (dy_type == TB_FP32) TB_WITH_TYPE(type, T, TB_SUM(TB_FP32, T));
  TB_WITH_TYPE(dy_type, G, TB_SUM(G, TB_FP32));
#undef TB_SUM
}
