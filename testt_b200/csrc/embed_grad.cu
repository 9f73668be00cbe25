// The scaled token embedding and its gradient by sorted tokens, for sm_100a.
//
//   forward    y[t] = scale * W[id_t]
//   gradient   dW[v] = scale * sum over the tokens t with id_t = v of dy[t]   (0 without tokens)
//
// The gradient sorts the keys (id << 32 | t), all different, so the order does not depend on
// timing: tiles of kTile keys in shared memory (see sort_tiles), then groups of kWays sorted
// runs are merged by ranks (a key's place in the merged run is its place in its own run plus the
// number of smaller keys in each other run, found by bisection). The tokens of one id are then
// neighbours. A CTA of the sum kernel takes kChunk places of the sorted order and all columns of
// a slice, adds rows in fp32 while the id stays, and writes an id's row when it ends. An id that
// crosses chunks leaves one fp32 partial row per chunk, which the join kernel adds in the order of
// the chunks. So each dy row is read once, each dW row is rounded once and no float atomics run.
// Rows of ids without tokens are zeros. The sort's launches clear the first of them with idle CTAs,
// the sum launch writes the rest with CTAs that look the ids with tokens up in the sorted keys:
// they are most of the dense gradient's bytes ([151936, 1536] fp16 is 467 MB, against 621 tokens'
// 2 MB). With accumulate set nothing is zeroed and the sums are added to what dW holds.
//
// Measured, in us (sum of the launches' device times; DRAM as a share of the nominal rate):
//   621 tokens, [151936, 1536] fp16: forward 3.4, gradient 84 (sort 12, sums and zeros 68, join 4),
//     bound by the 467 MB it writes (71 at the rate of a copy).
//   32749 tokens, [50021, 2056] bf16: forward 33 (42 % of DRAM), gradient 102 (sort 14, merge 24,
//     sums and zeros 51 at 61 % of DRAM, join 13): no unit is full in any of the four, which wait
//     for one another; added to an existing gradient 99 (11, 15, 58, 14).
//   Up to 256 tokens in one launch: [151936, 1536] fp16 76 to 79, bound by its writes; [2048, 512]
//     4 to 8, and as much when added to an existing gradient: the sort.
//   Rows not of 8 columns or off 16 bytes take a column a thread: 32749 tokens, [50021, 2052] fp32
//     forward 135 (91 with 2056 columns; issue 68 %), gradient 185 (159).
//
// Reference: solution/model.py:220-225 embeds the real tokens with a frozen table.
#include "dtypes.cuh"

namespace tb {
namespace {

constexpr int kTile = 2048;         // keys of one shared-memory sort
constexpr int kSortThreads = 1024;
constexpr int kFwdPerSm = 4;        // resident CTAs of the forward (33 us; 5, at 48 registers: 45)
constexpr int kWays = 16;           // runs merged per launch
constexpr int kSample = 64;         // sampled keys of a run in a merge
constexpr int kSumThreads = 256;
constexpr int kSmall = 256;         // tokens the one-launch gradient takes
constexpr int kFillRows = 32;       // ids whose zero rows a CTA looks for at a time
constexpr int64_t kSortClears = 40 << 20, kMergeClears = 64 << 20;  // bytes cleared meanwhile
constexpr int kMaxChunk = 32;       // places of the sorted order a CTA sums
// Tokens whose merge groups, and one more for the clearing, a grid's y holds.
constexpr int64_t kMaxTokens = 0x7fff0000;
constexpr uint64_t kNoKey = ~0ull;  // padding of the last tile

__device__ unsigned int g_invalid = 0;

// The first place of the sorted keys whose id is at least `id`, by a warp: 32 probes a round.
__device__ __forceinline__ int64_t place_of(const uint64_t *keys, int64_t n, int64_t id) {
  const int lane = threadIdx.x & 31;
  int64_t lo = 0, hi = n;  // keys below lo are smaller, keys from hi on are not
  while (lo < hi) {
    const int64_t step = (hi - lo + 31) / 32, at = lo + lane * step;
    const bool smaller = at < hi && (int64_t)(__ldg(keys + at) >> 32) < id;
    const int found = __popc(__ballot_sync(0xffffffffu, smaller));
    if (found == 0) return lo;
    const int64_t last = lo + (found - 1) * step;  // the last probe that is smaller
    lo = last + 1;
    if (last + step < hi) hi = last + step;
  }
  return lo;
}

// The first rows of the gradient, [lo, hi) in bytes, that a launch of the sort clears with its CTAs
// from `first` on, before it is known which of them have tokens (the sums overwrite those): enough
// to hide the sort behind.
struct Early {
  uint8_t *base;
  int64_t lo, hi;
};

__device__ __forceinline__ void clear_early(const Early &e, int me, int all) {
  uint8_t *p = e.base + e.lo;
  const int64_t bytes = e.hi - e.lo;
  int64_t head = (16 - (int64_t)(reinterpret_cast<uintptr_t>(p) & 15)) & 15;
  if (head > bytes) head = bytes;
  const int64_t words = (bytes - head) / 16, tail = bytes - head - words * 16;
  uint4 *w = reinterpret_cast<uint4 *>(p + head);
  const int64_t step = (int64_t)all * blockDim.x;
  for (int64_t i = (int64_t)me * blockDim.x + threadIdx.x; i < words; i += step)
    w[i] = make_uint4(0, 0, 0, 0);
  if (me == 0 && threadIdx.x < head) p[threadIdx.x] = 0;
  if (me == 0 && threadIdx.x < tail) p[bytes - tail + threadIdx.x] = 0;
}

// A token's id in the sort: ids without a gradient sort behind all others, as id `vocab`.
template <typename I>
__device__ __forceinline__ int64_t sort_id(const I *ids, int64_t t, int64_t vocab, int64_t pad) {
  const int64_t id = (int64_t)ids[t];
  return id < 0 || id >= vocab || id == pad ? vocab : id;
}

// One step of a bitonic network over the warp's lanes.
template <typename K>
__device__ __forceinline__ K lane_step(K k, int lane, int size, int stride) {
  const K o = __shfl_xor_sync(0xffffffffu, k, stride);
  const bool up = (lane & size) == 0 || size == 32, lower = (lane & stride) == 0;
  return (up == lower) == (k < o) ? k : o;
}

// A CTA a tile of kTile tokens. Inside a tile the keys are (id, place in the tile): in 32 bits (K =
// uint32_t) where the vocabulary is below 2^21 - 1, else in 64. Each warp sorts runs of 32 in its
// lanes, then neighbouring runs are merged by ranks in shared memory (a key's place is its place in
// its run plus the smaller keys of the other, by bisection). The 66-step bitonic network over 2048
// keys took 21 us for any number of tokens.
template <typename I, typename K>
__global__ void __launch_bounds__(kSortThreads)
    sort_tiles(const I *__restrict__ ids, int64_t n, int64_t vocab, int64_t pad,
               uint64_t *__restrict__ keys, int tiles, Early early) {
  pdl_wait();
  pdl_release();
  if ((int)blockIdx.x >= tiles) {
    clear_early(early, (int)blockIdx.x - tiles, (int)gridDim.x - tiles);
    return;
  }
  constexpr int kEach = kTile / kSortThreads, kBits = 11;
  constexpr K kPad = (K)(sizeof(K) == 4 ? 0x1fffffu : 0xffffffffull) << kBits;
  static_assert(kTile == 1 << kBits, "a place in the tile has kBits bits");
  __shared__ K buf[2][kTile];
  const int lane = threadIdx.x & 31;
  const int64_t base = (int64_t)blockIdx.x * kTile;
  const int count = (int)(n - base < kTile ? n - base : kTile);
  K k[kEach];
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int i = threadIdx.x + e * kSortThreads;
    k[e] = i < count ? (K)sort_id(ids, base + i, vocab, pad) << kBits | (K)i : kPad | (K)i;
  }
#pragma unroll
  for (int size = 2; size <= 32; size *= 2)
#pragma unroll
    for (int stride = size / 2; stride > 0; stride /= 2)
#pragma unroll
      for (int e = 0; e < kEach; ++e) k[e] = lane_step(k[e], lane, size, stride);
#pragma unroll
  for (int e = 0; e < kEach; ++e) buf[0][threadIdx.x + e * kSortThreads] = k[e];
  __syncthreads();
  int from = 0;
  for (int run = 32; run < count; run *= 2) {
    int place[kEach];
    const K *other[kEach];
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int i = threadIdx.x + e * kSortThreads;
      k[e] = buf[from][i];
      other[e] = buf[from] + ((i / run) ^ 1) * run;
      place[e] = 0;
    }
    for (int half = run; half > 0; half /= 2)
#pragma unroll
      for (int e = 0; e < kEach; ++e)
        if (place[e] + half <= run && other[e][place[e] + half - 1] < k[e]) place[e] += half;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int i = threadIdx.x + e * kSortThreads;
      buf[from ^ 1][i / (2 * run) * (2 * run) + i % run + place[e]] = k[e];
    }
    __syncthreads();
    from ^= 1;
  }
  for (int i = threadIdx.x; i < count; i += kSortThreads) {
    const K key = buf[from][i];
    keys[base + i] = (uint64_t)(key >> kBits) << 32 | (uint64_t)(base + (key & (kTile - 1)));
  }
}

// Sorted runs of `run` (a power of two) keys of `in` -> runs of run * kWays keys in `out`: kWays
// lanes to a key, a lane counts the smaller keys of one run by bisection, the first steps over a
// sample of kSample keys of each run in shared memory (the probes, not the latencies, are the cost:
// one thread a key over all runs took 44 us for 32749 keys, kWays lanes without the sample 22 us).
// A CTA takes keys of one group of runs only: group blockIdx.y.
__global__ void __launch_bounds__(256)
    merge_runs(const uint64_t *__restrict__ in, uint64_t *__restrict__ out, int64_t n,
               int64_t run, int groups, Early early) {
  pdl_wait();
  pdl_release();
  if ((int)blockIdx.y >= groups) {
    clear_early(early, (int)blockIdx.x, (int)gridDim.x);
    return;
  }
  __shared__ uint64_t sample[kWays][kSample + 1];
  const int64_t start = (int64_t)blockIdx.y * run * kWays;  // the group's first key
  const int64_t end = start + run * kWays < n ? start + run * kWays : n;
  const int64_t each = run / kSample;  // sample j is key (j + 1) each - 1 of its run
  for (int i = threadIdx.x; i < kWays * kSample; i += 256) {
    const int r = i / kSample, j = i % kSample;
    const int64_t at = start + r * run + (j + 1) * each - 1;
    sample[r][j] = at < end ? in[at] : kNoKey;
  }
  __syncthreads();
  const int lane = threadIdx.x % kWays;
  const int64_t per = 256 / kWays, all = start + (end - start + per - 1) / per * per;
  const int64_t lo = start + lane * run;
  const int64_t len = lo >= end ? 0 : end - lo < run ? end - lo : run;
  for (int64_t i = start + blockIdx.x * per + threadIdx.x / kWays; i < all;
       i += (int64_t)gridDim.x * per) {
    const bool live = i < end;
    const uint64_t key = live ? in[i] : 0;
    const int mine = (int)((i - start) / run);
    int64_t smaller = 0;  // keys of the lane's run known to be smaller
    if (live && lane == mine) {
      smaller = i - lo;
    } else if (live && len > 0) {
      int s = 0;
#pragma unroll
      for (int half = kSample; half > 0; half /= 2)
        if (s + half <= kSample && sample[lane][s + half - 1] < key) s += half;
      smaller = s * each;
      for (int64_t half = each / 2; half > 0; half /= 2)
        if (smaller + half <= len && in[lo + smaller + half - 1] < key) smaller += half;
    }
#pragma unroll
    for (int o = kWays / 2; o > 0; o /= 2) smaller += __shfl_xor_sync(0xffffffffu, smaller, o);
    if (live && lane == 0) out[start + smaller] = key;
  }
}

struct SumArgs {
  const uint64_t *keys;
  const void *dy;
  void *dw;
  float *part;  // [chunks, 2, wide]: a chunk's first id (begun before), its last (going on)
  int64_t n, hidden, vocab, wide;  // wide: hidden rounded up to four columns
  int64_t cleared;  // rows the sort's launches have cleared
  int chunk;
  float scale;
  bool accumulate;
};

__device__ __forceinline__ int64_t id_at(const uint64_t *keys, int64_t i, int64_t n) {
  return i >= 0 && i < n ? (int64_t)(__ldg(keys + i) >> 32) : -1;
}

// Writes an id's finished sum (V columns at c).
template <int T, int V>
__device__ __forceinline__ void write_row(const SumArgs &a, int64_t id, int64_t c, float (&f)[V]) {
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

// V columns of a row as loaded, and their fp32 sums (packed in pairs for V = 8).
template <int G, int V>
struct RawRow {
  using type = typename Elem<G>::type;
  using Sum = float[1];
  type v;
  __device__ __forceinline__ void load(const void *p, int64_t at) {
    v = __ldg(static_cast<const type *>(p) + at);
  }
  __device__ __forceinline__ void add_to(Sum &acc) const { acc[0] += Elem<G>::get(v); }
  static __device__ __forceinline__ void clear(Sum &acc) { acc[0] = 0.f; }
  static __device__ __forceinline__ void get(const Sum &acc, float (&f)[1]) { f[0] = acc[0]; }
};

template <int G>
struct RawRow<G, 8> {
  using Sum = F2[4];
  uint4 v[G == TB_FP32 ? 2 : 1];
  __device__ __forceinline__ void load(const void *p, int64_t at) {
    const uint4 *q = reinterpret_cast<const uint4 *>(
        static_cast<const typename Elem<G>::type *>(p) + at);
    v[0] = __ldg(q);
    if constexpr (G == TB_FP32) v[1] = __ldg(q + 1);
  }
  __device__ __forceinline__ void add_to(Sum &acc) const {
    if constexpr (G == TB_FP32) {
      const float *f = reinterpret_cast<const float *>(v);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] = add2(acc[i], make_f2(f[2 * i], f[2 * i + 1]));
    } else {
      const uint32_t *w = reinterpret_cast<const uint32_t *>(v);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = Elem<G>::get2(w[i]);
        acc[i] = add2(acc[i], make_f2(f.x, f.y));
      }
    }
  }
  static __device__ __forceinline__ void clear(Sum &acc) {
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = both(0.f);
  }
  static __device__ __forceinline__ void get(const Sum &acc, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = parts(acc[i]);
      f[2 * i] = p.x;
      f[2 * i + 1] = p.y;
    }
  }
};

// Zeros over `bytes` from p by a warp: 16-byte words between the unaligned edges.
__device__ __forceinline__ void warp_zero(uint8_t *p, int64_t bytes) {
  const int lane = threadIdx.x & 31;
  int64_t head = (16 - (int64_t)(reinterpret_cast<uintptr_t>(p) & 15)) & 15;
  if (head > bytes) head = bytes;
  const int64_t words = (bytes - head) / 16, tail = bytes - head - words * 16;
  uint4 *w = reinterpret_cast<uint4 *>(p + head);
  for (int64_t i = lane; i < words; i += 32) w[i] = make_uint4(0, 0, 0, 0);
  if (lane < head) p[lane] = 0;
  if (lane < tail) p[bytes - tail + lane] = 0;
}

// The zero rows, kFillRows ids to a CTA at a time: the ids among them that have tokens are marked
// from the sorted keys, the warps clear the others.
__device__ __forceinline__ void fill_rows(const SumArgs &a, int row_bytes, int me, int all) {
  __shared__ uint8_t used[kFillRows];
  __shared__ int64_t range[2];
  const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  for (int64_t r0 = a.cleared + (int64_t)me * kFillRows; r0 < a.vocab;
       r0 += (int64_t)all * kFillRows) {
    const int count = (int)(a.vocab - r0 < kFillRows ? a.vocab - r0 : kFillRows);
    for (int i = threadIdx.x; i < kFillRows; i += blockDim.x) used[i] = 0;
    if (warp < 2) {
      const int64_t at = place_of(a.keys, a.n, warp == 0 ? r0 : r0 + count);
      if ((threadIdx.x & 31) == 0) range[warp] = at;
    }
    __syncthreads();
    for (int64_t i = range[0] + threadIdx.x; i < range[1]; i += blockDim.x)
      used[(int64_t)(__ldg(a.keys + i) >> 32) - r0] = 1;
    __syncthreads();
    for (int i = warp; i < count; i += warps)
      if (!used[i]) warp_zero(static_cast<uint8_t *>(a.dw) + (r0 + i) * row_bytes, row_bytes);
    __syncthreads();
  }
}

// Adds the rows of places [from, to) while their id stays, kAhead rows of dy in flight whatever ids
// they belong to, and writes each id's row where it ends (tok has bit 31 set there), or a partial
// row of the chunk. earlier: the first id began in an earlier chunk.
template <int G, int T, int V>
__device__ __forceinline__ void sum_places(const SumArgs &a, const uint32_t *tok,
                                           const uint32_t *ids, int from, int to, bool earlier,
                                           int chunk, int64_t c) {
  constexpr int kAhead = 8;
  using Row = RawRow<G, V>;
  typename Row::Sum acc;
  Row::clear(acc);
  for (int i0 = from; i0 < to; i0 += kAhead) {
    Row row[kAhead];
    const int m = to - i0;
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (j < m) row[j].load(a.dy, (int64_t)(tok[i0 + j] & 0x7fffffffu) * a.hidden + c);
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (j >= m) break;
      const bool ends = (tok[i0 + j] & 0x80000000u) != 0;
      row[j].add_to(acc);
      if (!ends && i0 + j + 1 < to) continue;
      const int64_t id = ids[i0 + j];
      if (id >= a.vocab) return;  // the ids without a gradient are the last
      float f[V];
      Row::get(acc, f);
      if (ends && !earlier) {
        write_row<T, V>(a, id, c, f);
      } else {
        float *dst = a.part + ((int64_t)chunk * 2 + (earlier ? 0 : 1)) * a.wide + c;
        if constexpr (V == 8) {
          store8f(dst, f);
        } else {
          dst[0] = f[0];
        }
      }
      earlier = false;
      Row::clear(acc);
    }
  }
}

// `sums` CTAs (chunks x slices) sum, the others fill zeros: both only need the sorted keys and
// write different rows, so the fill hides the sums' latencies and the sums cost their bytes.
// G: dy's type, T: dW's. V columns a thread (8 on 16-byte aligned rows, else 1).
template <int G, int T, int V>
__global__ void __launch_bounds__(kSumThreads) sum_chunks(SumArgs a, int chunks, int sums) {
  pdl_wait();
  pdl_release();
  // the fill's CTAs are spread among the others: fills(b) of the first b CTAs
  const int64_t fill = (int64_t)gridDim.x - sums;
  const int before = (int)(fill * blockIdx.x / gridDim.x);
  if ((int)(fill * (blockIdx.x + 1) / gridDim.x) != before) {
    fill_rows(a, (int)a.hidden * elem_size<T>(), before, (int)fill);
    return;
  }
  const int me = (int)blockIdx.x - before, slice = me / chunks, chunk = me - slice * chunks;
  // of the chunk's places: the token, with bit 31 set where its id ends; the id
  __shared__ uint32_t sh_tok[kMaxChunk];
  __shared__ uint32_t sh_id[kMaxChunk];
  __shared__ bool sh_earlier;  // the first id began in an earlier chunk
  const int64_t p0 = (int64_t)chunk * a.chunk;
  const int count = (int)(a.n - p0 < a.chunk ? a.n - p0 : a.chunk);
  for (int i = threadIdx.x; i < count; i += blockDim.x) {
    const int64_t p = p0 + i;
    const uint64_t key = __ldg(a.keys + p);
    const uint32_t id = (uint32_t)(key >> 32);
    const bool ends = p + 1 >= a.n || (uint32_t)(__ldg(a.keys + p + 1) >> 32) != id;
    sh_tok[i] = (uint32_t)key | (ends ? 0x80000000u : 0u);
    sh_id[i] = id;
    if (i == 0) sh_earlier = p0 > 0 && (uint32_t)(__ldg(a.keys + p0 - 1) >> 32) == id;
  }
  __syncthreads();
  const int64_t c = ((int64_t)slice * blockDim.x + threadIdx.x) * V;
  if (c >= a.hidden) return;
  sum_places<G, T, V>(a, sh_tok, sh_id, 0, count, sh_earlier, chunk, c);
}

// Adds partials i0, i0 + step, ... of `count` to s (partial 0 is the second row of chunk `first`,
// partial i the first row of chunk first + i), eight in flight.
__device__ __forceinline__ void add_partials(const SumArgs &a, int64_t first, int64_t count,
                                             int64_t i0, int step, int64_t c, float4 &s) {
  constexpr int kAhead = 8;
  for (; i0 < count; i0 += (int64_t)step * kAhead) {
    float4 f[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int64_t i = i0 + (int64_t)j * step;
      f[j] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i < count)
        f[j] = *reinterpret_cast<const float4 *>(
            a.part + ((first + i) * 2 + (i == 0 ? 1 : 0)) * a.wide + c);
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      s.x += f[j].x;
      s.y += f[j].y;
      s.z += f[j].z;
      s.w += f[j].w;
    }
  }
}

template <int T>
__device__ __forceinline__ void write_quad(const SumArgs &a, int64_t id, int64_t c, float4 s) {
  const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float f[1] = {v[e]};
    if (c + e < a.hidden) write_row<T, 1>(a, id, c + e, f);
  }
}

// The ids that cross chunks, 128 columns to a CTA. Warp w looks at chunk 8 x + w: whether an id
// begins in it and goes on, and how far; up to kAlone partial rows it adds itself, in order. Longer
// ones the CTA adds together afterwards, a warp every eighth row, then the warps' sums in order.
template <int T>
__global__ void __launch_bounds__(kSumThreads, 4) join_chunks(SumArgs a, int64_t chunks) {
  pdl_wait();
  pdl_release();
  constexpr int kWarps = kSumThreads / 32, kAlone = 24;
  __shared__ int64_t sh_id[kWarps], sh_count[kWarps];
  __shared__ float4 sh_sum[kWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t chunk = (int64_t)blockIdx.x * kWarps + warp;
  const int64_t c = (int64_t)blockIdx.y * 128 + lane * 4;
  int64_t id = -1, count = 0;
  const int64_t p0 = chunk * a.chunk, p1 = p0 + a.chunk;
  if (chunk < chunks && p1 < a.n) {
    const int64_t here = id_at(a.keys, p1 - 1, a.n), next = id_at(a.keys, p1, a.n);
    const int64_t start = id_at(a.keys, p0, a.n), before = id_at(a.keys, p0 - 1, a.n);
    if (here < a.vocab && next == here && !(start == here && before == here)) {
      id = here;
      // most go on into the next chunk only
      const int64_t behind = id_at(a.keys, p1 + a.chunk, a.n);
      const int64_t end = behind == id ? place_of(a.keys, a.n, id + 1) : p1 + 1;
      count = behind == id ? (end - 1) / a.chunk - chunk + 1 : 2;
    }
  }
  if (lane == 0) {
    sh_id[warp] = id;
    sh_count[warp] = count > kAlone ? count : 0;
  }
  if (count > 0 && count <= kAlone && c < a.wide) {
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    add_partials(a, chunk, count, 0, 1, c, s);
    write_quad<T>(a, id, c, s);
  }
  __syncthreads();
  for (int w = 0; w < kWarps; ++w) {
    if (sh_count[w] == 0) continue;  // for the whole CTA
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (c < a.wide)
      add_partials(a, (int64_t)blockIdx.x * kWarps + w, sh_count[w], warp, kWarps, c, s);
    sh_sum[warp][lane] = s;
    __syncthreads();
    if (warp == 0) {
      for (int i = 1; i < kWarps; ++i) {
        const float4 o = sh_sum[i][lane];
        s.x += o.x;
        s.y += o.y;
        s.z += o.z;
        s.w += o.w;
      }
      if (c < a.wide) write_quad<T>(a, sh_id[w], c, s);
    }
    __syncthreads();
  }
}

// Up to kSmall tokens in one launch, without a workspace: every CTA sorts the keys for itself (2
// us), then sums the ids that begin in its places, whole, or fills zeros.
template <int G, int T, int V>
__global__ void __launch_bounds__(kSmall)
    grad_small(SumArgs a, const void *__restrict__ ids, bool ids64, int64_t pad, int chunks,
               int sums) {
  pdl_wait();
  pdl_release();
  __shared__ uint64_t buf[2][kSmall];
  __shared__ uint32_t sh_tok[kSmall], sh_id[kSmall], sh_starts[kSmall / 32];
  __shared__ uint8_t used[kFillRows];
  const int t = threadIdx.x, lane = t & 31, n = (int)a.n;
  uint64_t k = 0xffffffffull << 32 | (uint32_t)t;
  if (t < n)
    k = (uint64_t)(ids64 ? sort_id(static_cast<const int64_t *>(ids), t, a.vocab, pad)
                         : sort_id(static_cast<const int32_t *>(ids), t, a.vocab, pad)) << 32 |
        (uint32_t)t;
#pragma unroll
  for (int size = 2; size <= 32; size *= 2)
#pragma unroll
    for (int stride = size / 2; stride > 0; stride /= 2) k = lane_step(k, lane, size, stride);
  int from = 0;
  buf[0][t] = k;
  __syncthreads();
  for (int run = 32; run < n; run *= 2) {
    const uint64_t *other = buf[from] + ((t / run) ^ 1) * run;
    int place = 0;
    k = buf[from][t];
    for (int half = run; half > 0; half /= 2)
      if (place + half <= run && other[place + half - 1] < k) place += half;
    buf[from ^ 1][t / (2 * run) * (2 * run) + t % run + place] = k;
    __syncthreads();
    from ^= 1;
  }
  k = buf[from][t];
  const uint32_t id = (uint32_t)(k >> 32);
  const bool ends = t + 1 >= n || (uint32_t)(buf[from][t + 1] >> 32) != id;
  const bool starts = t >= n || t == 0 || (uint32_t)(buf[from][t - 1] >> 32) != id;
  sh_tok[t] = (uint32_t)k | (ends ? 0x80000000u : 0u);
  sh_id[t] = id;
  const uint32_t word = __ballot_sync(0xffffffffu, starts);
  if (lane == 0) sh_starts[t / 32] = word;
  __syncthreads();
  const int64_t fill = (int64_t)gridDim.x - sums;
  const int before = (int)(fill * blockIdx.x / gridDim.x);
  if ((int)(fill * (blockIdx.x + 1) / gridDim.x) != before) {
    const int64_t row_bytes = a.hidden * elem_size<T>();
    for (int64_t r0 = (int64_t)before * kFillRows; r0 < a.vocab; r0 += fill * kFillRows) {
      const int count = (int)(a.vocab - r0 < kFillRows ? a.vocab - r0 : kFillRows);
      if (t < kFillRows) used[t] = 0;
      __syncthreads();
      if (t < n && (int64_t)id >= r0 && (int64_t)id < r0 + count) used[id - r0] = 1;
      __syncthreads();
      for (int i = t / 32; i < count; i += kSmall / 32)
        if (!used[i]) warp_zero(static_cast<uint8_t *>(a.dw) + (r0 + i) * row_bytes, row_bytes);
      __syncthreads();
    }
    return;
  }
  const int me = (int)blockIdx.x - before, slice = me / chunks, chunk = me - slice * chunks;
  const int64_t c = ((int64_t)slice * kSmall + t) * V;
  if (c >= a.hidden) return;
  // the first start at or behind a place (n behind the last)
  auto start_from = [&](int p) {
    for (int w = p / 32; w < kSmall / 32; ++w) {
      const uint32_t bits = sh_starts[w] & (w == p / 32 ? 0xffffffffu << (p % 32) : 0xffffffffu);
      if (bits) return w * 32 + __ffs(bits) - 1;
    }
    return kSmall;
  };
  const int s = start_from(chunk * a.chunk);
  const int e = (chunk + 1) * a.chunk < n ? start_from((chunk + 1) * a.chunk) : n;
  if (s < n) sum_places<G, T, V>(a, sh_tok, sh_id, s, e < n ? e : n, false, 0, c);
}

// Vectors of V columns, numbered through the tokens (`cols` to a token), kAhead in flight a thread;
// the next ones' ids are on their way meanwhile.
template <int T, int O, int V, int kAhead, typename I>
__global__ void __launch_bounds__(256, kAhead == 1 ? 8 : kFwdPerSm)
    embedding_fwd(const I *__restrict__ ids, const void *__restrict__ table, int64_t ld,
                  void *__restrict__ out, uint32_t all, FastDiv cols, int64_t hidden,
                  int64_t vocab, float scale) {
  pdl_wait();
  pdl_release();
  uint32_t tok[kAhead], vec[kAhead];
  I id[kAhead];
  auto look = [&](uint32_t first) {
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const uint32_t i = first + j * 256;
      cols.divmod(i < all ? i : 0, tok[j], vec[j]);
      id[j] = i < all ? __ldg(ids + tok[j]) : (I)-1;
    }
  };
  const uint32_t step = gridDim.x * 256 * kAhead;
  uint32_t first = blockIdx.x * 256 * kAhead + threadIdx.x;
  look(first);
  while (first < all) {
    RawRow<T, V> row[kAhead];
    int64_t at[kAhead];
    bool ok[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      ok[j] = id[j] >= 0 && (int64_t)id[j] < vocab;
      at[j] = (int64_t)tok[j] * hidden + vec[j] * V;
      if (ok[j]) row[j].load(table, (int64_t)id[j] * ld + vec[j] * V);
      else if (first + j * 256 < all && vec[j] == 0) atomicAdd(&g_invalid, 1u);
    }
    const uint32_t now = first;
    first = all - first > step ? first + step : all;
    look(first);
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (now + j * 256 >= all) break;
      typename RawRow<T, V>::Sum sum;
      RawRow<T, V>::clear(sum);
      if (ok[j]) row[j].add_to(sum);
      float f[V];
      RawRow<T, V>::get(sum, f);
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] *= scale;
      if constexpr (V == 8) store8<O>(out, at[j], f);
      else store1<O>(out, at[j], f[0]);
    }
  }
}

template <int T, int O, int V, typename I>
int launch_fwd(const I *ids, const void *table, int64_t ld, void *out, int64_t all, int64_t cols,
               int64_t hidden, int64_t vocab, float scale, cudaStream_t st) {
  const FastDiv fd((uint32_t)cols);
  const int64_t resident = (int64_t)sm_count() * 8 * 256;
  if (all <= resident)  // a vector a thread when that does not fill the device
    return launch("embedding_fwd", embedding_fwd<T, O, V, 1, I>,
                  dim3((unsigned)((all + 255) / 256)), 256, 0, st, ids, table, ld, out,
                  (uint32_t)all, fd, hidden, vocab, scale);
  int64_t blocks = (all + 1023) / 1024;
  const int64_t cap = (int64_t)sm_count() * kFwdPerSm;
  if (blocks > cap) blocks = cap;
  return launch("embedding_fwd", embedding_fwd<T, O, V, 4, I>, dim3((unsigned)blocks), 256, 0, st,
                ids, table, ld, out, (uint32_t)all, fd, hidden, vocab, scale);
}

template <int T, int O, typename I>
int run_fwd(const I *ids, const void *table, int64_t ld, void *out, int64_t n, int64_t hidden,
            int64_t vocab, float scale, cudaStream_t st) {
  const bool vec = hidden % 8 == 0 && aligned(table, 16) && aligned(out, 16) &&
                   ld * elem_size<T>() % 16 == 0;
  const int64_t cols = vec ? hidden / 8 : hidden;
  const int64_t most = 0x7fff0000LL / cols;  // tokens a launch numbers in 32 bits
  for (int64_t t = 0; t < n; t += most) {
    const int64_t all = (n - t < most ? n - t : most) * cols;
    void *o = static_cast<char *>(out) + t * hidden * elem_size<O>();
    const auto run = vec ? launch_fwd<T, O, 8, I> : launch_fwd<T, O, 1, I>;
    const int rc = run(ids + t, table, ld, o, all, cols, hidden, vocab, scale, st);
    if (rc != TB_OK) return rc;
  }
  return TB_OK;
}

// Places of the sorted order a CTA sums: two or more CTAs an SM where there are as many tokens.
int chunk_of(int64_t n) { return n >= 16384 ? kMaxChunk : n >= 8192 ? 16 : 8; }

struct GradPlan {
  int64_t tiles, chunks, keys_bytes, part_bytes, wide;
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
  p.wide = (hidden + 3) / 4 * 4;
  p.part_bytes = p.chunks * 2 * p.wide * 4;
  return p;
}

template <int G, int T>
int run_small(SumArgs a, const void *ids, bool ids64, int64_t pad, cudaStream_t st) {
  const bool vec = a.hidden % 8 == 0 && aligned(a.dy, 16) && aligned(a.dw, 16);
  const int64_t slices = ((vec ? a.hidden / 8 : a.hidden) + kSmall - 1) / kSmall;
  a.chunk = a.n > 64 ? 4 : 1;
  const int chunks = (int)((a.n + a.chunk - 1) / a.chunk);
  int64_t fill = 0;
  if (!a.accumulate) {
    fill = (int64_t)sm_count() * 4;
    const int64_t units = (a.vocab + kFillRows - 1) / kFillRows;
    if (fill > units) fill = units;
  }
  const int64_t sums = chunks * slices;
  const dim3 grid((unsigned)(sums + fill));
  if (vec)
    return launch("embedding_grad", grad_small<G, T, 8>, grid, kSmall, 0, st, a, ids, ids64, pad,
                  chunks, (int)sums);
  return launch("embedding_grad", grad_small<G, T, 1>, grid, kSmall, 0, st, a, ids, ids64, pad,
                chunks, (int)sums);
}

template <typename I>
int run_sort(const I *ids, int64_t n, int64_t vocab, int64_t pad, uint64_t *keys, int64_t tiles,
             const Early &early, cudaStream_t st) {
  const dim3 grid((unsigned)(tiles + (early.hi > early.lo ? sm_count() : 0)));
  if (vocab < (1 << 21) - 1)
    return launch("embedding_grad", sort_tiles<I, uint32_t>, grid, kSortThreads, 0, st, ids, n,
                  vocab, pad, keys, (int)tiles, early);
  return launch("embedding_grad", sort_tiles<I, uint64_t>, grid, kSortThreads, 0, st, ids, n, vocab,
                pad, keys, (int)tiles, early);
}

template <int G, int T>
int run_sums(const SumArgs &a, int64_t chunks, cudaStream_t st) {
  const bool vec = a.hidden % 8 == 0 && aligned(a.dy, 16) && aligned(a.dw, 16);
  const int64_t cols = vec ? a.hidden / 8 : a.hidden;
  const int64_t slices = (cols + kSumThreads - 1) / kSumThreads;
  int threads = (int)((cols + slices - 1) / slices);
  threads = (threads + 31) / 32 * 32;
  if (threads < 64) threads = 64;  // two warps look for the fill's ids
  const int64_t sums = chunks * slices;
  // the fill: enough resident CTAs to run at the memory's rate, fewer when there are few rows
  int64_t fill = 0;
  if (!a.accumulate) {
    fill = (int64_t)sm_count() * (1024 / threads);
    const int64_t units = (a.vocab - a.cleared + kFillRows - 1) / kFillRows;
    if (fill > units) fill = units;
  }
  if (sums + fill > 0x7fffffffLL)
    return set_error(TB_EINVAL, "embedding_grad: %lld tokens of %lld columns", (long long)a.n,
                     (long long)a.hidden);
  if (sums + fill == 0) return TB_OK;
  const dim3 grid((unsigned)(sums + fill));
  int rc = vec ? launch("embedding_grad", sum_chunks<G, T, 8>, grid, threads, 0, st, a, (int)chunks,
                        (int)sums)
               : launch("embedding_grad", sum_chunks<G, T, 1>, grid, threads, 0, st, a, (int)chunks,
                        (int)sums);
  if (rc != TB_OK || chunks <= 1) return rc;
  const dim3 jgrid((unsigned)((chunks + 7) / 8), (unsigned)((a.hidden + 127) / 128));
  return launch("embedding_grad", join_chunks<T>, jgrid, kSumThreads, 0, st, a, chunks);
}

int check_sizes(const char *what, int64_t n, int64_t hidden, int64_t vocab) {
  if (n < 0 || hidden <= 0 || vocab <= 0 || n > kMaxTokens || vocab > 0x7fffffffLL ||
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
  if (n <= kSmall || hidden <= 0) return 0;
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
  if (n > kSmall && (!workspace || workspace_bytes < tb_embedding_grad_workspace(n, hidden)))
    return set_error(TB_EINVAL, "embedding_grad: workspace of %lld bytes, %lld needed",
                     (long long)workspace_bytes,
                     (long long)tb_embedding_grad_workspace(n, hidden));
  cudaStream_t st = as_stream(stream);
#define TB_WITH_GRAD(RUN)                                            \
  do {                                                               \
    if (dy_type == type) TB_WITH_TYPE(type, T, RUN(T, T));           \
    if (dy_type == TB_FP32) TB_WITH_TYPE(type, T, RUN(TB_FP32, T));  \
    TB_WITH_TYPE(dy_type, G, RUN(G, TB_FP32));                       \
  } while (0)
  if (n <= kSmall) {
    const SumArgs a{nullptr, dy, dw, nullptr, n,     hidden,
                    vocab,   hidden, 0, 1, scale, accumulate != 0};
#define TB_SMALL(G, T) return run_small<G, T>(a, ids, ids_int64 != 0, padding_idx, st)
    TB_WITH_GRAD(TB_SMALL);
#undef TB_SMALL
  }
  const GradPlan p = grad_plan(n, hidden);
  uint8_t *ws = static_cast<uint8_t *>(workspace);
  uint64_t *keys = reinterpret_cast<uint64_t *>(ws);
  uint64_t *other = reinterpret_cast<uint64_t *>(ws + p.keys_bytes);
  // rows the sort's launches clear, whole ones
  const int64_t row_bytes = hidden * es;
  int64_t cleared = 0;
  Early early{static_cast<uint8_t *>(dw), 0, 0};
  auto clear_rows = [&](int64_t bytes) {
    early.lo = cleared * row_bytes;
    const int64_t next = cleared + bytes / row_bytes;
    if (!accumulate) cleared = next < vocab ? next : vocab;
    early.hi = cleared * row_bytes;
  };
  {
    clear_rows(kSortClears);
    rc = ids_int64 ? run_sort(static_cast<const int64_t *>(ids), n, vocab, padding_idx, keys,
                              p.tiles, early, st)
                   : run_sort(static_cast<const int32_t *>(ids), n, vocab, padding_idx, keys,
                              p.tiles, early, st);
    if (rc != TB_OK) return rc;
  }
  for (int64_t run = kTile; run < n; run *= kWays) {
    const int64_t group = run * kWays, groups = (n + group - 1) / group;
    int64_t blocks = ((n < group ? n : group) * kWays + 255) / 256;
    const int64_t cap = (int64_t)sm_count() * 8 / groups + 1;
    if (blocks > cap) blocks = cap;
    clear_rows(kMergeClears);
    rc = launch("embedding_grad", merge_runs,
                dim3((unsigned)blocks, (unsigned)(groups + (early.hi > early.lo ? 1 : 0))), 256, 0,
                st, keys, other, n, run, (int)groups, early);
    if (rc != TB_OK) return rc;
    uint64_t *t = keys;
    keys = other;
    other = t;
  }
  const SumArgs a{keys,  dy,    dw,      reinterpret_cast<float *>(ws + 2 * p.keys_bytes),
                  n,     hidden, vocab, p.wide, cleared, p.chunk, scale, accumulate != 0};
#define TB_SUM(G, T) return run_sums<G, T>(a, p.chunks, st)
  TB_WITH_GRAD(TB_SUM);
#undef TB_SUM
#undef TB_WITH_GRAD
}
