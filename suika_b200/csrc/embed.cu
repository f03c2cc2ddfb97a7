// Scaled embedding lookup in a vocabulary shard and its gradient by sorted tokens (sm_100a).
//
// Lookup: out[i] = scale * weight[id_i - lo] where the shard [lo, lo + rows) holds id_i, else zeros; the
// sum of all shards' outputs is the whole table's. One read of the rows and one write of the output.
//
// Gradient: d weight[r] = scale * sum of grad_out[i] over the tokens i with id_i - lo == r, in the tokens'
// order. Tokens are sorted by row (stable), so that a row's tokens are neighbours, and every sum is
// taken in 32 bits in an order that depends on the ids alone: no float atomics, the same bits on
// every run. Three launches: (1) one cluster sorts in distributed shared memory while every other
// CTA clears the output, (2) tiles of 16 sorted tokens are summed, (3) rows longer than a tile are
// joined from their pieces. The bound is HBM: grad_out read once, the gradient written once.
#include "train.cuh"

#include <cooperative_groups.h>

#include <algorithm>

namespace cg = cooperative_groups;

namespace {

using namespace suika_train;

template <class T, int E>
struct alignas(sizeof(T) * E) Pack {
  T x[E];
};

__device__ __forceinline__ int64_t load_id(const void* ids, bool wide, int64_t i) {
  return wide ? reinterpret_cast<const int64_t*>(ids)[i] : (int64_t)reinterpret_cast<const int32_t*>(ids)[i];
}

// ---- lookup -------------------------------------------------------------------------------

// A warp takes a unit of 4 x 32 vectors of one token's row: 64 bytes in flight per thread at the full
// vector width, whole 128-byte lines per warp, and for one token several warps on several SMs.
template <class T, int E>
__global__ void __launch_bounds__(256) lookup_kernel(const void* ids, bool wide, int64_t n, const T* weight, int64_t row_stride,
                                                     int64_t rows, int hidden, int64_t lo, float scale, T* out, int segs) {
  const int lane = threadIdx.x & 31;
  const int64_t units = n * segs;
  const int vecs = hidden / E;
  using P = Pack<T, E>;
  const int64_t u = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (u < units) {
    const int64_t i = u / segs;
    const int v0 = (int)(u - i * segs) * 128 + lane;
    const int64_t r = load_id(ids, wide, i) - lo;
    const bool held = r >= 0 && r < rows;
    const P* src = reinterpret_cast<const P*>(weight + (held ? r : 0) * row_stride);
    P* dst = reinterpret_cast<P*>(out + i * hidden);
    P v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (held && v0 + k * 32 < vecs) v[k] = src[v0 + k * 32];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (v0 + k * 32 >= vecs) break;
#pragma unroll
      for (int e = 0; e < E; ++e) v[k].x[e] = held ? from_f32<T>(to_f32<T>(v[k].x[e]) * scale) : from_f32<T>(0.f);
      dst[v0 + k * 32] = v[k];
    }
  }
}

// ---- sort ---------------------------------------------------------------------------------

constexpr int kSortThreads = 1024;
constexpr int kSortMaxItems = 8;      // per thread
constexpr int kSortMaxCluster = 8;    // the portable cluster size
constexpr int64_t kSortMax = (int64_t)kSortThreads * kSortMaxItems * kSortMaxCluster;  // 65536 tokens
constexpr int kBins = 512;
constexpr uint32_t kPadKey = 0xffffffffu;

struct SortArgs {
  const void* ids;
  bool wide;
  int32_t n;
  int64_t lo;
  int64_t rows;
  int bits;        // of the largest key, `rows` (a token the shard does not hold)
  int digit;       // bits a pass, at most 9
  uint32_t* keys;  // sorted rows
  int32_t* toks;   // their tokens
  int32_t* long_rows;  // a count for the sums, cleared here
  char* fill;      // output to clear, or null
  uint64_t fill_bytes;
};

// A clearing CTA writes one run of 64 KB.
constexpr int kClearBytes = 64 * 1024;
__device__ void clear_run(char* p, uint64_t bytes, uint64_t cta) {
  const uint64_t head = min(bytes, (uint64_t)((16 - ((uintptr_t)p & 15)) & 15));
  const uint64_t vecs = (bytes - head) / 16, tail = bytes - head - vecs * 16;
  if (cta == 0 && threadIdx.x < head) p[threadIdx.x] = 0;
  if (cta == 0 && threadIdx.x < tail) p[head + vecs * 16 + threadIdx.x] = 0;
  char* body = p + head;
  const uint64_t v0 = cta * (kClearBytes / 16) + threadIdx.x;
#pragma unroll
  for (int u = 0; u < kClearBytes / 16 / kSortThreads; ++u)
    if (v0 + u * kSortThreads < vecs) st16(body + (v0 + u * kSortThreads) * 16, make_uint4(0, 0, 0, 0));
}

// Stable radix sort by one cluster, up to 9 bits a pass (18 bits, 262143 rows, are two passes). CTA c holds positions [c * CAP, (c + 1) * CAP) of the
// array as (key, token) pairs in its shared memory; per pass a warp ranks its items among equal
// digits (match_any), counts are summed over warps, CTAs (through distributed shared memory) and
// digits, and every item is stored where it belongs, in whichever CTA that is. Items sit in
// registers between the load and the store of a pass, so one buffer is enough. Two cluster barriers
// a pass: totals visible, then stores visible.
template <int R>
__global__ void __launch_bounds__(kSortThreads) sort_fill_kernel(SortArgs a) {
  constexpr int CAP = R * kSortThreads;
  constexpr int SHIFT = R == 1 ? 10 : R == 2 ? 11 : R == 4 ? 12 : 13;
  static_assert(CAP == 1 << SHIFT, "capacity is a power of two");
  extern __shared__ uint4 smem[];
  uint2* buf = reinterpret_cast<uint2*>(smem);                    // CAP pairs
  uint16_t(*cnt)[kBins] = reinterpret_cast<uint16_t(*)[kBins]>(buf + CAP);  // per warp and digit, at most 32 * R
  __shared__ uint32_t total[kBins], base[kBins], scan[kBins / 32];
  let_successor_start();
  cg::cluster_group cluster = cg::this_cluster();
  const int cs = cluster.num_blocks();
  if (blockIdx.x >= cs) {  // not in the sorting cluster
    clear_run(a.fill, a.fill_bytes, blockIdx.x - cs);
    return;
  }
  const int me = cluster.block_rank(), w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t below = (1u << lane) - 1;
  if (me == 0 && threadIdx.x == 0) *a.long_rows = 0;
  uint2 item[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int i = me * CAP + w * 32 * R + r * 32 + lane;
    uint32_t key = kPadKey;
    if (i < a.n) {
      const int64_t row = load_id(a.ids, a.wide, i) - a.lo;
      key = row >= 0 && row < a.rows ? (uint32_t)row : (uint32_t)a.rows;
    }
    item[r] = make_uint2(key, (uint32_t)i);
  }
  const uint32_t mask = (1u << a.digit) - 1;
  for (int shift = 0; shift < a.bits; shift += a.digit) {
    if (shift) {
#pragma unroll
      for (int r = 0; r < R; ++r) item[r] = buf[w * 32 * R + r * 32 + lane];
    }
    for (int i = threadIdx.x; i < 32 * kBins / 2; i += kSortThreads) reinterpret_cast<uint32_t*>(cnt)[i] = 0;
    __syncthreads();
    uint32_t rank[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint32_t d = (item[r].x >> shift) & mask;
      const uint32_t peers = __match_any_sync(~0u, d);
      const uint32_t before = cnt[w][d];
      __syncwarp();
      rank[r] = before + __popc(peers & below);
      if ((peers & below) == 0) cnt[w][d] = (uint16_t)(before + __popc(peers));
      __syncwarp();
    }
    __syncthreads();
    if (threadIdx.x < kBins) {
      uint32_t sum = 0;
#pragma unroll 8
      for (int k = 0; k < 32; ++k) {
        const uint32_t c = cnt[k][threadIdx.x];
        cnt[k][threadIdx.x] = (uint16_t)sum;  // at most CAP - 1 = 8191
        sum += c;
      }
      total[threadIdx.x] = sum;
    }
    cluster.sync();
    uint32_t all = 0, before = 0, excl = 0;
    if (threadIdx.x < kBins) {
      for (int c = 0; c < cs; ++c) {
        const uint32_t t = cluster.map_shared_rank(total, c)[threadIdx.x];
        if (c < me) before += t;
        all += t;
      }
      uint32_t incl = all;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t t = __shfl_up_sync(~0u, incl, o);
        if (lane >= o) incl += t;
      }
      excl = incl - all;
      if (lane == 31) scan[w] = incl;
    }
    __syncthreads();
    if (threadIdx.x < kBins) {
      for (int k = 0; k < w; ++k) excl += scan[k];
      base[threadIdx.x] = excl + before;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint32_t d = (item[r].x >> shift) & mask;
      const uint32_t to = base[d] + cnt[w][d] + rank[r];
      cluster.map_shared_rank(buf, to >> SHIFT)[to & (CAP - 1)] = item[r];
    }
    cluster.sync();
  }
  for (int k = threadIdx.x; k < CAP; k += kSortThreads) {
    const int i = me * CAP + k;
    if (i < a.n) {
      a.keys[i] = buf[k].x;
      a.toks[i] = (int32_t)buf[k].y;
    }
  }
}

// ---- sums ---------------------------------------------------------------------------------

constexpr int kTile = 16;  // sorted tokens per tile
constexpr int kCols = 8;   // columns per lane
constexpr int kSpan = 32 * kCols;

struct SumArgs {
  const uint32_t* keys;
  const int32_t* toks;
  int32_t n;
  int64_t rows;
  int32_t hidden;
  int32_t spans;  // of kSpan columns
  int64_t grad_stride;
  float scale;
  float* partial;     // [tiles][2][hidden]: the piece of a long row that enters a tile, and the one that leaves it
  int32_t* long_rows; // [0]: how many; then, from [2], (tile where a long row starts, its pieces)
};

template <class G, int E>
__device__ __forceinline__ void store_out(G* out, int64_t at, const float* x) {
  Pack<G, E> v;
#pragma unroll
  for (int e = 0; e < E; ++e) v.x[e] = from_f32<G>(x[e]);
  *reinterpret_cast<Pack<G, E>*>(out + at) = v;
}

// A warp sums the rows that start among the 16 sorted tokens of its tile, for 256 columns. A row of at most 16
// tokens is summed whole by the tile where it starts (up to 15 tokens of the next tile are read); a
// longer one is cut at the tiles' borders, and its pieces go to `partial` for the join. So no warp sums more than
// 31 tokens, however uneven the ids are. The keys from one tile before to one after are held
// two to a lane; where rows start is one 64-bit mask; warps need no barrier. Tokens are taken one by one: two or
// four in flight per warp cost the registers of more warps than they are worth (30011 tokens of 3584 columns added
// to an fp32 gradient, the whole gradient when these three were compared: 155 us, 174 and 209; now 122 with cold
// caches). That is a size with warps to spare: 8192 tokens of which half are held leave some idle.
template <class T, class G, int E, bool ACC>
__global__ void __launch_bounds__(256) sum_kernel(SumArgs a, const T* grad, G* out, int64_t units) {
  let_successor_start();
  after_predecessor();
  constexpr int NV = kCols / E;
  const int64_t unit = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (unit >= units) return;
  const int lane = threadIdx.x & 31;
  const int tile = (int)(unit / a.spans);
  const int col0 = (int)(unit - (int64_t)tile * a.spans) * kSpan + lane * E;
  // window position j is sorted position w0 + j; the tile is [kTile, 2 kTile)
  const int w0 = tile * kTile - kTile;
  auto key_at = [&](int j) { return w0 + j < 0 ? kPadKey - 1 : w0 + j < a.n && j < 3 * kTile ? a.keys[w0 + j] : kPadKey; };
  const uint32_t k0 = key_at(lane), k1 = key_at(lane + 32);
  auto tok_at = [&](int j) { return j >= kTile && j < 3 * kTile && w0 + j < a.n ? a.toks[w0 + j] : 0; };
  const int t0 = tok_at(lane), t1 = tok_at(lane + 32);
  const uint32_t p0 = __shfl_up_sync(~0u, k0, 1), q1 = __shfl_up_sync(~0u, k1, 1), last0 = __shfl_sync(~0u, k0, 31);
  const uint64_t starts = (uint64_t)__ballot_sync(~0u, lane > 0 && k0 != p0) | (uint64_t)__ballot_sync(~0u, k1 != (lane ? q1 : last0)) << 32;
  const uint64_t held = (uint64_t)__ballot_sync(~0u, k0 < a.rows) | (uint64_t)__ballot_sync(~0u, k1 < a.rows) << 32;
  auto start_after = [&](int j) { const uint64_t m = starts >> (j + 1); return m ? j + __ffsll(m) : 3 * kTile; };
  int pos = kTile, end = 2 * kTile;
  bool head = false, tail = false;
  if (!(starts >> kTile & 1)) {  // a row that started earlier
    const uint64_t m = starts & ((1ull << kTile) - 1);
    const int b = start_after(kTile);
    // without a start in the window it reaches back more than a tile
    if (m == 0 || b - (63 - __clzll(m)) > kTile) head = true; else pos = min(b, end);
  }
  if (pos >= end) return;
  {
    const uint64_t m = starts & ((1ull << 2 * kTile) - 1) & ~((1ull << pos) - 1);
    if (m) {  // the last row starts in this tile
      const int b = start_after(2 * kTile - 1);
      if (b - (63 - __clzll(m)) > kTile) tail = true; else end = b;
    }
  }
  {  // tokens that the shard does not hold are sorted last
    const uint64_t m = ~held >> pos;
    const int stop = m ? pos + __ffsll(m) - 1 : end;
    if (stop < end) {
      end = stop;
      tail = false;
    }
  }
  if (pos >= end) return;
  const uint32_t head_key = __shfl_sync(~0u, k0, kTile);
  if (tail && col0 == lane * E) {  // one piece leaves this tile, one enters each of the next as long as the row goes on
    const uint32_t k = __shfl_sync(~0u, k0, 2 * kTile - 1);
    int pieces = 1, got;
    do {
      const int64_t at = (int64_t)(tile + pieces + lane) * kTile;
      got = __popc(__ballot_sync(~0u, at < a.n && a.keys[at] == k));
      pieces += got;
    } while (got == 32);
    if (lane == 0) {
      const int slot = atomicAdd(a.long_rows, 1);  // the order of the list does not matter
      reinterpret_cast<int2*>(a.long_rows)[1 + slot] = make_int2(tile, pieces);
    }
  }
  bool on[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) on[v] = col0 + v * 32 * E < a.hidden;
  float acc[NV][E];
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int c = 0; c < E; ++c) acc[v][c] = 0.f;
  for (int q = pos; q < end; ++q) {
    const int64_t t = q < 32 ? __shfl_sync(~0u, t0, q & 31) : __shfl_sync(~0u, t1, q & 31);
    const uint32_t row = q < 32 ? __shfl_sync(~0u, k0, q & 31) : __shfl_sync(~0u, k1, q & 31);
    const bool last = q + 1 == end || (starts >> (q + 1) & 1);
    const bool enters = head && row == head_key, piece = enters || (tail && q + 1 == end);
    Pack<T, E> x[NV];
    Pack<G, E> old[NV];
    const T* g = grad + t * a.grad_stride + col0;
    G* o = out + (int64_t)row * a.hidden + col0;
#pragma unroll
    for (int v = 0; v < NV; ++v)
      if (on[v]) x[v] = *reinterpret_cast<const Pack<T, E>*>(g + v * 32 * E);
    if (ACC && last && !piece) {
#pragma unroll
      for (int v = 0; v < NV; ++v)
        if (on[v]) old[v] = *reinterpret_cast<const Pack<G, E>*>(o + v * 32 * E);
    }
#pragma unroll
    for (int v = 0; v < NV; ++v)
      if (on[v]) {
#pragma unroll
        for (int c = 0; c < E; ++c) acc[v][c] += to_f32<T>(x[v].x[c]);
      }
    if (!last) continue;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (on[v]) {
        if (piece) {
          store_out<float, E>(a.partial, ((int64_t)tile * 2 + !enters) * a.hidden + col0 + v * 32 * E, acc[v]);
        } else {
#pragma unroll
          for (int c = 0; c < E; ++c) acc[v][c] = ACC ? fmaf(acc[v][c], a.scale, to_f32<G>(old[v].x[c])) : acc[v][c] * a.scale;
          store_out<G, E>(o, v * 32 * E, acc[v]);
        }
      }
#pragma unroll
      for (int c = 0; c < E; ++c) acc[v][c] = 0.f;
    }
  }
}

// Joins the pieces of the rows longer than a tile: the piece that leaves the tile where the row starts and
// those that enter the next ones. A CTA takes 32 x V columns of a row; its 8 warps each add an equal run
// of consecutive pieces in order, and the runs are added in order: the same bits always.
template <class G, int V>
__global__ void __launch_bounds__(256) join_kernel(SumArgs a, G* out, bool accumulate) {
  after_predecessor();
  using P = Pack<float, V>;
  __shared__ P sums[8][32];
  const int chunks = (a.hidden + 32 * V - 1) / (32 * V), lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t units = (int64_t)a.long_rows[0] * chunks;
  for (int64_t unit = blockIdx.x; unit < units; unit += gridDim.x) {
    const int2 row = reinterpret_cast<const int2*>(a.long_rows)[1 + unit / chunks];
    const int tile = row.x, pieces = row.y, col = (int)(unit % chunks) * 32 * V + lane * V;
    const int i0 = (int)((int64_t)pieces * w / 8), i1 = (int)((int64_t)pieces * (w + 1) / 8);
    P acc{};
    if (col < a.hidden) {
      const float* p = a.partial + (int64_t)tile * 2 * a.hidden + col;  // piece i of the row: [tile + i][i == 0]
#pragma unroll 8
      for (int i = i0; i < i1; ++i) {
        const P x = *reinterpret_cast<const P*>(p + ((int64_t)i * 2 + (i == 0)) * a.hidden);
#pragma unroll
        for (int e = 0; e < V; ++e) acc.x[e] += x.x[e];
      }
    }
    sums[w][lane] = acc;
    __syncthreads();
    if (w == 0 && col < a.hidden) {
      const uint32_t k = a.keys[tile * kTile + kTile - 1];
      G* to = out + (int64_t)k * a.hidden + col;
#pragma unroll
      for (int q = 1; q < 8; ++q) {
        const P x = sums[q][lane];
#pragma unroll
        for (int e = 0; e < V; ++e) acc.x[e] += x.x[e];
      }
#pragma unroll
      for (int e = 0; e < V; ++e) to[e] = from_f32<G>(accumulate ? fmaf(acc.x[e], a.scale, to_f32<G>(to[e])) : acc.x[e] * a.scale);
    }
    __syncthreads();
  }
}

// ---- host ---------------------------------------------------------------------------------

// Elements of a vector that every row of the two operands allows: up to 16 bytes.
int vector_elements(int most, uint64_t a, uint64_t a_stride_bytes, int a_bytes, uint64_t b, uint64_t b_stride_bytes, int b_bytes, int hidden) {
  for (int e = most; e > 1; e >>= 1)
    if (hidden % e == 0 && a % (uint64_t)(e * a_bytes) == 0 && a_stride_bytes % (uint64_t)(e * a_bytes) == 0 &&
        b % (uint64_t)(e * b_bytes) == 0 && b_stride_bytes % (uint64_t)(e * b_bytes) == 0)
      return e;
  return 1;
}

template <class T>
int launch_lookup(const rs_embed_opts& o, const void* ids, const void* weight, void* out, cudaStream_t st) {
  const int b = sizeof(T);
  const int e = vector_elements(16 / b, (uint64_t)weight, (uint64_t)o.weight_stride * b, b, (uint64_t)out, (uint64_t)o.hidden * b, b, (int)o.hidden);
  const int segs = (int)((o.hidden / e + 127) / 128);
  const int64_t units = o.n_tokens * segs;
  if ((units + 7) / 8 > 0x7fffffff) return tfail(RS_ERR_CAPACITY, "rs_embed_lookup: too many tokens and columns in one call");
  const unsigned grid = (unsigned)((units + 7) / 8);
  auto go = [&](auto E) {
    constexpr int EE = decltype(E)::value;
    lookup_kernel<T, EE><<<grid, 256, 0, st>>>(ids, o.wide_ids != 0, o.n_tokens, (const T*)weight, o.weight_stride, o.rows, (int)o.hidden, o.lo,
                                               o.scale, (T*)out, segs);
  };
  if (e == 8) { if constexpr (sizeof(T) == 2) go(std::integral_constant<int, 8>{}); }
  else if (e == 4) go(std::integral_constant<int, 4>{});
  else if (e == 2) go(std::integral_constant<int, 2>{});
  else go(std::integral_constant<int, 1>{});
  return tcuda(cudaGetLastError(), "rs_embed_lookup: launch");
}

int check_opts(const char* what, const rs_embed_opts* o) {
  const std::string w(what);
  if (!o) return tfail(RS_ERR_ARG, w + ": NULL options");
  if (o->n_tokens < 0 || o->rows < 0 || o->hidden < 0 || o->weight_stride < 0 || o->grad_stride < 0)
    return tfail(RS_ERR_ARG, w + ": a negative size or stride");
  if (o->hidden > (1 << 30)) return tfail(RS_ERR_CAPACITY, w + ": more than 2^30 columns");
  if (o->rows > 0x7fffffff) return tfail(RS_ERR_CAPACITY, w + ": more than 2^31 rows");
  if (!dtype_known(o->dtype) || !dtype_known(o->grad_dtype)) return tfail(RS_ERR_ARG, w + ": unknown dtype");
  return RS_OK;
}

// Whether `bytes` at `out` touch one of n rows of `width` bytes, `pitch` apart.
bool touches_rows(uint64_t rows, int64_t n, uint64_t pitch, uint64_t width, uint64_t out, uint64_t bytes) {
  if (n == 0 || width == 0 || bytes == 0 || out + bytes <= rows) return false;
  // the first row that ends past `out`
  uint64_t i = 0;
  if (rows + width <= out) {
    if (pitch == 0) return false;
    i = (out - rows - width) / pitch + 1;
  }
  return i < (uint64_t)n && rows + i * pitch < out + bytes;
}

struct GradPlan {
  int cluster = 1, items = 1, tiles = 0;
  uint64_t keys = 0, toks = 0, partial = 0, long_rows = 0, bytes = 0;
};

// The cluster grows before the items per thread do (eight CTAs sort 8192 tokens one per thread).
GradPlan plan_grad(const rs_embed_opts& o) {
  GradPlan p;
  const int64_t n = o.n_tokens;
  while (p.cluster < kSortMaxCluster && (int64_t)p.cluster * kSortThreads < n) p.cluster *= 2;
  while ((int64_t)p.cluster * kSortThreads * p.items < n) p.items *= 2;
  p.tiles = (int)((n + kTile - 1) / kTile);
  auto slot = [&](uint64_t b) { const uint64_t at = p.bytes; p.bytes += (b + 255) / 256 * 256; return at; };
  p.keys = slot((uint64_t)n * 4);
  p.toks = slot((uint64_t)n * 4);
  p.long_rows = slot((uint64_t)(p.tiles + 1) * 8);
  p.partial = slot(p.tiles > 1 ? (uint64_t)p.tiles * 2 * o.hidden * 4 : 0);
  return p;
}

template <int R>
int launch_sort(const SortArgs& a, int cluster, int grid, cudaStream_t st) {
  const size_t smem = (size_t)R * kSortThreads * sizeof(uint2) + 32 * kBins * sizeof(uint16_t);
  if (smem > 40 * 1024) {  // with the static arrays, past the 48 KB that need no opt-in
    cudaError_t e = cudaFuncSetAttribute(sort_fill_kernel<R>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return tcuda(e, "rs_embed_grad: cudaFuncSetAttribute");
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kSortThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cluster;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = cluster > 1;
  return tcuda(cudaLaunchKernelEx(&cfg, sort_fill_kernel<R>, a), "rs_embed_grad: launch (sort)");
}

template <class T, class G>
int launch_sums(const SumArgs& a, const GradPlan& p, const void* grad, void* out, bool accumulate, int sms, cudaStream_t st) {
  const int e = vector_elements(16 / (int)sizeof(T), (uint64_t)grad, (uint64_t)a.grad_stride * sizeof(T), sizeof(T), (uint64_t)out,
                                (uint64_t)a.hidden * sizeof(G), sizeof(G), a.hidden);
  const int64_t units = (int64_t)p.tiles * a.spans;
  if ((units + 7) / 8 > 0x7fffffff) return tfail(RS_ERR_CAPACITY, "rs_embed_grad: too many tokens and columns in one call");
  const unsigned grid = (unsigned)((units + 7) / 8);
  auto go = [&](auto E) {
    constexpr int EE = decltype(E)::value;
    return launch_after(accumulate ? sum_kernel<T, G, EE, true> : sum_kernel<T, G, EE, false>, grid, 256, st, a, (const T*)grad, (G*)out, units);
  };
  cudaError_t launched = cudaErrorInvalidValue;
  if (e == 8) { if constexpr (sizeof(T) == 2) launched = go(std::integral_constant<int, 8>{}); }
  else if (e == 4) launched = go(std::integral_constant<int, 4>{});
  else if (e == 2) launched = go(std::integral_constant<int, 2>{});
  else launched = go(std::integral_constant<int, 1>{});
  int rc = tcuda(launched, "rs_embed_grad: launch (sums)");
  if (rc != RS_OK || p.tiles < 2) return rc;  // one tile has no row longer than a tile
  const int v = a.hidden % 4 == 0 ? 4 : 1;  // columns per lane
  const int64_t most = (int64_t)(p.tiles - 1) * ((a.hidden + 32 * v - 1) / (32 * v));
  const unsigned ctas = (unsigned)std::min<int64_t>(most, (int64_t)sms * 8);
  return tcuda(launch_after(v == 4 ? join_kernel<G, 4> : join_kernel<G, 1>, ctas, 256, st, a, (G*)out, accumulate), "rs_embed_grad: launch (join)");
}

template <class T>
int sums_of(const SumArgs& a, const GradPlan& p, const rs_embed_opts& o, const void* grad, void* out, int sms, cudaStream_t st) {
  const bool acc = o.accumulate != 0;
  if (o.grad_dtype == RS_F32) return launch_sums<T, float>(a, p, grad, out, acc, sms, st);
  if (o.grad_dtype == RS_BF16) return launch_sums<T, __nv_bfloat16>(a, p, grad, out, acc, sms, st);
  return launch_sums<T, __half>(a, p, grad, out, acc, sms, st);
}

}  // namespace

extern "C" {

int rs_embed_lookup(const rs_embed_opts* opts, const void* ids_dev, const void* weight_dev, void* out_dev, int32_t device, void* stream) {
  return guarded("rs_embed_lookup", [&]() -> int {
    int rc = check_opts("rs_embed_lookup", opts);
    if (rc != RS_OK) return rc;
    const rs_embed_opts& o = *opts;
    if (o.n_tokens == 0 || o.hidden == 0) return RS_OK;
    if (!ids_dev || !out_dev || (!weight_dev && o.rows > 0)) return tfail(RS_ERR_ARG, "rs_embed_lookup: NULL address");
    const int b = dtype_bytes(o.dtype);
    if ((uint64_t)ids_dev % (o.wide_ids ? 8 : 4) || (uint64_t)weight_dev % b || (uint64_t)out_dev % b)
      return tfail(RS_ERR_ARG, "rs_embed_lookup: an address is not aligned to its elements");
    DeviceGuard guard(device);
    if (guard.err != cudaSuccess) return tcuda(guard.err, "rs_embed_lookup: cudaSetDevice");
    cudaStream_t st = (cudaStream_t)stream;
    if (o.dtype == RS_F32) return launch_lookup<float>(o, ids_dev, weight_dev, out_dev, st);
    if (o.dtype == RS_BF16) return launch_lookup<__nv_bfloat16>(o, ids_dev, weight_dev, out_dev, st);
    return launch_lookup<__half>(o, ids_dev, weight_dev, out_dev, st);
  });
}

int rs_embed_grad_workspace_bytes(const rs_embed_opts* opts, int32_t device, uint64_t* bytes) {
  return guarded("rs_embed_grad_workspace_bytes", [&]() -> int {
    int rc = check_opts("rs_embed_grad_workspace_bytes", opts);
    if (rc != RS_OK) return rc;
    if (!bytes) return tfail(RS_ERR_ARG, "rs_embed_grad_workspace_bytes: NULL result");
    if (opts->n_tokens > kSortMax) return tfail(RS_ERR_CAPACITY, "rs_embed_grad: more than 65536 tokens in one call");
    *bytes = std::max<uint64_t>(256, plan_grad(*opts).bytes);
    return RS_OK;
  });
}

int rs_embed_grad(const rs_embed_opts* opts, const void* ids_dev, const void* grad_out_dev, void* grad_dev, void* workspace,
                  uint64_t workspace_bytes, int32_t device, void* stream) {
  return guarded("rs_embed_grad", [&]() -> int {
    int rc = check_opts("rs_embed_grad", opts);
    if (rc != RS_OK) return rc;
    const rs_embed_opts& o = *opts;
    if (o.n_tokens > kSortMax) return tfail(RS_ERR_CAPACITY, "rs_embed_grad: more than 65536 tokens in one call");
    if (o.rows == 0 || o.hidden == 0) return RS_OK;
    const int b = dtype_bytes(o.dtype), gb = dtype_bytes(o.grad_dtype);
    if (!grad_dev || (uint64_t)grad_dev % gb) return tfail(RS_ERR_ARG, "rs_embed_grad: NULL or misaligned gradient");
    cudaStream_t st = (cudaStream_t)stream;
    const uint64_t out_bytes = (uint64_t)o.rows * o.hidden * gb;
    if (o.n_tokens == 0) {
      if (o.accumulate) return RS_OK;
      DeviceGuard guard(device);
      if (guard.err != cudaSuccess) return tcuda(guard.err, "rs_embed_grad: cudaSetDevice");
      return tcuda(cudaMemsetAsync(grad_dev, 0, out_bytes, st), "rs_embed_grad: cudaMemsetAsync");
    }
    if (!ids_dev || !grad_out_dev || (uint64_t)ids_dev % (o.wide_ids ? 8 : 4) || (uint64_t)grad_out_dev % b)
      return tfail(RS_ERR_ARG, "rs_embed_grad: NULL or misaligned ids or output gradient");
    // the output is cleared and written while these rows are read
    if (touches_rows((uint64_t)grad_out_dev, o.n_tokens, (uint64_t)o.grad_stride * b, (uint64_t)o.hidden * b, (uint64_t)grad_dev, out_bytes))
      return tfail(RS_ERR_ARG, "rs_embed_grad: the gradient overlaps the output's gradient");
    const GradPlan p = plan_grad(o);
    if (!workspace || workspace_bytes < p.bytes || (uintptr_t)workspace % 256)
      return tfail(RS_ERR_CAPACITY, "rs_embed_grad: workspace too small or not 256-byte aligned");
    DeviceGuard guard(device);
    if (guard.err != cudaSuccess) return tcuda(guard.err, "rs_embed_grad: cudaSetDevice");
    const int sms = sm_count(device);
    char* ws = (char*)workspace;
    SortArgs s{};
    s.ids = ids_dev;
    s.wide = o.wide_ids != 0;
    s.n = (int32_t)o.n_tokens;
    s.lo = o.lo;
    s.rows = o.rows;
    while (s.bits < 32 && (uint64_t)o.rows >> s.bits) ++s.bits;
    const int passes = (s.bits + 8) / 9;
    s.digit = (s.bits + passes - 1) / passes;
    s.keys = (uint32_t*)(ws + p.keys);
    s.toks = (int32_t*)(ws + p.toks);
    s.long_rows = (int32_t*)(ws + p.long_rows);
    int grid = p.cluster;
    if (!o.accumulate) {
      s.fill = (char*)grad_dev;
      s.fill_bytes = out_bytes;
      const uint64_t runs = (out_bytes + kClearBytes - 1) / kClearBytes;
      if (runs > 0x7fffff00) return tfail(RS_ERR_CAPACITY, "rs_embed_grad: gradient too large");
      grid += (int)((runs + p.cluster - 1) / p.cluster * p.cluster);
    }
    rc = p.items == 1 ? launch_sort<1>(s, p.cluster, grid, st) : p.items == 2 ? launch_sort<2>(s, p.cluster, grid, st)
       : p.items == 4 ? launch_sort<4>(s, p.cluster, grid, st) : launch_sort<8>(s, p.cluster, grid, st);
    if (rc != RS_OK) return rc;
    SumArgs a{};
    a.keys = s.keys;
    a.toks = s.toks;
    a.n = s.n;
    a.rows = o.rows;
    a.hidden = (int32_t)o.hidden;
    a.spans = (int32_t)((o.hidden + kSpan - 1) / kSpan);
    a.grad_stride = o.grad_stride;
    a.scale = o.scale;
    a.partial = (float*)(ws + p.partial);
    a.long_rows = s.long_rows;
    if (o.dtype == RS_F32) return sums_of<float>(a, p, o, grad_out_dev, grad_dev, sms, st);
    if (o.dtype == RS_BF16) return sums_of<__nv_bfloat16>(a, p, o, grad_out_dev, grad_dev, sms, st);
    return sums_of<__half>(a, p, o, grad_out_dev, grad_dev, sms, st);
  });
}

}  // extern "C"
