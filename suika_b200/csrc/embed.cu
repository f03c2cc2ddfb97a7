// Scaled embedding lookup in a vocabulary shard and its gradient by sorted tokens (sm_100a).
//
// Lookup: out[i] = scale * weight[id_i - lo] where the shard [lo, lo + rows) holds id_i, else zeros; the
// sum of all shards' outputs is the whole table's. One read of the rows and one write of the output.
//
// Gradient: d weight[r] = scale * sum of grad_out[i] over the tokens i with id_i - lo == r, in the tokens'
// order. Tokens are sorted by row (stable), so that a row's tokens are neighbours, and every sum is
// taken in 32 bits in an order that depends on the ids alone: no float atomics, the same bits on
// every run. Three launches: (1) one cluster sorts in distributed shared memory while every other
// CTA clears the output, (2) tiles of sorted tokens are summed, (3) rows longer than a tile are
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
  for (int64_t u = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); u < units; u += (int64_t)gridDim.x * 8) {
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
constexpr uint32_t kPadKey = 0xffffffffu;

struct SortArgs {
  const void* ids;
  bool wide;
  int32_t n;
  int64_t lo;
  int64_t rows;
  int bits;        // of the largest key, `rows` (a token the shard does not hold)
  uint32_t* keys;  // sorted rows
  int32_t* toks;   // their tokens
  char* fill;      // output to clear, or null
  uint64_t fill_bytes;
};

__device__ void clear_range(char* p, uint64_t bytes, uint64_t cta, uint64_t ctas) {
  const uint64_t head = min(bytes, (uint64_t)((16 - ((uintptr_t)p & 15)) & 15));
  const uint64_t vecs = (bytes - head) / 16, tail = bytes - head - vecs * 16;
  if (cta == 0 && threadIdx.x < head) p[threadIdx.x] = 0;
  if (cta == 0 && threadIdx.x < tail) p[head + vecs * 16 + threadIdx.x] = 0;
  char* body = p + head;
  for (uint64_t i = cta * kSortThreads + threadIdx.x; i < vecs; i += ctas * kSortThreads) st16(body + i * 16, make_uint4(0, 0, 0, 0));
}

// Stable radix sort, 8 bits a pass, by one cluster. CTA c holds positions [c * CAP, (c + 1) * CAP) of the
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
  uint16_t(*cnt)[256] = reinterpret_cast<uint16_t(*)[256]>(buf + CAP);  // per warp and digit, at most 32 * R
  __shared__ uint32_t total[256], base[256], scan[8];
  cg::cluster_group cluster = cg::this_cluster();
  const int cs = cluster.num_blocks();
  if (blockIdx.x >= cs) {  // not in the sorting cluster
    clear_range(a.fill, a.fill_bytes, blockIdx.x - cs, gridDim.x - cs);
    return;
  }
  const int me = cluster.block_rank(), w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t below = (1u << lane) - 1;
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
  for (int shift = 0; shift < a.bits; shift += 8) {
    if (shift) {
#pragma unroll
      for (int r = 0; r < R; ++r) item[r] = buf[w * 32 * R + r * 32 + lane];
    }
    for (int i = threadIdx.x; i < 32 * 128; i += kSortThreads) reinterpret_cast<uint32_t*>(cnt)[i] = 0;
    __syncthreads();
    uint32_t rank[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint32_t d = (item[r].x >> shift) & 255;
      const uint32_t peers = __match_any_sync(~0u, d);
      const uint32_t before = cnt[w][d];
      __syncwarp();
      rank[r] = before + __popc(peers & below);
      if ((peers & below) == 0) cnt[w][d] = (uint16_t)(before + __popc(peers));
      __syncwarp();
    }
    __syncthreads();
    if (threadIdx.x < 256) {
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
    if (threadIdx.x < 256) {
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
    if (threadIdx.x < 256) {
      for (int k = 0; k < w; ++k) excl += scan[k];
      base[threadIdx.x] = excl + before;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint32_t d = (item[r].x >> shift) & 255;
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

constexpr int kMaxTile = 64;  // sorted tokens per CTA
constexpr int kCols = 8;      // columns per thread

struct SumArgs {
  const uint32_t* keys;
  const int32_t* toks;
  int32_t n;
  int32_t tile;
  int64_t rows;
  int32_t hidden;
  int64_t grad_stride;
  float scale;
  bool accumulate;
  float* partial;  // [tiles][2][hidden]: the piece of a long row that enters a tile, and the one that leaves it
};

// First position in [lo, hi) whose key is not below `key` (upper: above it).
__device__ __forceinline__ int bound_of(const uint32_t* keys, int lo, int hi, uint32_t key, bool upper) {
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (upper ? keys[mid] <= key : keys[mid] < key) lo = mid + 1; else hi = mid;
  }
  return lo;
}

template <class G, int E>
__device__ __forceinline__ void add_out(G* out, int64_t at, const float* x, bool accumulate) {
  Pack<G, E>* p = reinterpret_cast<Pack<G, E>*>(out + at);
  Pack<G, E> v;
  if (accumulate) v = *p;
#pragma unroll
  for (int e = 0; e < E; ++e) v.x[e] = from_f32<G>(accumulate ? to_f32<G>(v.x[e]) + x[e] : x[e]);
  *p = v;
}

// A CTA sums the rows that start among its `tile` sorted tokens, for blockDim.x * 8 columns. A row of
// at most `tile` tokens is summed whole by the CTA where it starts (reading at most tile - 1 tokens of the next
// tile); a longer one is cut at the tiles' borders and its pieces go to `partial` for the join. So
// no CTA sums more than 2 * tile - 1 tokens, however uneven the ids are. Four tokens' vectors are
// loaded before the first is added: with 16-bit gradients that is 64 bytes in flight per thread.
template <class T, class G, int E>
__global__ void __launch_bounds__(256) sum_kernel(SumArgs a, const T* grad, G* out) {
  constexpr int NV = kCols / E;
  __shared__ uint32_t keys[3 * kMaxTile];
  __shared__ int32_t toks[2 * kMaxTile];
  const int s = blockIdx.x * a.tile, e = min(s + a.tile, a.n);
  const int w0 = max(s - a.tile, 0), w1 = min(e + a.tile, a.n);
  for (int i = w0 + threadIdx.x; i < w1; i += blockDim.x) keys[i - w0] = a.keys[i];
  for (int i = s + threadIdx.x; i < w1; i += blockDim.x) toks[i - s] = a.toks[i];
  __syncthreads();
  // the range [pos, end) of positions this CTA sums
  int pos = s, end = e;
  bool head = false, tail = false;
  if (s > 0 && keys[s - 1 - w0] == keys[s - w0]) {  // a row that started earlier
    const uint32_t k = keys[s - w0];
    const int a0 = w0 + bound_of(keys, 0, s - w0, k, false), b0 = w0 + bound_of(keys, s - w0, w1 - w0, k, true);
    // where the window cuts the row off, it is longer than a tile
    const bool is_long = (a0 == w0 && w0 > 0) || b0 - a0 > a.tile;
    if (is_long) head = true; else pos = min(b0, e);
  }
  if (pos < e) {
    const uint32_t k = keys[e - 1 - w0];
    const int a1 = w0 + bound_of(keys, pos - w0, e - w0, k, false), b1 = w0 + bound_of(keys, e - 1 - w0, w1 - w0, k, true);
    if (!(head && a1 == s)) {  // the last row starts in this tile
      if (b1 - a1 > a.tile) tail = true; else end = b1;
    }
  }
  if (pos >= end) return;
  const int col0 = (int)blockIdx.y * blockDim.x * kCols + threadIdx.x * E;
  const int step = blockDim.x * E;
  bool on[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) on[v] = col0 + v * step < a.hidden;
  float acc[NV][E];
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int q = 0; q < E; ++q) acc[v][q] = 0.f;
  constexpr int U = 4;
  for (int p = pos; p < end; p += U) {
    Pack<T, E> x[U][NV];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (p + u < end && keys[p + u - w0] < a.rows) {
        const T* g = grad + (int64_t)toks[p + u - s] * a.grad_stride + col0;
#pragma unroll
        for (int v = 0; v < NV; ++v)
          if (on[v]) x[u][v] = *reinterpret_cast<const Pack<T, E>*>(g + v * step);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int q = p + u;
      if (q >= end) break;
      const uint32_t row = keys[q - w0];
      if (row >= a.rows) return;  // tokens that this shard does not hold, sorted last
#pragma unroll
      for (int v = 0; v < NV; ++v)
        if (on[v]) {
#pragma unroll
          for (int c = 0; c < E; ++c) acc[v][c] += to_f32<T>(x[u][v].x[c]);
        }
      const bool last = q + 1 == end || keys[q + 1 - w0] != row;
      if (!last) continue;
      const bool is_head = head && row == keys[s - w0], is_tail = tail && q + 1 == end && !is_head;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        if (on[v]) {
          const int col = col0 + v * step;
          if (is_head || is_tail) {
            float* to = a.partial + ((int64_t)blockIdx.x * 2 + (is_tail ? 1 : 0)) * a.hidden + col;
#pragma unroll
            for (int c = 0; c < E; ++c) to[c] = acc[v][c];
          } else {
#pragma unroll
            for (int c = 0; c < E; ++c) acc[v][c] *= a.scale;
            add_out<G, E>(out, (int64_t)row * a.hidden + col, acc[v], a.accumulate);
          }
        }
#pragma unroll
        for (int c = 0; c < E; ++c) acc[v][c] = 0.f;
      }
    }
  }
}

// Joins the pieces of a row longer than a tile: the CTA of the tile where the row starts adds the piece
// that leaves this tile and those that enter the next ones, in order.
template <class G>
__global__ void __launch_bounds__(256) join_kernel(SumArgs a, G* out) {
  const int s = blockIdx.x * a.tile, e = s + a.tile;
  if (e >= a.n) return;
  const uint32_t k = a.keys[e - 1];
  if (k >= a.rows || a.keys[e] != k || (s > 0 && a.keys[s - 1] == k)) return;
  const int a0 = bound_of(a.keys, s, e, k, false);
  if (a0 + a.tile >= a.n || a.keys[a0 + a.tile] != k) return;  // at most a tile long: summed whole already
  int pieces = 0;  // tiles after this one that the row enters
  for (int t = blockIdx.x + 1;; t += blockDim.x) {
    const int64_t at = (int64_t)(t + (int)threadIdx.x) * a.tile;
    const int got = __syncthreads_count(at < a.n && a.keys[at] == k);
    pieces += got;
    if (got < (int)blockDim.x) break;
  }
  for (int col = blockIdx.y * blockDim.x + threadIdx.x; col < a.hidden; col += gridDim.y * blockDim.x) {
    const float* p = a.partial + (int64_t)blockIdx.x * 2 * a.hidden + col;
    float acc = p[a.hidden];
    int t = 1;
    for (; t + 7 <= pieces; t += 8) {
      float x[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) x[u] = p[(int64_t)(t + u) * 2 * a.hidden];
#pragma unroll
      for (int u = 0; u < 8; ++u) acc += x[u];
    }
    for (; t <= pieces; ++t) acc += p[(int64_t)t * 2 * a.hidden];
    acc *= a.scale;
    add_out<G, 1>(out, (int64_t)k * a.hidden + col, &acc, a.accumulate);
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
int launch_lookup(const rs_embed_opts& o, const void* ids, const void* weight, void* out, int sms, cudaStream_t st) {
  const int b = sizeof(T);
  const int e = vector_elements(16 / b, (uint64_t)weight, (uint64_t)o.weight_stride * b, b, (uint64_t)out, (uint64_t)o.hidden * b, b, (int)o.hidden);
  const int segs = (int)((o.hidden / e + 127) / 128);
  const int64_t units = o.n_tokens * segs;
  const int grid = (int)std::min<int64_t>((units + 7) / 8, (int64_t)sms * 16);
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

struct GradPlan {
  int cluster = 1, items = 1, tile = 8, tiles = 0, threads = 32, chunks = 1;
  uint64_t keys = 0, toks = 0, partial = 0, bytes = 0;
};

// The cluster grows before the items per thread do (eight CTAs sort 8192 tokens one per thread). A tile
// holds as many tokens as still leave about six CTAs to an SM, 8 to 64: short tiles keep the sums of a
// few tokens parallel, long ones cost fewer pieces.
GradPlan plan_grad(const rs_embed_opts& o, int sms) {
  GradPlan p;
  const int64_t n = o.n_tokens;
  while (p.cluster < kSortMaxCluster && (int64_t)p.cluster * kSortThreads < n) p.cluster *= 2;
  while ((int64_t)p.cluster * kSortThreads * p.items < n) p.items *= 2;
  const int64_t threads = (o.hidden + kCols - 1) / kCols;
  p.threads = (int)std::min<int64_t>(256, std::max<int64_t>(32, (threads + 31) / 32 * 32));
  p.chunks = (int)std::max<int64_t>(1, (o.hidden + (int64_t)p.threads * kCols - 1) / ((int64_t)p.threads * kCols));
  while (p.tile < kMaxTile && n * p.chunks / p.tile > (int64_t)sms * 6) p.tile *= 2;
  p.tiles = (int)((n + p.tile - 1) / p.tile);
  auto slot = [&](uint64_t b) { const uint64_t at = p.bytes; p.bytes += (b + 255) / 256 * 256; return at; };
  p.keys = slot((uint64_t)n * 4);
  p.toks = slot((uint64_t)n * 4);
  p.partial = slot(p.tiles > 1 ? (uint64_t)p.tiles * 2 * o.hidden * 4 : 0);
  return p;
}

template <int R>
int launch_sort(const SortArgs& a, int cluster, int grid, cudaStream_t st) {
  const size_t smem = (size_t)R * kSortThreads * sizeof(uint2) + 32 * 256 * sizeof(uint16_t);
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
  cfg.numAttrs = 1;
  return tcuda(cudaLaunchKernelEx(&cfg, sort_fill_kernel<R>, a), "rs_embed_grad: launch (sort)");
}

template <class T, class G>
int launch_sums(const SumArgs& a, const GradPlan& p, const void* grad, void* out, cudaStream_t st) {
  const int e = vector_elements(16 / (int)sizeof(T), (uint64_t)grad, (uint64_t)a.grad_stride * sizeof(T), sizeof(T),
                                (uint64_t)out, (uint64_t)a.hidden * sizeof(G), sizeof(G), a.hidden);
  const dim3 grid(p.tiles, p.chunks);
  auto go = [&](auto E) {
    constexpr int EE = decltype(E)::value;
    sum_kernel<T, G, EE><<<grid, p.threads, 0, st>>>(a, (const T*)grad, (G*)out);
  };
  if (e == 8) { if constexpr (sizeof(T) == 2) go(std::integral_constant<int, 8>{}); }
  else if (e == 4) go(std::integral_constant<int, 4>{});
  else if (e == 2) go(std::integral_constant<int, 2>{});
  else go(std::integral_constant<int, 1>{});
  int rc = tcuda(cudaGetLastError(), "rs_embed_grad: launch (sums)");
  if (rc != RS_OK || p.tiles < 2) return rc;
  join_kernel<G><<<dim3(p.tiles, (a.hidden + 255) / 256), 256, 0, st>>>(a, (G*)out);
  return tcuda(cudaGetLastError(), "rs_embed_grad: launch (join)");
}

template <class T>
int sums_of(const SumArgs& a, const GradPlan& p, uint32_t grad_dtype, const void* grad, void* out, cudaStream_t st) {
  if (grad_dtype == RS_F32) return launch_sums<T, float>(a, p, grad, out, st);
  if (grad_dtype == RS_BF16) return launch_sums<T, __nv_bfloat16>(a, p, grad, out, st);
  return launch_sums<T, __half>(a, p, grad, out, st);
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
    const int sms = sm_count(device);
    cudaStream_t st = (cudaStream_t)stream;
    if (o.dtype == RS_F32) return launch_lookup<float>(o, ids_dev, weight_dev, out_dev, sms, st);
    if (o.dtype == RS_BF16) return launch_lookup<__nv_bfloat16>(o, ids_dev, weight_dev, out_dev, sms, st);
    return launch_lookup<__half>(o, ids_dev, weight_dev, out_dev, sms, st);
  });
}

int rs_embed_grad_workspace_bytes(const rs_embed_opts* opts, int32_t device, uint64_t* bytes) {
  int rc = check_opts("rs_embed_grad_workspace_bytes", opts);
  if (rc != RS_OK) return rc;
  if (!bytes) return tfail(RS_ERR_ARG, "rs_embed_grad_workspace_bytes: NULL result");
  if (opts->n_tokens > kSortMax) return tfail(RS_ERR_CAPACITY, "rs_embed_grad: more than 65536 tokens in one call");
  *bytes = std::max<uint64_t>(256, plan_grad(*opts, sm_count(device)).bytes);
  return RS_OK;
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
    DeviceGuard guard(device);
    if (guard.err != cudaSuccess) return tcuda(guard.err, "rs_embed_grad: cudaSetDevice");
    const int sms = sm_count(device);
    cudaStream_t st = (cudaStream_t)stream;
    const uint64_t out_bytes = (uint64_t)o.rows * o.hidden * gb;
    if (o.n_tokens == 0)
      return o.accumulate ? RS_OK : tcuda(cudaMemsetAsync(grad_dev, 0, out_bytes, st), "rs_embed_grad: cudaMemsetAsync");
    if (!ids_dev || !grad_out_dev || (uint64_t)ids_dev % (o.wide_ids ? 8 : 4) || (uint64_t)grad_out_dev % b)
      return tfail(RS_ERR_ARG, "rs_embed_grad: NULL or misaligned ids or output gradient");
    const GradPlan p = plan_grad(o, sms);
    if (!workspace || workspace_bytes < p.bytes || (uintptr_t)workspace % 256)
      return tfail(RS_ERR_CAPACITY, "rs_embed_grad: workspace too small or not 256-byte aligned");
    char* ws = (char*)workspace;
    SortArgs s{};
    s.ids = ids_dev;
    s.wide = o.wide_ids != 0;
    s.n = (int32_t)o.n_tokens;
    s.lo = o.lo;
    s.rows = o.rows;
    while (s.bits < 32 && (uint64_t)o.rows >> s.bits) ++s.bits;
    s.keys = (uint32_t*)(ws + p.keys);
    s.toks = (int32_t*)(ws + p.toks);
    int grid = p.cluster;
    if (!o.accumulate) {
      s.fill = (char*)grad_dev;
      s.fill_bytes = out_bytes;
      // one clearing CTA per SM, fewer where there is little to clear (64 KB each)
      const int64_t ctas = std::min<int64_t>(sms, (int64_t)((out_bytes + 65535) / 65536));
      grid += (int)((ctas + p.cluster - 1) / p.cluster * p.cluster);
    }
    rc = p.items == 1 ? launch_sort<1>(s, p.cluster, grid, st) : p.items == 2 ? launch_sort<2>(s, p.cluster, grid, st)
       : p.items == 4 ? launch_sort<4>(s, p.cluster, grid, st) : launch_sort<8>(s, p.cluster, grid, st);
    if (rc != RS_OK) return rc;
    SumArgs a{};
    a.keys = s.keys;
    a.toks = s.toks;
    a.n = s.n;
    a.tile = p.tile;
    a.rows = o.rows;
    a.hidden = (int32_t)o.hidden;
    a.grad_stride = o.grad_stride;
    a.scale = o.scale;
    a.accumulate = o.accumulate != 0;
    a.partial = (float*)(ws + p.partial);
    if (o.dtype == RS_F32) return sums_of<float>(a, p, o.grad_dtype, grad_out_dev, grad_dev, st);
    if (o.dtype == RS_BF16) return sums_of<__nv_bfloat16>(a, p, o.grad_dtype, grad_out_dev, grad_dev, st);
    return sums_of<__half>(a, p, o.grad_dtype, grad_out_dev, grad_dev, st);
  });
}

}  // extern "C"
