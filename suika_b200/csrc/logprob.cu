// Log probabilities of given tokens, entropy and top alternatives of a vocabulary shard's logits, and
// their gradient (sm_100a).
//
// One pass over the logits keeps, per thread, the running maximum m, S = sum of e^(z - m) and
// A = sum of e^(z - m) (z - m), rescaled where m grows; then lse = m + log S and the entropy is
// log S - A / S. The differences z - m are taken first, so logits of any size (the type's lowest
// value as a mask among them) neither overflow nor lose the digits that the exponent needs. The
// top alternatives need no second pass over the row: each thread notes the maximum of every 64
// bytes it reads, the k-th largest of the block's 32 lane maxima is a bound that at least k logits reach, and
// only the noted places that reach it are read again. All sums are in 32 bits.
//
// HBM is the bound for many rows (each logit is read once, the gradient reads and writes once).
// Few rows are split over the CTAs of a cluster, which join through distributed shared memory.
#include "train.cuh"

#include <cooperative_groups.h>

#include <algorithm>
#include <climits>

namespace cg = cooperative_groups;

namespace {

using namespace suika_train;

constexpr int kThreads = 256;
constexpr int kUnroll = 4;     // 16-byte vectors a thread has in flight
constexpr int kMaxTop = 32;    // lane maxima that bound the k-th largest
constexpr int kMaxCand = 1024; // logits kept for the exact choice
constexpr int kNotes = 40;     // noted maxima per thread: 40 KB for 256 threads
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float exp2_fast(float t) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
  return r;
}

__device__ __forceinline__ int64_t load_target(const void* t, bool wide, int64_t i) {
  return wide ? reinterpret_cast<const int64_t*>(t)[i] : (int64_t)reinterpret_cast<const int32_t*>(t)[i];
}

struct Stat {
  float m, s, a;  // maximum, sum of e^(z - m), sum of e^(z - m) (z - m) in units of ln 2
};

// z - base for the exponent; a row of -inf so far has base 0, whose e^(-inf) is 0.
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }

__device__ __forceinline__ Stat join(const Stat& x, const Stat& y) {
  Stat r;
  r.m = fmaxf(x.m, y.m);
  const float b = base_of(r.m);
  const float tx = fmaxf((base_of(x.m) - b) * kLog2e, -1e4f), ty = fmaxf((base_of(y.m) - b) * kLog2e, -1e4f);
  const float ex = x.m == -INFINITY ? 0.f : exp2_fast(tx), ey = y.m == -INFINITY ? 0.f : exp2_fast(ty);
  // where m is not finite the sums carry the NaN themselves
  r.s = x.s * (x.m == -INFINITY ? 1.f : ex) + y.s * (y.m == -INFINITY ? 1.f : ey);
  r.a = (x.m == -INFINITY ? x.a : ex * (x.a + x.s * tx)) + (y.m == -INFINITY ? y.a : ey * (y.a + y.s * ty));
  return r;
}

// One more logit below or at the maximum.
__device__ __forceinline__ void add_logit(Stat& st, float base, float z) {
  const float t = (z - base) * kLog2e;
  const float e = exp2_fast(t);
  st.s += e;
  st.a = fmaf(e, fmaxf(t, -1e4f), st.a);  // 0 * -inf would be NaN; e is 0 there
}

__device__ __forceinline__ void raise_max(Stat& st, float m) {
  if (m > st.m) {
    const float t = fmaxf((base_of(st.m) - m) * kLog2e, -1e4f);
    if (st.m == -INFINITY) {
      // sums so far are 0, or NaN
    } else {
      const float c = exp2_fast(t);
      st.a = c * (st.a + st.s * t);
      st.s *= c;
    }
    st.m = m;
  }
}

// The order of the alternatives: larger logit first, then the lower index.
__device__ __forceinline__ bool before(float v, int i, float w, int j) { return v > w || (v == w && i < j); }

struct FwdArgs {
  const void* logits;
  int64_t n, cols, stride;
  const void* targets;
  bool wide;
  int64_t lo;
  int top;
  int per_note;    // iterations that share a note
  float* logprob;  // null: write records
  float* entropy;
  float* lse;
  float* top_value;
  int64_t* top_index;
  float* record;   // [n][4 + 2 top]: m, S, A, target's logit (+inf: not here), values, local indices as bits
};

// What one row ends as. S = 0: every logit is -inf. Nothing is possible there: lse and every log
// probability are -inf, the entropy 0.
__device__ __forceinline__ void finish_row(const FwdArgs& a, int64_t row, const Stat& st, float target) {
  const float b = base_of(st.m);
  const bool empty = st.s == 0.f;
  const float log_s = logf(st.s);
  const float lse = empty ? -INFINITY : b + log_s;
  // target - m first: both are logits, their difference is small where it matters
  const float lp = target == INFINITY && !isnan(lse) ? 0.f : empty ? -INFINITY : (target - b) - log_s;
  a.logprob[row] = lp;
  a.entropy[row] = empty ? 0.f : fmaf(-kLn2, st.a / st.s, log_s);
  a.lse[row] = lse;
}

__device__ __forceinline__ float log_prob_of(float z, const Stat& st) {
  return st.s == 0.f ? -INFINITY : (z - base_of(st.m)) - logf(st.s);
}

template <class T>
__device__ __forceinline__ float max_of(uint4 v);
template <> __device__ __forceinline__ float max_of<float>(uint4 v) {
  return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
}
template <> __device__ __forceinline__ float max_of<__nv_bfloat16>(uint4 v) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
  const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
  return fmaxf(__low2float(m), __high2float(m));
}
template <> __device__ __forceinline__ float max_of<__half>(uint4 v) {
  const __half2* h = reinterpret_cast<const __half2*>(&v);
  const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
  return fmaxf(__low2float(m), __high2float(m));
}

__device__ __forceinline__ Stat warp_join(Stat st) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    Stat y;
    y.m = __shfl_xor_sync(~0u, st.m, o);
    y.s = __shfl_xor_sync(~0u, st.s, o);
    y.a = __shfl_xor_sync(~0u, st.a, o);
    st = join(st, y);
  }
  return st;
}

// One 64-bit number per logit whose order is that of the alternatives: larger logit first (-0 as 0), then
// lower index.
__device__ __forceinline__ uint64_t rank_key(float v, int i) {
  uint32_t b = __float_as_uint(v + 0.f);
  b ^= b >> 31 ? 0xffffffffu : 0x80000000u;
  return (uint64_t)b << 32 | (uint32_t)~i;
}
__device__ __forceinline__ float key_value(uint64_t k) {
  uint32_t b = (uint32_t)(k >> 32);
  return __uint_as_float(b ^ (b >> 31 ? 0x80000000u : 0xffffffffu));
}
constexpr uint64_t kNoKey = 0;  // below every logit's (that of -inf is 0x007fffff << 32 and more)
__device__ __forceinline__ int key_index(uint64_t k) { return (int)~(uint32_t)k; }

// The k first of `count` candidates in shared memory, by counting how many come before each.
__device__ __forceinline__ void place_candidates(const uint64_t* cand, int count, int k, uint64_t* best) {
  for (int c = threadIdx.x; c < count; c += kThreads) {
    const uint64_t mine = cand[c];
    int r = 0;
#pragma unroll 8
    for (int d = 0; d < count; ++d) r += cand[d] > mine;
    if (r < k) best[r] = mine;
  }
}

// A cluster of CTAs per row; CTA c takes the c-th share of the row's vectors. Logits before the first
// 16-byte border of a row and after its last whole vector go to single threads of CTA 0.
template <class T>
__global__ void __launch_bounds__(kThreads) forward_kernel(FwdArgs a) {
  constexpr int N = Vec16<T>::N;
  extern __shared__ float notes[];  // [kNotes][kThreads] where alternatives are asked for
  __shared__ Stat warp_stat[8];
  __shared__ float lane_max[8][32];
  __shared__ uint64_t cand[kMaxCand];
  __shared__ uint64_t best[kMaxTop];
  __shared__ Stat cta_stat;
  __shared__ float bound;
  __shared__ int n_cand;
  cg::cluster_group cluster = cg::this_cluster();
  const int cs = cluster.num_blocks(), part = cluster.block_rank();
  const int64_t row = blockIdx.x / cs;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const T* z = reinterpret_cast<const T*>(a.logits) + row * a.stride;
  const int cols = (int)a.cols;
  const int head = min(cols, (int)((16 - ((uintptr_t)z & 15)) & 15) / (int)sizeof(T));
  const int vecs = (cols - head) / N;
  const int v0 = (int)((int64_t)vecs * part / cs), v1 = (int)((int64_t)vecs * (part + 1) / cs);
  const uint4* body = reinterpret_cast<const uint4*>(z + head);
  const int loose = part == 0 ? cols - vecs * N : 0;  // head and tail logits, one per thread (at most 14)
  const int loose_at = tid < head ? tid : tid + vecs * N;
  const int k = a.top;

  Stat st{-INFINITY, 0.f, 0.f};
  float own_max = -INFINITY;  // of whole vectors, for the bound
  int note = 0, in_note = 0;
  float noted = -INFINITY;
  for (int v = v0 + tid; v < v1; v += kUnroll * kThreads) {
    uint4 x[kUnroll];
    float mx = -INFINITY;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (v + u * kThreads < v1) x[u] = ld16(body + v + u * kThreads);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (v + u * kThreads < v1) mx = fmaxf(mx, max_of<T>(x[u]));
    raise_max(st, mx);
    const float base = base_of(st.m);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (v + u * kThreads < v1) {
        float f[N];
        unpack16<T>(x[u], f);
#pragma unroll
        for (int q = 0; q < N; ++q) add_logit(st, base, f[q]);
      }
    }
    if (k) {
      noted = fmaxf(noted, mx);
      if (++in_note == a.per_note) {
        notes[note * kThreads + tid] = noted;
        ++note;
        in_note = 0;
        noted = -INFINITY;
      }
    }
  }
  if (k && in_note) notes[note * kThreads + tid] = noted;
  if (tid < loose) {
    const float f = to_f32<T>(z[loose_at]);
    raise_max(st, f);
    add_logit(st, base_of(st.m), f);
  }
  own_max = st.m;
  const Stat ws = warp_join(st);
  if (lane == 0) warp_stat[w] = ws;
  if (k) lane_max[w][lane] = own_max;
  if (tid == 0) n_cand = 0;
  __syncthreads();

  if (w == 0) {
    Stat t = lane < 8 ? warp_stat[lane] : Stat{-INFINITY, 0.f, 0.f};
    t = warp_join(t);
    if (lane == 0) cta_stat = t;
    if (k) {  // the k-th largest of 32 lane maxima: k logits at least are as large
      float x = lane_max[0][lane];
#pragma unroll
      for (int r = 1; r < 8; ++r) x = fmaxf(x, lane_max[r][lane]);
      int rank = 0;
#pragma unroll
      for (int o = 0; o < 32; ++o) {
        const float y = __shfl_sync(~0u, x, o);
        rank += before(y, o, x, lane);
      }
      if (rank == k - 1) bound = x;
    }
  }
  if (k) {
    if (tid < kMaxTop) best[tid] = kNoKey;
    __syncthreads();
    const float least = bound;
    auto offer = [&](float f, int i) {
      if (f >= least) {
        const int at = atomicAdd(&n_cand, 1);  // their order does not matter: they are ranked by value and index
        if (at < kMaxCand) cand[at] = rank_key(f, i);
      }
    };
    for (int s = 0, v = v0 + tid; v < v1; ++s) {
      const bool look = notes[s * kThreads + tid] >= least;
      for (int q = 0; q < a.per_note && v < v1; ++q, v += kUnroll * kThreads) {
        if (!look) continue;
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          if (v + u * kThreads < v1) {
            float f[N];
            unpack16<T>(ld16(body + v + u * kThreads), f);
#pragma unroll
            for (int e = 0; e < N; ++e) offer(f[e], head + (v + u * kThreads) * N + e);
          }
        }
      }
    }
    if (tid < loose) offer(to_f32<T>(z[loose_at]), loose_at);
    __syncthreads();
    const int count = n_cand;
    if (count <= kMaxCand) {
      place_candidates(cand, count, k, best);
      __syncthreads();
    } else {
      // Too many logits as large as the bound (a nearly constant or mostly masked row): k searches
      // for the first logit after the last one chosen.
      uint64_t chosen = ~0ull;
      for (int r = 0; r < k; ++r) {
        uint64_t next = kNoKey;
        auto look = [&](float f, int i) {
          const uint64_t key = rank_key(f, i);
          if (!isnan(f) && key < chosen && key > next) next = key;
        };
        for (int v = v0 + tid; v < v1; v += kThreads) {
          float f[N];
          unpack16<T>(ld16(body + v), f);
#pragma unroll
          for (int e = 0; e < N; ++e) look(f[e], head + v * N + e);
        }
        if (tid < loose) look(to_f32<T>(z[loose_at]), loose_at);
#pragma unroll
        for (int o = 16; o; o >>= 1) {
          const uint64_t other = __shfl_xor_sync(~0u, next, o);
          if (other > next) next = other;
        }
        __syncthreads();  // the last round's reads of cand are over
        if (lane == 0) cand[w] = next;
        __syncthreads();
        for (int q = 0; q < 8; ++q)
          if (cand[q] > next) next = cand[q];
        if (tid == 0) best[r] = next;
        chosen = next;
      }
      __syncthreads();
    }
  }

  // join the CTAs of the row
  if (cs > 1) {
    cluster.sync();
    if (part == 0) {
      Stat t = cta_stat;
      for (int c = 1; c < cs; ++c) t = join(t, *cluster.map_shared_rank(&cta_stat, c));
      __syncthreads();
      if (tid == 0) cta_stat = t;
      if (k) {
        for (int i = tid; i < cs * k; i += kThreads) {
          const int c = i / k, r = i - c * k;
          cand[i] = cluster.map_shared_rank(best, c)[r];
        }
        __syncthreads();
        if (tid < kMaxTop) best[tid] = kNoKey;
        __syncthreads();
        place_candidates(cand, cs * k, k, best);
      }
    }
    cluster.sync();  // the others' shared memory is read until here
    if (part != 0) return;
  } else {
    __syncthreads();
  }

  const Stat t = cta_stat;
  if (tid == 0) {
    const int64_t at = a.targets ? load_target(a.targets, a.wide, row) - a.lo : -1;
    const float target = at >= 0 && at < a.cols ? to_f32<T>(z[at]) : INFINITY;
    if (a.record) {
      float* r = a.record + row * (4 + 2 * k);
      r[0] = t.m;
      r[1] = t.s;
      r[2] = t.a;
      r[3] = target;
    } else {
      finish_row(a, row, t, target);
    }
  }
  if (tid < k) {
    const bool none = best[tid] == kNoKey;
    const float v = none ? -INFINITY : key_value(best[tid]);
    const int i = none ? -1 : key_index(best[tid]);
    if (a.record) {
      float* r = a.record + row * (4 + 2 * k) + 4;
      r[tid] = v;
      r[k + tid] = __int_as_float(i);
    } else {
      a.top_value[row * k + tid] = log_prob_of(v, t);
      a.top_index[row * k + tid] = none ? -1 : a.lo + i;
    }
  }
}

// Joins the records of the vocabulary's shards, [shards][n][4 + 2 top], one warp per row. Shard s starts at
// vocabulary index starts.lo[s]; shards in ascending order, so that ties go to the lowest index.
constexpr int kMaxShards = 64;
struct Starts {
  int64_t lo[kMaxShards];
};
__global__ void __launch_bounds__(kThreads) merge_kernel(FwdArgs a, const float* records, const __grid_constant__ Starts starts, int shards) {
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= a.n) return;
  const int lane = threadIdx.x & 31, k = a.top, words = 4 + 2 * k;
  Stat st{-INFINITY, 0.f, 0.f};
  float target = INFINITY;
  for (int s = 0; s < shards; ++s) {
    const float* r = records + ((int64_t)s * a.n + row) * words;
    st = join(st, Stat{r[0], r[1], r[2]});
    if (r[3] != INFINITY) target = r[3];
  }
  if (lane == 0) finish_row(a, row, st, target);
  if (lane < k) {
    a.top_value[row * k + lane] = log_prob_of(-INFINITY, st);
    a.top_index[row * k + lane] = -1;
  }
  __syncwarp();
  for (int i = lane; i < shards * k; i += 32) {
    const int s = i / k, q = i - s * k;
    const float* r = records + ((int64_t)s * a.n + row) * words + 4;
    const float v = r[q];
    if (__float_as_int(r[k + q]) < 0) continue;
    int rank = 0;  // a shard's own list is in order, so (shard, place) breaks ties like the index
    for (int t = 0; t < shards; ++t) {
      const float* o = records + ((int64_t)t * a.n + row) * words + 4;
      for (int p = 0; p < k; ++p) {
        const float y = o[p];
        if (__float_as_int(o[k + p]) < 0) break;
        rank += y > v || (y == v && (t < s || (t == s && p < q)));
      }
    }
    if (rank < k) {
      a.top_value[row * k + rank] = log_prob_of(v, st);
      a.top_index[row * k + rank] = starts.lo[s] + __float_as_int(r[k + q]);
    }
  }
}

// ---- gradient -----------------------------------------------------------------------------

struct BwdArgs {
  const void* logits;
  int64_t n, cols, stride;
  const void* targets;
  bool wide;
  bool sharded;  // a target outside [lo, lo + cols) is another shard's; else it is none
  int64_t lo;
  const float* lse;
  const float* entropy;
  const float* grad_logprob;
  const float* grad_entropy;  // null: none
  const float* grad_lse;      // null: none
  void* out;
  int64_t out_stride;
  int units;  // pieces of kUnroll * kThreads vectors in a row
  int ctas;   // CTAs per row: one per piece, or one where the output is the logits (a row that is read again is then read before it is written)
};

// d z_j = g_lp (1[j = t] - p_j) - g_H p_j (log p_j + H) + g_lse p_j, p_j = e^(z_j - lse): one read and one
// write of the row. A row whose gradients are all zero (an ignored token) is written without being read.
template <class T>
__global__ void __launch_bounds__(kThreads) backward_kernel(BwdArgs a) {
  constexpr int N = Vec16<T>::N;
  const int64_t row = blockIdx.x / a.ctas;
  const int first = (int)(blockIdx.x - row * a.ctas);
  const T* z = reinterpret_cast<const T*>(a.logits) + row * a.stride;
  T* out = reinterpret_cast<T*>(a.out) + row * a.out_stride;
  const int64_t target = load_target(a.targets, a.wide, row) - a.lo;
  const float lse = a.lse[row];
  const float h = a.entropy ? a.entropy[row] : 0.f, gh = a.grad_entropy ? a.grad_entropy[row] : 0.f;
  const bool ignored = a.sharded ? target + a.lo < 0 : target < 0 || target >= a.cols;
  const float gl = ignored ? 0.f : a.grad_logprob[row];
  const float gz = a.grad_lse ? a.grad_lse[row] : 0.f, gp = gl - gz;
  const bool none = (gl == 0.f && gh == 0.f && gz == 0.f) || lse == -INFINITY;  // an empty row has no gradient
  const int cols = (int)a.cols;
  // vectors where logits and output have the same place in their 16 bytes
  const bool together = (((uintptr_t)z ^ (uintptr_t)out) & 15) == 0;
  const int head = together ? min(cols, (int)((16 - ((uintptr_t)z & 15)) & 15) / (int)sizeof(T)) : cols;
  const int vecs = (cols - head) / N;
  // log p = (z - base) - rest. The 32 bits of lse are enough for base up to 1024 (p is off by 6e-5 there);
  // a row further out, such as one masked with the type's lowest value, has its maximum and sum taken
  // again, by each of its CTAs. (A shard alone cannot, and stays with lse.)
  float base = lse, rest = 0.f;
  if (!none && !a.sharded && fabsf(lse) > 1024.f && isfinite(lse)) {
    Stat st{-INFINITY, 0.f, 0.f};
    for (int j = threadIdx.x; j < cols; j += kThreads) {
      const float f = to_f32<T>(z[j]);
      raise_max(st, f);
      add_logit(st, base_of(st.m), f);
    }
    st = warp_join(st);
    __shared__ Stat part[8];
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = st;
    __syncthreads();  // every thread has read the row
    st = part[0];
    for (int q = 1; q < 8; ++q) st = join(st, part[q]);
    base = st.m;
    rest = logf(st.s);
  }
  auto one = [&](float f, int j) {
    const float t = (f - base) - rest;
    const float d = fmaxf(t, -1e4f);  // e is 0 below; -inf * 0 would be NaN
    const float p = exp2_fast(t * kLog2e);
    float g = -p * fmaf(gh, d + h, gp);
    if (j == target) g += gl;
    return none ? 0.f : g;
  };
  const int per = kUnroll * kThreads;
  const uint4* src = reinterpret_cast<const uint4*>(z + head);
  uint4* dst = reinterpret_cast<uint4*>(out + head);
  for (int unit = first; unit < a.units; unit += a.ctas) {
    const int v = unit * per + threadIdx.x;
    uint4 x[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (!none && v + u * kThreads < vecs) x[u] = ld16(src + v + u * kThreads);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int q = v + u * kThreads;
      if (q >= vecs) break;
      float f[N];
      if (!none) {
        unpack16<T>(x[u], f);
#pragma unroll
        for (int e = 0; e < N; ++e) f[e] = one(f[e], head + q * N + e);
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) f[e] = 0.f;
      }
      st16(dst + q, pack16<T>(f));
    }
  }
  // what the vectors leave out: a few logits, or the whole row where the two lie differently
  const int loose = cols - vecs * N;
  for (int i = first * kThreads + threadIdx.x; i < loose; i += a.ctas * kThreads) {
    const int j = i < head ? i : i + vecs * N;
    out[j] = from_f32<T>(one(none ? 0.f : to_f32<T>(z[j]), j));
  }
}

// ---- host ---------------------------------------------------------------------------------

int check_opts(const char* what, const rs_logprob_opts* o) {
  const std::string w(what);
  if (!o) return tfail(RS_ERR_ARG, w + ": NULL options");
  if (o->n_rows < 0 || o->cols < 1) return tfail(RS_ERR_ARG, w + ": no columns, or a negative number of rows");
  if (o->cols > INT_MAX - 4 * kUnroll * kThreads * 8) return tfail(RS_ERR_CAPACITY, w + ": more than 2^31 columns");
  if (o->n_rows > (int64_t)INT_MAX / 64) return tfail(RS_ERR_CAPACITY, w + ": too many rows");
  if (o->top < 0 || o->top > kMaxTop) return tfail(RS_ERR_ARG, w + ": top must be in 0..32");
  if (!dtype_known(o->dtype)) return tfail(RS_ERR_ARG, w + ": unknown dtype");
  if (o->stride < 0) return tfail(RS_ERR_ARG, w + ": a negative stride");
  return RS_OK;
}

template <class T>
int launch_forward(FwdArgs a, int sms, cudaStream_t st) {
  constexpr int N = Vec16<T>::N;
  const int64_t vecs = a.cols / N + 1;
  // CTAs per row: few rows are split until two CTAs per SM are busy, while a share keeps two rounds of loads
  int cs = 1;
  while (cs < 8 && a.n * cs * 2 <= (int64_t)sms * 2 && vecs >= (int64_t)cs * 2 * kUnroll * kThreads) cs *= 2;
  size_t smem = 0;
  a.per_note = 1;
  if (a.top) {
    const int64_t its = ((vecs + cs - 1) / cs + 1 + kUnroll * kThreads - 1) / (kUnroll * kThreads);
    a.per_note = (int)((its + kNotes - 1) / kNotes);
    smem = (size_t)((its + a.per_note - 1) / a.per_note) * kThreads * sizeof(float);
    cudaError_t e = cudaFuncSetAttribute(forward_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kNotes * kThreads * (int)sizeof(float));
    if (e != cudaSuccess) return tcuda(e, "rs_token_logprobs: cudaFuncSetAttribute");
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(a.n * cs));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cs;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return tcuda(cudaLaunchKernelEx(&cfg, forward_kernel<T>, a), "rs_token_logprobs: launch");
}

int forward(const char* what, const rs_logprob_opts* o, const void* logits, const void* targets, float* logprob, float* entropy, float* lse,
            float* top_value, int64_t* top_index, float* record, int32_t device, void* stream) {
  int rc = check_opts(what, o);
  if (rc != RS_OK) return rc;
  if (o->n_rows == 0) return RS_OK;
  const std::string w(what);
  if (!logits || !targets) return tfail(RS_ERR_ARG, w + ": NULL logits or targets");
  if (!record && (!logprob || !entropy || !lse || (o->top && (!top_value || !top_index)))) return tfail(RS_ERR_ARG, w + ": NULL output");
  if ((uint64_t)logits % dtype_bytes(o->dtype) || (uint64_t)targets % (o->wide_targets ? 8 : 4))
    return tfail(RS_ERR_ARG, w + ": an address is not aligned to its elements");
  DeviceGuard guard(device);
  if (guard.err != cudaSuccess) return tcuda(guard.err, (w + ": cudaSetDevice").c_str());
  FwdArgs a{};
  a.logits = logits;
  a.n = o->n_rows;
  a.cols = o->cols;
  a.stride = o->stride;
  a.targets = targets;
  a.wide = o->wide_targets != 0;
  a.lo = o->lo;
  a.top = o->top;
  a.logprob = logprob;
  a.entropy = entropy;
  a.lse = lse;
  a.top_value = top_value;
  a.top_index = top_index;
  a.record = record;
  const int sms = sm_count(device);
  cudaStream_t st = (cudaStream_t)stream;
  if (o->dtype == RS_F32) return launch_forward<float>(a, sms, st);
  if (o->dtype == RS_BF16) return launch_forward<__nv_bfloat16>(a, sms, st);
  return launch_forward<__half>(a, sms, st);
}

}  // namespace

extern "C" {

int rs_token_logprobs(const rs_logprob_opts* opts, const void* logits_dev, const void* targets_dev, float* logprob_dev, float* entropy_dev,
                      float* lse_dev, float* top_logprob_dev, int64_t* top_index_dev, int32_t device, void* stream) {
  return guarded("rs_token_logprobs", [&]() -> int {
    return forward("rs_token_logprobs", opts, logits_dev, targets_dev, logprob_dev, entropy_dev, lse_dev, top_logprob_dev, top_index_dev,
                   nullptr, device, stream);
  });
}

int rs_token_record(const rs_logprob_opts* opts, const void* logits_dev, const void* targets_dev, float* record_dev, int32_t device,
                    void* stream) {
  return guarded("rs_token_record", [&]() -> int {
    if (opts && opts->n_rows > 0 && !record_dev) return tfail(RS_ERR_ARG, "rs_token_record: NULL record");
    return forward("rs_token_record", opts, logits_dev, targets_dev, nullptr, nullptr, nullptr, nullptr, nullptr, record_dev, device, stream);
  });
}

int rs_token_merge(const float* records_dev, const int64_t* starts, int32_t n_shards, int64_t n_rows, int32_t top, float* logprob_dev,
                   float* entropy_dev, float* lse_dev, float* top_logprob_dev, int64_t* top_index_dev, int32_t device, void* stream) {
  return guarded("rs_token_merge", [&]() -> int {
    if (n_shards < 1 || n_shards > kMaxShards || n_rows < 0 || top < 0 || top > kMaxTop)
      return tfail(RS_ERR_ARG, "rs_token_merge: a size is out of range (1..64 shards, top 0..32)");
    if (n_rows > INT_MAX) return tfail(RS_ERR_CAPACITY, "rs_token_merge: too many rows");
    if (n_rows == 0) return RS_OK;
    if (!records_dev || !starts || !logprob_dev || !entropy_dev || !lse_dev || (top && (!top_logprob_dev || !top_index_dev)))
      return tfail(RS_ERR_ARG, "rs_token_merge: NULL address");
    DeviceGuard guard(device);
    if (guard.err != cudaSuccess) return tcuda(guard.err, "rs_token_merge: cudaSetDevice");
    FwdArgs a{};
    a.n = n_rows;
    a.top = top;
    a.logprob = logprob_dev;
    a.entropy = entropy_dev;
    a.lse = lse_dev;
    a.top_value = top_logprob_dev;
    a.top_index = top_index_dev;
    Starts at{};
    for (int i = 0; i < n_shards; ++i) {
      at.lo[i] = starts[i];
      if (i && starts[i] < starts[i - 1]) return tfail(RS_ERR_ARG, "rs_token_merge: shards are not in ascending order");
    }
    merge_kernel<<<(unsigned)((n_rows + 7) / 8), kThreads, 0, (cudaStream_t)stream>>>(a, records_dev, at, n_shards);
    return tcuda(cudaGetLastError(), "rs_token_merge: launch");
  });
}

int rs_token_logprobs_grad(const rs_logprob_opts* opts, const void* logits_dev, const void* targets_dev, const float* lse_dev,
                           const float* entropy_dev, const float* grad_logprob_dev, const float* grad_entropy_dev,
                           const float* grad_lse_dev, void* grad_dev, int64_t grad_stride, int32_t device, void* stream) {
  return guarded("rs_token_logprobs_grad", [&]() -> int {
    int rc = check_opts("rs_token_logprobs_grad", opts);
    if (rc != RS_OK) return rc;
    const rs_logprob_opts& o = *opts;
    if (o.n_rows == 0) return RS_OK;
    const int b = dtype_bytes(o.dtype);
    if (!logits_dev || !targets_dev || !lse_dev || !grad_logprob_dev || !grad_dev || (grad_entropy_dev && !entropy_dev))
      return tfail(RS_ERR_ARG, "rs_token_logprobs_grad: NULL address");
    if ((uint64_t)logits_dev % b || (uint64_t)grad_dev % b || (uint64_t)targets_dev % (o.wide_targets ? 8 : 4))
      return tfail(RS_ERR_ARG, "rs_token_logprobs_grad: an address is not aligned to its elements");
    if (o.n_rows > 1 && grad_stride < o.cols) return tfail(RS_ERR_ARG, "rs_token_logprobs_grad: the gradient's rows overlap");
    BwdArgs a{};
    a.logits = logits_dev;
    a.n = o.n_rows;
    a.cols = o.cols;
    a.stride = o.stride;
    a.targets = targets_dev;
    a.wide = o.wide_targets != 0;
    a.sharded = o.sharded != 0;
    a.lo = o.lo;
    a.lse = lse_dev;
    a.entropy = entropy_dev;
    a.grad_logprob = grad_logprob_dev;
    a.grad_entropy = grad_entropy_dev;
    a.grad_lse = grad_lse_dev;
    a.out = grad_dev;
    a.out_stride = grad_stride;
    const int64_t per = (int64_t)kUnroll * kThreads * (16 / b);
    const int64_t units = (o.cols + per - 1) / per;
    if (units * o.n_rows > INT_MAX) return tfail(RS_ERR_CAPACITY, "rs_token_logprobs_grad: too many logits in one call");
    a.units = (int)units;
    // the output is the logits, lies beside them (columns of one buffer), or shares no memory with them
    const uint64_t z0 = (uint64_t)logits_dev, g0 = (uint64_t)grad_dev;
    const uint64_t z1 = z0 + ((uint64_t)(o.n_rows - 1) * o.stride + o.cols) * b, g1 = g0 + ((uint64_t)(o.n_rows - 1) * grad_stride + o.cols) * b;
    const bool same = z0 == g0 && (o.stride == grad_stride || o.n_rows == 1);
    if (!same && z0 < g1 && g0 < z1) {
      const uint64_t pitch = (uint64_t)o.stride * b, width = (uint64_t)o.cols * b;
      const uint64_t apart = pitch ? (g0 > z0 ? (g0 - z0) % pitch : (pitch - (z0 - g0) % pitch) % pitch) : 0;
      if (o.stride != grad_stride || o.n_rows == 1 || apart < width || apart + width > pitch)
        return tfail(RS_ERR_ARG, "rs_token_logprobs_grad: the gradient overlaps the logits without being them");
    }
    a.ctas = same ? 1 : (int)units;
    DeviceGuard guard(device);
    if (guard.err != cudaSuccess) return tcuda(guard.err, "rs_token_logprobs_grad: cudaSetDevice");
    cudaStream_t st = (cudaStream_t)stream;
    const unsigned grid = (unsigned)(a.ctas * o.n_rows);
    if (o.dtype == RS_F32) backward_kernel<float><<<grid, kThreads, 0, st>>>(a);
    else if (o.dtype == RS_BF16) backward_kernel<__nv_bfloat16><<<grid, kThreads, 0, st>>>(a);
    else backward_kernel<__half><<<grid, kThreads, 0, st>>>(a);
    return tcuda(cudaGetLastError(), "rs_token_logprobs_grad: launch");
  });
}

}  // extern "C"
