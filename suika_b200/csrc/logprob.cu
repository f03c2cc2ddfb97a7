// Log probabilities of given tokens, entropy and top alternatives of a vocabulary shard's logits, and
// their gradient (sm_100a).
//
// One pass over the logits keeps, per thread, the running maximum m, S = sum of e^(z - m) and
// A = sum of e^(z - m) (z - m), rescaled where m grows; then lse = m + log S and the entropy is
// log S - A / S. The differences z - m are taken first, so logits of any size (the type's lowest
// value as a mask among them) neither overflow nor lose the digits that the exponent needs. The
// top alternatives need no second pass over the row: each thread notes up to 16 maxima, of 64 bytes that it
// reads each (or of more where it reads more than 1 KB), the k-th largest maximum of 64 groups of threads is a
// bound that at least k logits reach (44 do for k = 32, fewer for less), and only the noted places that reach
// it are read again. All sums are in 32 bits.
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

constexpr int kThreads = 256;  // of the gradient and the merge
constexpr int kUnroll = 4;     // 16-byte vectors of a batch of loads, per thread
constexpr int kMaxTop = 32;
constexpr int kMaxCand = 1024; // logits kept for the exact choice
constexpr int kMaxHits = 512;  // noted places read again
constexpr int kNotes = 16;     // noted maxima per thread: 16 KB for 256 threads, so that they do not cost resident CTAs
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

// Two fp32 values in a register pair, for the packed add, multiply and fused multiply-add.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair(float x, float y) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 unpair(f32x2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 exp2_pair(f32x2 t) {
  const float2 v = unpair(t);
  return pair(exp2_fast(v.x), exp2_fast(v.y));
}

// Vectors of 16-bit logits with -inf raised to a finite value whose exponential is 0 just the same (0 * -inf
// would be NaN), two at a time; NaN stays. The value has to lie far below the row's base, and their
// difference times log2(e) must not overflow: a base beyond moderate() takes the other path.
template <class T> __device__ __forceinline__ uint4 raise_low(uint4 v) { return v; }
template <> __device__ __forceinline__ uint4 raise_low<__nv_bfloat16>(uint4 v) {
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&v);
  const __nv_bfloat162 low = __float2bfloat162_rn(-1e37f);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __hmax2_nan(h[i], low);
  return v;
}
template <> __device__ __forceinline__ uint4 raise_low<__half>(uint4 v) {
  __half2* h = reinterpret_cast<__half2*>(&v);
  const __half2 low = __float2half2_rn(-65504.f);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __hmax2_nan(h[i], low);
  return v;
}
template <class T> __device__ __forceinline__ bool moderate(float) { return false; }
template <> __device__ __forceinline__ bool moderate<__nv_bfloat16>(float base) { return fabsf(base) <= 1e36f; }
template <> __device__ __forceinline__ bool moderate<__half>(float base) { return fabsf(base) <= 60000.f; }

// A thread's running sums, two of each.
struct Sums {
  float m;
  f32x2 s, a;
};

__device__ __forceinline__ void raise_max(Sums& st, float m) {
  if (m > st.m) {
    if (st.m != -INFINITY) {  // before that the sums are 0, or NaN
      const float t = fmaxf((st.m - m) * kLog2e, -1e4f), c = exp2_fast(t);
      st.a = mul2(pair(c, c), fma2(st.s, pair(t, t), st.a));
      st.s = mul2(pair(c, c), st.s);
    }
    st.m = m;
  }
}

// One vector of logits at or below the maximum: s += e, a += e t with t = (z - m) log2(e), e = 2^t. RAISED: the
// vector went through raise_low, and no t has to be kept from -inf.
template <class T, bool RAISED>
__device__ __forceinline__ void add_vector(Sums& st, float base, uint4 v) {
  constexpr int N = Vec16<T>::N;
  const f32x2 minus = pair(-base, -base), scale = pair(kLog2e, kLog2e);
  float f[N];
  unpack16<T>(RAISED ? raise_low<T>(v) : v, f);
#pragma unroll
  for (int q = 0; q < N; q += 2) {
    const f32x2 t = mul2(add2(pair(f[q], f[q + 1]), minus), scale);
    const f32x2 e = exp2_pair(t);
    st.s = add2(st.s, e);
    if (RAISED) {
      st.a = fma2(e, t, st.a);
    } else {
      const float2 u = unpair(t);
      st.a = fma2(e, pair(fmaxf(u.x, -1e4f), fmaxf(u.y, -1e4f)), st.a);
    }
  }
}
__device__ __forceinline__ void add_logit(Sums& st, float z) {
  const float t = (z - base_of(st.m)) * kLog2e, e = exp2_fast(t);
  st.s = add2(st.s, pair(e, 0.f));
  st.a = fma2(pair(e, 0.f), pair(fmaxf(t, -1e4f), 0.f), st.a);
}
__device__ __forceinline__ Stat total(const Sums& st) {
  const float2 s = unpair(st.s), a = unpair(st.a);
  return Stat{st.m, s.x + s.y, a.x + a.y};
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
  int index_base;  // added to the indices of a record
  int per_note;    // iterations that share a note
  float* logprob;  // null: write records
  float* entropy;
  float* lse;
  float* top_value;
  int64_t* top_index;
  float* record;   // [n][4 + 2 top]: m, S, A, target's logit (+inf: not here; one that is +inf: NaN), values, indices as bits
};

// What one row ends as. S = 0: every logit is -inf. Nothing is possible there: lse and every log
// probability are -inf, the entropy 0.
__device__ __forceinline__ void finish_row(const FwdArgs& a, int64_t row, const Stat& st, float target) {
  const float b = base_of(st.m);
  const bool empty = st.s == 0.f;
  const float log_s = logf(st.s);
  const float lse = empty ? -INFINITY : b + log_s;
  // target - m first: both are logits, their difference is small where it matters
  const float lp = target == INFINITY ? 0.f : empty ? -INFINITY : (target - b) - log_s;
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
  for (int c = threadIdx.x; c < count; c += blockDim.x) {
    const uint64_t mine = cand[c];
    int r = 0;
#pragma unroll 8
    for (int d = 0; d < count; ++d) r += cand[d] > mine;
    if (r < k) best[r] = mine;
  }
}

// A CTA's share of a row: whole 16-byte vectors [v0, v1) from `body`. The logits before the row's first 16-byte
// border and after its last whole vector (at most 14) go to one thread each of the row's first CTA.
template <class T>
struct Share {
  const T* z;
  const uint4* body;
  int head, vecs, v0, v1, loose;
  __device__ __forceinline__ Share(const FwdArgs& a, int64_t row, int part, int cs) {
    constexpr int N = Vec16<T>::N;
    const int cols = (int)a.cols;
    z = reinterpret_cast<const T*>(a.logits) + row * a.stride;
    head = min(cols, (int)((16 - ((uintptr_t)z & 15)) & 15) / (int)sizeof(T));
    vecs = (cols - head) / N;
    v0 = (int)((int64_t)vecs * part / cs);
    v1 = (int)((int64_t)vecs * (part + 1) / cs);
    body = reinterpret_cast<const uint4*>(z + head);
    loose = part == 0 ? cols - vecs * N : 0;
  }
  __device__ __forceinline__ int loose_at(int t) const { return t < head ? t : t + vecs * Vec16<T>::N; }
};

// A cluster of cs CTAs per row. (Persistent CTAs that load the next row's first vectors while they finish one
// need the registers of a third of the warps: 4096 rows of 152064 bf16 logits took 244 us instead of 206.)
template <class T, int THREADS>
__global__ void __launch_bounds__(THREADS) forward_kernel(FwdArgs a, int cs) {
  constexpr int N = Vec16<T>::N, WARPS = THREADS / 32;
  extern __shared__ float notes[];  // [kNotes][THREADS] where alternatives are asked for
  __shared__ float warp_max[WARPS], lane_max[WARPS][32];
  __shared__ float2 warp_sum[WARPS];
  __shared__ uint64_t cand[kMaxCand];
  __shared__ uint64_t best[kMaxTop];
  __shared__ Stat cta_stat;
  __shared__ float bound;
  __shared__ float group_max[64];
  __shared__ int n_cand, n_hits, step_sum[WARPS];
  __shared__ int hits[kMaxHits];
  cg::cluster_group cluster = cg::this_cluster();
  const int part = cs > 1 ? (int)cluster.block_rank() : 0;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, k = a.top;
  const int64_t row = blockIdx.x / cs;
  const Share<T> sh(a, row, part, cs);
  // the target's logit, read now and used at the end
  float target = INFINITY;
  if (tid == 0) {
    const int64_t at = load_target(a.targets, a.wide, row) - a.lo;
    if (at >= 0 && at < a.cols) {
      target = to_f32<T>(sh.z[at]);
      if (target == INFINITY) target = NAN;  // +inf says that there is no target; in such a row the log probability is NaN
    }
  }
  const float loose_z = tid < sh.loose ? to_f32<T>(sh.z[sh.loose_at(tid)]) : -INFINITY;

  Sums st{-INFINITY, 0, 0};
  int note = 0, in_note = 0;
  float noted = -INFINITY;
  for (int v = sh.v0 + tid; v < sh.v1; v += kUnroll * THREADS) {
    uint4 x[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (v + u * THREADS < sh.v1) x[u] = ld16(sh.body + v + u * THREADS);
    float mx = -INFINITY;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (v + u * THREADS < sh.v1) mx = fmaxf(mx, max_of<T>(x[u]));
    raise_max(st, mx);
    const float base = base_of(st.m);
    if (sizeof(T) == 4 || moderate<T>(base)) {  // one branch per batch: one per vector cost a third of the rate
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (v + u * THREADS < sh.v1) add_vector<T, sizeof(T) == 2>(st, base, x[u]);
    } else {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (v + u * THREADS < sh.v1) add_vector<T, false>(st, base, x[u]);
    }
    if (k) {
      noted = fmaxf(noted, mx);
      if (++in_note == a.per_note) {
        notes[note * THREADS + tid] = noted;
        ++note;
        in_note = 0;
        noted = -INFINITY;
      }
    }
  }
  // every thread has a note for each of the CTA's batches, -inf past its last vector
  const int batches = (sh.v1 - sh.v0 + kUnroll * THREADS - 1) / (kUnroll * THREADS);
  const int notes_of_cta = (batches + a.per_note - 1) / a.per_note;
  if (k && in_note) notes[note++ * THREADS + tid] = noted;
  if (k && note < notes_of_cta) notes[note * THREADS + tid] = -INFINITY;
  if (tid < sh.loose) {
    raise_max(st, loose_z);
    add_logit(st, loose_z);
  }

  // the CTA's maximum first, then sums that are already relative to it
  float m = st.m;
#pragma unroll
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
  if (lane == 0) warp_max[w] = m;
  if (k) lane_max[w][lane] = st.m;
  if (tid == 0) n_cand = n_hits = 0;
  if (tid < kMaxTop) best[tid] = kNoKey;
  __syncthreads();
  m = warp_max[0];
#pragma unroll
  for (int q = 1; q < WARPS; ++q) m = fmaxf(m, warp_max[q]);
  {
    raise_max(st, m);
    Stat mine = total(st);
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      mine.s += __shfl_xor_sync(~0u, mine.s, o);
      mine.a += __shfl_xor_sync(~0u, mine.a, o);
    }
    if (lane == 0) warp_sum[w] = make_float2(mine.s, mine.a);
  }
  if (k && tid < 64) {  // threads t and t + 64 j form a group: its maximum
    float y = -INFINITY;
#pragma unroll
    for (int r = tid >> 5; r < WARPS; r += 2) y = fmaxf(y, lane_max[r][lane]);
    group_max[tid] = y;
  }
  __syncthreads();
  Stat t{m, warp_sum[0].x, warp_sum[0].y};
#pragma unroll
  for (int q = 1; q < WARPS; ++q) {
    t.s += warp_sum[q].x;
    t.a += warp_sum[q].y;
  }

  if (k) {
    if (tid < 64) {  // the k-th largest of the groups' maxima: k logits at least are as large
      const float y = group_max[tid];
      int rank = 0;
#pragma unroll 16
      for (int o = 0; o < 64; ++o) rank += before(group_max[o], o, y, tid);
      if (rank == k - 1) bound = y;
    }
    __syncthreads();
    const float least = bound;
    // Collects the logits from `least` on (strict: above it) from the noted places, one vector of them
    // per thread: one latency for all. Their order does not matter, they are ranked by value and index.
    auto collect = [&](bool strict) {
      auto wanted = [&](float f) { return strict ? f > least : f >= least; };
      auto offer = [&](float f, int i) {
        if (wanted(f)) {
          const int at = atomicAdd(&n_cand, 1);
          if (at < kMaxCand) cand[at] = rank_key(f, i);
        }
      };
      for (int s = 0; s < notes_of_cta; ++s)
        if (wanted(notes[s * THREADS + tid])) {
          const int at = atomicAdd(&n_hits, 1);
          if (at < kMaxHits) hits[at] = s * THREADS + tid;
        }
      __syncthreads();
      const int found = min(n_hits, kMaxHits), per_hit = a.per_note * kUnroll;
      for (int i = tid; i < found * per_hit; i += THREADS) {
        const int hit = hits[i / per_hit], s = hit / THREADS;
        const int v = sh.v0 + (hit - s * THREADS) + (s * per_hit + i % per_hit) * THREADS;
        if (v < sh.v1) {
          float f[N];
          unpack16<T>(ld16(sh.body + v), f);
#pragma unroll
          for (int e = 0; e < N; ++e) offer(f[e], sh.head + v * N + e);
        }
      }
      if (tid < sh.loose) offer(loose_z, sh.loose_at(tid));
      __syncthreads();
      return n_hits <= kMaxHits && n_cand <= kMaxCand;
    };
    if (collect(false)) {
      place_candidates(cand, n_cand, k, best);
    } else {
      // Very many logits equal the bound (a masked or nearly constant row): those above it, then the first
      // ones, in the order of the row, that equal it.
      __syncthreads();
      if (tid == 0) n_cand = n_hits = 0;
      __syncthreads();
      if (collect(true)) {
        const int above = n_cand;
        place_candidates(cand, above, k, best);
        int placed = min(above, k);
        // one step: each thread has up to N logits, in the order of the threads
        auto step = [&](const float* f, int n, int at) {
          int equal = 0;
          for (int e = 0; e < n; ++e) equal += f[e] == least;
          int before_me = equal;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(~0u, before_me, o);
            if (lane >= o) before_me += y;
          }
          if (lane == 31) step_sum[w] = before_me;
          __syncthreads();
          int slot = placed + before_me - equal;
          for (int q = 0; q < WARPS; ++q) {
            if (q < w) slot += step_sum[q];
            placed += step_sum[q];
          }
          for (int e = 0; e < n; ++e)
            if (f[e] == least) {
              if (slot < k) best[slot] = rank_key(f[e], at + e);
              ++slot;
            }
          __syncthreads();
        };
        float f[N];
        f[0] = loose_z;
        if (part == 0 && placed < k) step(f, tid < min(sh.loose, sh.head) ? 1 : 0, tid);
        for (int v = sh.v0; v < sh.v1 && placed < k; v += THREADS) {
          const bool mine = v + tid < sh.v1;
          if (mine) unpack16<T>(ld16(sh.body + v + tid), f);
          step(f, mine ? N : 0, sh.head + (v + tid) * N);
        }
        f[0] = loose_z;
        if (part == 0 && placed < k) step(f, tid >= sh.head && tid < sh.loose ? 1 : 0, sh.loose_at(tid));
      } else {
        // Large logits at a period that puts them all into a few groups: k searches for the first logit after
        // the last one chosen.
        uint64_t chosen = ~0ull;
        for (int r = 0; r < k; ++r) {
          uint64_t top = kNoKey;
          auto look = [&](float f, int i) {
            const uint64_t key = rank_key(f, i);
            if (!isnan(f) && key < chosen && key > top) top = key;
          };
          for (int v = sh.v0 + tid; v < sh.v1; v += THREADS) {
            float f[N];
            unpack16<T>(ld16(sh.body + v), f);
#pragma unroll
            for (int e = 0; e < N; ++e) look(f[e], sh.head + v * N + e);
          }
          if (tid < sh.loose) look(loose_z, sh.loose_at(tid));
#pragma unroll
          for (int o = 16; o; o >>= 1) {
            const uint64_t other = __shfl_xor_sync(~0u, top, o);
            if (other > top) top = other;
          }
          __syncthreads();  // the last round's reads of cand are over
          if (lane == 0) cand[w] = top;
          __syncthreads();
          for (int q = 0; q < WARPS; ++q)
            if (cand[q] > top) top = cand[q];
          if (tid == 0) best[r] = top;
          chosen = top;
        }
      }
    }
  }

  // join the CTAs of the row
  if (cs > 1) {
    if (tid == 0) cta_stat = t;
    cluster.sync();
    if (part == 0) {
      for (int c = 1; c < cs; ++c) t = join(t, *cluster.map_shared_rank(&cta_stat, c));
      if (k) {
        for (int i = tid; i < cs * k; i += THREADS) {
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
  } else if (k) {
    __syncthreads();
  }

  if (tid == 0) {
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
      r[k + tid] = __int_as_float(none ? -1 : a.index_base + i);
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
  bool sharded;  // one of several shards: a target outside [lo, lo + cols) may be another's
  int64_t lo;
  int64_t first, end;  // the whole vocabulary: a target outside it is none
  const float* lse;
  const float* entropy;
  const float* grad_logprob;
  const float* grad_entropy;  // null: none
  const float* grad_lse;      // null: none
  void* out;
  int64_t out_stride;
  int units;  // pieces of kUnroll * kThreads vectors in a row
  int ctas;   // CTAs per row; one where the output is the logits (a row that is read again is then read before it is written)
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
  const int64_t index = load_target(a.targets, a.wide, row), target = index - a.lo;
  const float lse = a.lse[row];
  const float h = a.entropy ? a.entropy[row] : 0.f, gh = a.grad_entropy ? a.grad_entropy[row] : 0.f;
  const int target_col = target >= 0 && target < a.cols ? (int)target : -1;
  const bool ignored = index < a.first || index >= a.end;
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
    Sums far{-INFINITY, 0, 0};
    for (int j = threadIdx.x; j < cols; j += kThreads) {
      const float f = to_f32<T>(z[j]);
      raise_max(far, f);
      add_logit(far, f);
    }
    Stat st = warp_join(total(far));
    __shared__ Stat part[8];
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = st;
    __syncthreads();  // every thread has read the row
    st = part[0];
    for (int q = 1; q < 8; ++q) st = join(st, part[q]);
    base = st.m;
    rest = logf(st.s);
  }
  // with t = log2 p: gradient = wd (p t) + w0 p, and g_lp more at the target. p is multiplied first: where it is 0 the
  // products are 0 whatever wd is, while wd t overflows for a masked logit's t (-1e37; |wd| > 34) and 0 * inf is NaN.
  // Taking t instead of log p makes up for the third product (4096 rows of 32000 bf16: 88.1 us, 90.1 with log p).
  const float wd = -gh * kLn2, w0 = -fmaf(gh, h, gp);
  const bool raised = moderate<T>(base);
  const f32x2 minus = pair(-base, -base), scale = pair(kLog2e, kLog2e), less = pair(-rest * kLog2e, -rest * kLog2e), wd2 = pair(wd, wd), w02 = pair(w0, w0);
  auto two = [&](float x, float y) {
    f32x2 t = fma2(add2(pair(x, y), minus), scale, less);
    const f32x2 p = exp2_pair(t);
    if (!raised) {  // p is 0 below; -inf * 0 would be NaN
      const float2 u = unpair(t);
      t = pair(fmaxf(u.x, -1e4f), fmaxf(u.y, -1e4f));
    }
    return unpair(fma2(wd2, mul2(p, t), mul2(w02, p)));
  };
  const int per = kUnroll * kThreads;
  const uint4* src = reinterpret_cast<const uint4*>(z + head);
  uint4* dst = reinterpret_cast<uint4*>(out + head);
  // the next piece is loaded before this one is worked on
  uint4 x[kUnroll];
  auto load = [&](int unit) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int q = unit * per + threadIdx.x + u * kThreads;
      if (!none && q < vecs) x[u] = ld16(src + q);
    }
  };
  load(first);
  for (int unit = first; unit < a.units; unit += a.ctas) {
    uint4 now[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) now[u] = x[u];
    load(unit + a.ctas);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int q = unit * per + threadIdx.x + u * kThreads;
      if (q >= vecs) break;
      float f[N];
      if (!none) {
        unpack16<T>(raised ? raise_low<T>(now[u]) : now[u], f);
#pragma unroll
        for (int e = 0; e < N; e += 2) {
          const float2 g = two(f[e], f[e + 1]);
          f[e] = g.x;
          f[e + 1] = g.y;
        }
        const int at = target_col - (head + q * N);
        if (at >= 0 && at < N) {
#pragma unroll
          for (int e = 0; e < N; ++e)
            if (e == at) f[e] += gl;
        }
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
    float f = none ? 0.f : to_f32<T>(z[j]);
    if (raised) f = fmaxf(f, -1e37f) + (isnan(f) ? f : 0.f);
    out[j] = from_f32<T>(none ? 0.f : two(f, 0.f).x + (j == target_col ? gl : 0.f));
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

template <class T, int THREADS>
int launch_forward_as(FwdArgs a, int cs, cudaStream_t st) {
  constexpr int N = Vec16<T>::N;
  const int64_t vecs = a.cols / N + 1;
  size_t smem = 0;
  a.per_note = 1;
  if (a.top) {
    const int64_t its = ((vecs + cs - 1) / cs + 1 + kUnroll * THREADS - 1) / (kUnroll * THREADS);
    a.per_note = (int)((its + kNotes - 1) / kNotes);
    smem = (size_t)((its + a.per_note - 1) / a.per_note) * THREADS * sizeof(float);
    static_assert(kNotes * THREADS * 4 + kMaxCand * 8 + kMaxHits * 4 + 4096 <= 48 * 1024, "the notes and the static arrays need no opt-in");
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(a.n * cs));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cs;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = cs > 1;  // without the attribute many short rows start faster (8192 of 1000 fp32: 17.5 us against 20.4)
  return tcuda(cudaLaunchKernelEx(&cfg, forward_kernel<T, THREADS>, a, cs), "rs_token_logprobs: launch");
}

// Few rows are split over a cluster of up to 8 CTAs: until two CTAs per SM are busy, while a share keeps 960
// vectors (15 KB; below that the join costs more than it saves), or, where shares stay above 64 KB, until five
// are (300 rows of 152064 fp32 logits: 29 us, 42 in one CTA each). Shares of few rows take 512 threads (3
// such rows: 10.2 us against 11.5 with 256), many short rows 128 (4096 rows of 1000: 12.2 us against 16.4), whose
// other threads would idle.
template <class T>
int launch_forward(const FwdArgs& a, int sms, cudaStream_t st) {
  const int64_t vecs = a.cols / Vec16<T>::N + 1;
  int cs = 1;
  while (cs < 8 && ((a.n * cs * 2 <= (int64_t)sms * 2 && vecs >= (int64_t)cs * 2 * 960) ||
                    (a.n * cs * 2 <= (int64_t)sms * 5 && vecs >= (int64_t)cs * 2 * 4096)))
    cs *= 2;
  if (a.n * cs <= (int64_t)sms * 2 && vecs / cs >= 900) return launch_forward_as<T, 512>(a, cs, st);
  if (vecs / cs <= 2048 && a.n > (int64_t)sms * 2) return launch_forward_as<T, 128>(a, cs, st);
  return launch_forward_as<T, 256>(a, cs, st);
}

int forward(const char* what, const rs_logprob_opts* o, const void* logits, const void* targets, float* logprob, float* entropy, float* lse,
            float* top_value, int64_t* top_index, float* record, int index_base, int32_t device, void* stream) {
  int rc = check_opts(what, o);
  if (rc != RS_OK) return rc;
  if (o->n_rows == 0) return RS_OK;
  const std::string w(what);
  if (!logits || !targets) return tfail(RS_ERR_ARG, w + ": NULL logits or targets");
  if (!record && (!logprob || !entropy || !lse || (o->top && (!top_value || !top_index)))) return tfail(RS_ERR_ARG, w + ": NULL output");
  if (misaligned(dtype_bytes(o->dtype), logits) || misaligned(o->wide_targets ? 8 : 4, targets) ||
      misaligned(4, logprob, entropy, lse, top_value, record) || misaligned(8, top_index))
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
  a.index_base = index_base;
  const int sms = sm_count(device);
  cudaStream_t st = (cudaStream_t)stream;
  if (o->dtype == RS_F32) return launch_forward<float>(a, sms, st);
  if (o->dtype == RS_BF16) return launch_forward<__nv_bfloat16>(a, sms, st);
  return launch_forward<__half>(a, sms, st);
}

// [first, end): the whole vocabulary, whose targets have a gradient.
int backward(const char* what, const rs_logprob_opts* opts, int64_t first, int64_t end, const void* logits, const void* targets, const float* lse,
             const float* entropy, const float* grad_logprob, const float* grad_entropy, const float* grad_lse, void* grad,
             int64_t grad_stride, int32_t device, void* stream) {
  int rc = check_opts(what, opts);
  if (rc != RS_OK) return rc;
  const rs_logprob_opts& o = *opts;
  const std::string w(what);
  if (o.n_rows == 0) return RS_OK;
  const int b = dtype_bytes(o.dtype);
  if (!logits || !targets || !lse || !grad_logprob || !grad || (grad_entropy && !entropy))
    return tfail(RS_ERR_ARG, w + ": NULL address");
  if (misaligned(b, logits, grad) || misaligned(o.wide_targets ? 8 : 4, targets) ||
      misaligned(4, lse, entropy, grad_logprob, grad_entropy, grad_lse))
    return tfail(RS_ERR_ARG, w + ": an address is not aligned to its elements");
  if (o.n_rows > 1 && grad_stride < o.cols) return tfail(RS_ERR_ARG, w + ": the gradient's rows overlap");
  BwdArgs a{};
  a.logits = logits;
  a.n = o.n_rows;
  a.cols = o.cols;
  a.stride = o.stride;
  a.targets = targets;
  a.wide = o.wide_targets != 0;
  a.sharded = o.sharded != 0;
  a.lo = o.lo;
  a.first = first;
  a.end = end;
  a.lse = lse;
  a.entropy = entropy;
  a.grad_logprob = grad_logprob;
  a.grad_entropy = grad_entropy;
  a.grad_lse = grad_lse;
  a.out = grad;
  a.out_stride = grad_stride;
  const int64_t per = (int64_t)kUnroll * kThreads * (16 / b);
  const int64_t units = (o.cols + per - 1) / per;
  if (units * o.n_rows > INT_MAX) return tfail(RS_ERR_CAPACITY, w + ": too many logits in one call");
  a.units = (int)units;
  // the output is the logits, lies beside them (columns of one buffer), or shares no memory with them
  const uint64_t z0 = (uint64_t)logits, g0 = (uint64_t)grad;
  const uint64_t z1 = z0 + ((uint64_t)(o.n_rows - 1) * o.stride + o.cols) * b, g1 = g0 + ((uint64_t)(o.n_rows - 1) * grad_stride + o.cols) * b;
  const bool same = z0 == g0 && (o.stride == grad_stride || o.n_rows == 1);
  if (!same && z0 < g1 && g0 < z1) {
    const uint64_t pitch = (uint64_t)o.stride * b, width = (uint64_t)o.cols * b;
    const uint64_t apart = pitch ? (g0 > z0 ? (g0 - z0) % pitch : (pitch - (z0 - g0) % pitch) % pitch) : 0;
    if (o.stride != grad_stride || o.n_rows == 1 || apart < width || apart + width > pitch)
      return tfail(RS_ERR_ARG, w + ": the gradient overlaps the logits without being them");
  }
  // up to four pieces per CTA, as long as sixteen CTAs per SM are left
  const int64_t pieces = std::min<int64_t>(4, std::max<int64_t>(1, units * o.n_rows / ((int64_t)sm_count(device) * 16)));
  a.ctas = same ? 1 : (int)((units + pieces - 1) / pieces);
  DeviceGuard guard(device);
  if (guard.err != cudaSuccess) return tcuda(guard.err, (w + ": cudaSetDevice").c_str());
  cudaStream_t st = (cudaStream_t)stream;
  const unsigned grid = (unsigned)(a.ctas * o.n_rows);
  if (o.dtype == RS_F32) backward_kernel<float><<<grid, kThreads, 0, st>>>(a);
  else if (o.dtype == RS_BF16) backward_kernel<__nv_bfloat16><<<grid, kThreads, 0, st>>>(a);
  else backward_kernel<__half><<<grid, kThreads, 0, st>>>(a);
  return tcuda(cudaGetLastError(), (w + ": launch").c_str());
}

}  // namespace

extern "C" {

int rs_token_logprobs(const rs_logprob_opts* opts, const void* logits_dev, const void* targets_dev, float* logprob_dev, float* entropy_dev,
                      float* lse_dev, float* top_logprob_dev, int64_t* top_index_dev, int32_t device, void* stream) {
  return guarded("rs_token_logprobs", [&]() -> int {
    return forward("rs_token_logprobs", opts, logits_dev, targets_dev, logprob_dev, entropy_dev, lse_dev, top_logprob_dev, top_index_dev,
                   nullptr, 0, device, stream);
  });
}

int rs_token_record(const rs_logprob_opts* opts, const void* logits_dev, const void* targets_dev, float* record_dev, int32_t device,
                    void* stream) {
  return guarded("rs_token_record", [&]() -> int {
    if (opts && opts->n_rows > 0 && !record_dev) return tfail(RS_ERR_ARG, "rs_token_record: NULL record");
    return forward("rs_token_record", opts, logits_dev, targets_dev, nullptr, nullptr, nullptr, nullptr, nullptr, record_dev, 0, device, stream);
  });
}

int rs_token_record_at(const rs_logprob_opts* opts, int64_t index_base, const void* logits_dev, const void* targets_dev, float* record_dev,
                       int32_t device, void* stream) {
  return guarded("rs_token_record_at", [&]() -> int {
    if (opts && opts->n_rows > 0 && !record_dev) return tfail(RS_ERR_ARG, "rs_token_record_at: NULL record");
    if (index_base < 0) return tfail(RS_ERR_ARG, "rs_token_record_at: a negative index");
    if (opts && (index_base > INT_MAX || opts->cols > INT_MAX - index_base))
      return tfail(RS_ERR_CAPACITY, "rs_token_record_at: indices past 31 bits");
    return forward("rs_token_record_at", opts, logits_dev, targets_dev, nullptr, nullptr, nullptr, nullptr, nullptr, record_dev, (int)index_base,
                   device, stream);
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
    if (misaligned(4, records_dev, logprob_dev, entropy_dev, lse_dev, top_logprob_dev) || misaligned(8, top_index_dev))
      return tfail(RS_ERR_ARG, "rs_token_merge: an address is not aligned to its elements");
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
    const bool whole = opts && !opts->sharded;
    return backward("rs_token_logprobs_grad", opts, whole ? opts->lo : 0, whole ? opts->lo + opts->cols : INT64_MAX, logits_dev, targets_dev,
                    lse_dev, entropy_dev, grad_logprob_dev, grad_entropy_dev, grad_lse_dev, grad_dev, grad_stride, device, stream);
  });
}

int rs_token_logprobs_shard_grad(const rs_logprob_opts* opts, int64_t vocab_first, int64_t vocab_end, const void* logits_dev,
                                 const void* targets_dev, const float* lse_dev, const float* entropy_dev, const float* grad_logprob_dev,
                                 const float* grad_entropy_dev, const float* grad_lse_dev, void* grad_dev, int64_t grad_stride,
                                 int32_t device, void* stream) {
  return guarded("rs_token_logprobs_shard_grad", [&]() -> int {
    if (!opts || !opts->sharded) return tfail(RS_ERR_ARG, "rs_token_logprobs_shard_grad: the options of a sharded gradient are taken");
    if (opts->lo < vocab_first || opts->cols > vocab_end - opts->lo)
      return tfail(RS_ERR_ARG, "rs_token_logprobs_shard_grad: the shard leaves the vocabulary");
    return backward("rs_token_logprobs_shard_grad", opts, vocab_first, vocab_end, logits_dev, targets_dev, lse_dev, entropy_dev,
                    grad_logprob_dev, grad_entropy_dev, grad_lse_dev, grad_dev, grad_stride, device, stream);
  });
}

}  // extern "C"
