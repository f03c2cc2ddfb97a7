// Global gradient norm, clipping and the AdamW update of a rank's training state (sm_100a).
//
// All three walk a table of tensors, like the copy kernels: a tensor is cut into tiles, the tile list is
// implicit (tile_begin per entry, binary-searched by a CTA). The update and the scaling launch a CTA per
// tile: short-lived CTAs keep to no lockstep, while persistent ones (4 per SM, round-robin) all read at the same
// place of their tiles, and the update's 7 streams then ran at 5.04 TB/s instead of 6.83 (840M elements with
// fp32 gradients). The table travels in the kernel's parameters, not in
// device memory, so a call uploads nothing, can be captured, and holds no address after it
// returns. Every pass reads each element once and writes it at most once; nothing here needs tensor
// cores, and HBM is the bound once a few MB are moved. Below that the launches are.
#include "train.cuh"

#include <cooperative_groups.h>

#include <algorithm>
#include <utility>
#include <vector>

namespace cg = cooperative_groups;

namespace {

using namespace suika_train;

constexpr int kThreads = 256;
constexpr int kSmallThreads = 1024, kSmallCtas = 8;  // the cluster that sums up to kSmallBytes
constexpr uint64_t kSmallBytes = 1 << 20;

struct SpanEnt {
  uint64_t ptr;
  uint64_t numel;
  uint32_t tile_begin;
  uint32_t dtype;
};

// Kernel parameters are copied at each launch whatever their use, so a short table takes a short
// parameter block: capacities 24, 160 and 1280 entries (30.8 KB of the 32,764 bytes allowed).
template <int CAP>
struct SpanTable {
  SpanEnt e[CAP];
  int32_t n;
  uint32_t n_tiles;
  uint32_t tile_bytes;
};

// Stores of results that this step does not read again: evict-first (2 % on the update, 4 % on the scaling).
__device__ __forceinline__ void st16_stream(void* p, uint4 v) {
  asm volatile("st.global.cs.v4.u32 [%0], {%1,%2,%3,%4};" :: "l"(p), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

template <class Ent>
__device__ __forceinline__ int find_entry(const Ent* e, int n, uint32_t tile) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    int mid = (lo + hi + 1) >> 1;
    if (e[mid].tile_begin <= tile) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ float load_scalar(uint64_t base, uint64_t i, uint32_t dtype) {
  if (dtype == RS_F32) return reinterpret_cast<const float*>(base)[i];
  if (dtype == RS_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(base)[i]);
  return __half2float(reinterpret_cast<const __half*>(base)[i]);
}
__device__ __forceinline__ void store_scalar(uint64_t base, uint64_t i, uint32_t dtype, float x) {
  if (dtype == RS_F32) reinterpret_cast<float*>(base)[i] = x;
  else if (dtype == RS_BF16) reinterpret_cast<__nv_bfloat16*>(base)[i] = __float2bfloat16_rn(x);
  else reinterpret_cast<__half*>(base)[i] = __float2half_rn(x);
}

// The values of a 16-byte vector; returns how many there are, 4 or 8.
__device__ __forceinline__ int decode_vec(uint4 v, uint32_t dtype, float* x) {
  if (dtype == RS_F32) { unpack16<float>(v, x); return 4; }
  if (dtype == RS_BF16) unpack16<__nv_bfloat16>(v, x); else unpack16<__half>(v, x);
  return 8;
}

// ---- norm ---------------------------------------------------------------------------------

// Sum of squares of one batch of vectors. Squares and their short sum are in 32 bits; a batch whose
// sum leaves [1e-30, 1e37] (values whose square overflows or goes under in 32 bits, and NaN or
// infinity) is taken again in 64 bits. Batches are added in 64 bits, so the length does not matter.
template <int U>
__device__ __forceinline__ double batch_sumsq(const uint4* v, uint32_t dtype) {
  float s = 0.f;
  float x[8];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    int n = decode_vec(v[u], dtype, x);
    float a = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) a = fmaf(x[k], x[k], a);
    if (n == 8) {
#pragma unroll
      for (int k = 4; k < 8; ++k) a = fmaf(x[k], x[k], a);
    }
    s += a;
  }
  if (s >= 1e-30f && s <= 1e37f) return (double)s;
  double d = 0.0;
#pragma unroll 1
  for (int u = 0; u < U; ++u) {
    uint4 w = u == 0 ? v[0] : u == 1 ? v[U > 1 ? 1 : 0] : u == 2 ? v[U > 2 ? 2 : 0] : v[U > 3 ? 3 : 0];
    int n = decode_vec(w, dtype, x);
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < n) d = fma((double)x[k], (double)x[k], d);
  }
  return d;
}

__device__ __forceinline__ double block_sum(double x) {
  __shared__ double part[32];
#pragma unroll
  for (int o = 16; o; o >>= 1) x += __shfl_down_sync(~0u, x, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = x;
  __syncthreads();
  if (threadIdx.x < 32) {
    x = threadIdx.x < (blockDim.x >> 5) ? part[threadIdx.x] : 0.0;
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_down_sync(~0u, x, o);
  }
  return x;  // thread 0's is the sum
}

// The sum over one CTA's tiles, as thread 0's result.
template <int CAP>
__device__ __forceinline__ double tiles_sumsq(const SpanTable<CAP>& t, uint32_t first, uint32_t apart) {
  double acc = 0.0;
  for (uint32_t tile = first; tile < t.n_tiles; tile += apart) {
    const SpanEnt& e = t.e[find_entry(t.e, t.n, tile)];
    const uint32_t dt = e.dtype, isz = dt == RS_F32 ? 4 : 2, per = 16 / isz, most = t.tile_bytes / isz;
    const uint64_t off = (uint64_t)(tile - e.tile_begin) * most;
    const uint32_t len = (uint32_t)min((uint64_t)most, e.numel - off);
    const uint64_t p = e.ptr + off * isz;
    const uint32_t head = min(len, (uint32_t)((16 - (p & 15)) & 15) / isz);
    const uint32_t nvec = (len - head) / per;
    const char* body = reinterpret_cast<const char*>(p + (uint64_t)head * isz);
    for (uint32_t i = threadIdx.x; i < nvec; i += 4 * blockDim.x) {
      uint4 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint32_t j = i + u * blockDim.x;
        v[u] = j < nvec ? ld16(body + (size_t)j * 16) : make_uint4(0, 0, 0, 0);
      }
      acc += batch_sumsq<4>(v, dt);
    }
    const uint32_t loose = len - nvec * per;  // head, then what follows the last whole vector
    if (threadIdx.x < loose) {
      const uint32_t i = threadIdx.x < head ? threadIdx.x : threadIdx.x + nvec * per;
      const double x = (double)load_scalar(p, i, dt);
      acc = fma(x, x, acc);
    }
  }
  return block_sum(acc);
}

// One partial sum per CTA. The tiles of a CTA depend on the table and the grid alone and every sum
// has a fixed order, so the same inputs give the same bits.
template <int CAP>
__global__ void __launch_bounds__(kThreads) sumsq_kernel(const __grid_constant__ SpanTable<CAP> t, double* partial) {
  let_successor_start();
  const double acc = tiles_sumsq(t, blockIdx.x, gridDim.x);
  if (threadIdx.x == 0) partial[blockIdx.x] = acc;
}

// Up to 1 MB: one cluster, whose first CTA adds the others' sums from their shared memory. A launch less than
// partial sums in memory take: a call of 0.9 MB is 8.7 us of host time against 11.5, and 6.1 us on the device
// against 5. (At 3 MB its 8 CTAs need 13 us, the two launches 5.)
template <int CAP>
__global__ void __launch_bounds__(kSmallThreads) sumsq_small_kernel(const __grid_constant__ SpanTable<CAP> t, double* sumsq) {
  __shared__ double sums[kSmallCtas];
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();  // the first CTA runs before its memory is written
  const double acc = tiles_sumsq(t, blockIdx.x, kSmallCtas);
  if (threadIdx.x == 0) cluster.map_shared_rank(sums, 0)[blockIdx.x] = acc;
  cluster.sync();
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    double total = 0.0;
    for (int i = 0; i < kSmallCtas; ++i) total += sums[i];
    *sumsq = total;
  }
}

constexpr int kFinishThreads = 1024;
__global__ void __launch_bounds__(kFinishThreads) sumsq_finish_kernel(const double* partial, int n, double* sumsq) {
  after_predecessor();
  double acc = 0.0;
  for (int i = threadIdx.x; i < n; i += kFinishThreads) acc += partial[i];
  acc = block_sum(acc);
  if (threadIdx.x == 0) *sumsq = acc;
}

// ---- clipping -----------------------------------------------------------------------------

// min(1, max_norm / (norm + 1e-6)) in 32 bits; a NaN norm stays NaN and so reaches the gradients.
__device__ __forceinline__ float clip_factor(double sumsq, float max_norm, float* norm) {
  *norm = (float)sqrt(sumsq);
  const float c = max_norm / (*norm + 1e-6f);
  return c >= 1.f ? 1.f : c;
}

template <int CAP>
__global__ void __launch_bounds__(kThreads) scale_kernel(const __grid_constant__ SpanTable<CAP> t, const double* sumsq,
                                                         float max_norm, float* norm_out) {
  after_predecessor();
  float norm;
  const float c = clip_factor(*sumsq, max_norm, &norm);
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = norm;
  if (c == 1.f) return;  // x * 1 is x: nothing to write
  if (blockIdx.x >= t.n_tiles) return;
  // last tile first: the norm's pass left the end of the table in L2
  const uint32_t tile = t.n_tiles - 1 - blockIdx.x;
  const SpanEnt& e = t.e[find_entry(t.e, t.n, tile)];
  const uint32_t dt = e.dtype, isz = dt == RS_F32 ? 4 : 2, per = 16 / isz, most = t.tile_bytes / isz;
  const uint64_t off = (uint64_t)(tile - e.tile_begin) * most;
  const uint32_t len = (uint32_t)min((uint64_t)most, e.numel - off);
  const uint64_t p = e.ptr + off * isz;
  const uint32_t head = min(len, (uint32_t)((16 - (p & 15)) & 15) / isz);
  const uint32_t nvec = (len - head) / per;
  char* body = reinterpret_cast<char*>(p + (uint64_t)head * isz);
  for (uint32_t i = threadIdx.x; i < nvec; i += 4 * kThreads) {
    uint4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i + u * kThreads < nvec) v[u] = ld16(body + (size_t)(i + u * kThreads) * 16);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const uint32_t j = i + u * kThreads;
      if (j >= nvec) break;
      float x[8];
      const int n = decode_vec(v[u], dt, x);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k < n) x[k] *= c;
      st16_stream(body + (size_t)j * 16, dt == RS_F32 ? pack16<float>(x) : dt == RS_BF16 ? pack16<__nv_bfloat16>(x) : pack16<__half>(x));
    }
  }
  const uint32_t loose = len - nvec * per;
  if (threadIdx.x < loose) {
    const uint32_t i = threadIdx.x < head ? threadIdx.x : threadIdx.x + nvec * per;
    store_scalar(p, i, dt, load_scalar(p, i, dt) * c);
  }
}

// ---- AdamW --------------------------------------------------------------------------------

struct AdamEnt {
  uint64_t grad, param, master, m, v;
  uint64_t numel;
  uint32_t tile_begin;
  uint32_t kinds;  // grad dtype | param dtype << 2 | moment dtype << 4 | (all 16-byte aligned) << 6
};
template <int CAP>
struct AdamTable {
  AdamEnt e[CAP];
  int32_t n;
  uint32_t n_tiles;
  uint32_t tile;
  float beta2, one_minus_beta1, one_minus_beta2, eps;
};

struct PrepEnt {
  uint64_t step;
  float weight_decay;
  uint32_t reserved;
};
template <int CAP>
struct PrepTable {
  PrepEnt e[CAP];
  int32_t n;
  double lr, beta1, beta2;
};

// Per tensor: step += 1 and, from it, the factors of the update; bias corrections in 64 bits
// (1 - beta^t loses digits in 32). One thread per tensor, so no CTA of the update reads a step that
// another one advances. {lr / (1 - b1^t), 1 / sqrt(1 - b2^t), 1 - lr * wd, clip factor}.
template <int CAP>
__global__ void __launch_bounds__(kThreads) prep_kernel(const __grid_constant__ PrepTable<CAP> t, const double* partial, int n_partial,
                                                        float max_norm, float* norm_out, float4* scal) {
  let_successor_start();
  after_predecessor();
  __shared__ float factor;
  float c = 1.f;
  if (n_partial) {  // the sum of squares, in one piece or in the norm's partial sums
    double sumsq = 0.0;
    for (int i = threadIdx.x; i < n_partial; i += kThreads) sumsq += partial[i];
    sumsq = block_sum(sumsq);
    if (threadIdx.x == 0) {
      float norm;
      factor = clip_factor(sumsq, max_norm, &norm);
      if (norm_out) *norm_out = norm;
    }
    __syncthreads();
    c = factor;
  }
  for (int i = threadIdx.x; i < t.n; i += kThreads) {
    float* sp = reinterpret_cast<float*>(t.e[i].step);
    const float step = *sp + 1.f;
    *sp = step;
    const double b1 = 1.0 - pow(t.beta1, (double)step), b2 = 1.0 - pow(t.beta2, (double)step);
    scal[i] = make_float4((float)(t.lr / b1), (float)(1.0 / sqrt(b2)), (float)(1.0 - t.lr * (double)t.e[i].weight_decay), c);
  }
}

struct AdamHyper {
  float beta2, omb1, omb2, eps;
};

// One element. All in 32 bits whatever the state's types: p, m and v are rounded once, when stored.
__device__ __forceinline__ void adam_one(float g, float& p, float& m, float& v, const float4& s, const AdamHyper& h) {
  g *= s.w;
  p *= s.z;
  m = fmaf(g - m, h.omb1, m);
  v = fmaf(v, h.beta2, g * g * h.omb2);
  p -= s.x * m / fmaf(sqrtf(v), s.y, h.eps);
}

struct Raw8 {
  uint4 a, b;
};
// 8 elements: one 16-byte load for 16-bit types, two for fp32. Loads only, so that those of all
// operands are in flight before the first conversion waits.
__device__ __forceinline__ Raw8 load_raw8(uint64_t base, uint64_t i, uint32_t dt) {
  Raw8 r;
  const char* p = reinterpret_cast<const char*>(base + i * (dt == RS_F32 ? 4 : 2));
  r.a = ld16(p);
  r.b = dt == RS_F32 ? ld16(p + 16) : make_uint4(0, 0, 0, 0);
  return r;
}
__device__ __forceinline__ void decode8(const Raw8& r, uint32_t dt, float* x) {
  if (dt == RS_F32) {
    unpack16<float>(r.a, x);
    unpack16<float>(r.b, x + 4);
  } else if (dt == RS_BF16) {
    unpack16<__nv_bfloat16>(r.a, x);
  } else {
    unpack16<__half>(r.a, x);
  }
}
__device__ __forceinline__ void store8(uint64_t base, uint64_t i, uint32_t dt, const float* x) {
  char* p = reinterpret_cast<char*>(base + i * (dt == RS_F32 ? 4 : 2));
  if (dt == RS_F32) {
    st16_stream(p, pack16<float>(x));
    st16_stream(p + 16, pack16<float>(x + 4));
  } else {
    st16_stream(p, dt == RS_BF16 ? pack16<__nv_bfloat16>(x) : pack16<__half>(x));
  }
}

// One pass over gradient, weights and moments: with a master copy in fp32, bf16 parameters and fp32
// moments it reads 14 and writes 14 bytes an element. The types are looked up per tensor (uniform
// over the CTA), so one launch takes tables of mixed types.
template <int CAP>
__global__ void __launch_bounds__(kThreads) adamw_kernel(const __grid_constant__ AdamTable<CAP> t, const float4* scal) {
  after_predecessor();
  const AdamHyper h{t.beta2, t.one_minus_beta1, t.one_minus_beta2, t.eps};
  const uint32_t tile = t.n_tiles - 1 - blockIdx.x;  // last tile first: the norm's pass left those gradients in L2
  const int k = find_entry(t.e, t.n, tile);
  const AdamEnt& e = t.e[k];
  const float4 s = scal[k];
  const uint64_t off = (uint64_t)(tile - e.tile_begin) * t.tile;
  const uint32_t len = (uint32_t)min((uint64_t)t.tile, e.numel - off);
  const uint32_t gd = e.kinds & 3, pd = (e.kinds >> 2) & 3, md = (e.kinds >> 4) & 3;
  const bool has_master = e.master != 0;
  const uint64_t wbase = has_master ? e.master : e.param;
  const uint32_t wd = has_master ? (uint32_t)RS_F32 : pd;
  const uint32_t whole = (e.kinds >> 6) & 1 ? len / 8 * 8 : 0;
  for (uint32_t i = threadIdx.x * 8; i < whole; i += kThreads * 8) {
    const uint64_t j = off + i;
    const Raw8 rg = load_raw8(e.grad, j, gd), rw = load_raw8(wbase, j, wd), rm = load_raw8(e.m, j, md), rv = load_raw8(e.v, j, md);
    float g[8], w[8], m[8], v[8];
    decode8(rg, gd, g);
    decode8(rw, wd, w);
    decode8(rm, md, m);
    decode8(rv, md, v);
#pragma unroll
    for (int q = 0; q < 8; ++q) adam_one(g[q], w[q], m[q], v[q], s, h);
    store8(wbase, j, wd, w);
    if (has_master) store8(e.param, j, pd, w);
    store8(e.m, j, md, m);
    store8(e.v, j, md, v);
  }
  for (uint32_t i = whole + threadIdx.x; i < len; i += kThreads) {
    const uint64_t j = off + i;
    float w = load_scalar(wbase, j, wd), m = load_scalar(e.m, j, md), v = load_scalar(e.v, j, md);
    adam_one(load_scalar(e.grad, j, gd), w, m, v, s, h);
    store_scalar(wbase, j, wd, w);
    if (has_master) store_scalar(e.param, j, pd, w);
    store_scalar(e.m, j, md, m);
    store_scalar(e.v, j, md, v);
  }
}

// ---- host ---------------------------------------------------------------------------------

// Size of a tile, in units of one round of a CTA (256 threads x 16 bytes, or x 8 elements of the update):
// about eight tiles for each SM, so that a small table still fills the GPU, and at most `most` rounds.
uint32_t tile_rounds(uint64_t rounds, int sms, uint32_t most) {
  const uint64_t want = (rounds + (uint64_t)sms * 8 - 1) / ((uint64_t)sms * 8);
  return (uint32_t)std::min<uint64_t>(std::max<uint64_t>(want, 1), most);
}

template <class Ent, class Tiles>
int lay_tiles(Ent* e, int n, Tiles tiles, uint32_t* n_tiles) {
  uint64_t at = 0;
  for (int i = 0; i < n; ++i) {
    e[i].tile_begin = (uint32_t)at;
    at += tiles(i);
    if (at > 0x7fffffffull) return tfail(RS_ERR_CAPACITY, "a tensor table of more than 2^31 tiles");
  }
  *n_tiles = (uint32_t)at;
  return RS_OK;
}

constexpr uint32_t kRoundBytes = kThreads * 16;
constexpr uint32_t kSumRounds = 8;     // 32 KB tiles, at most 64 CTAs to an SM: 7.04 TB/s; 8 CTAs to an SM 6.13
constexpr uint32_t kSmallRounds = 16;  // one batch of loads of 1024 threads
constexpr uint32_t kScaleRounds = 4;   // 16 KB tiles, one batch of loads: 6.85 TB/s; 32 KB 6.36
constexpr uint32_t kUpdateRounds = 4;  // 8192 elements
constexpr int kSumCtas = 64;           // per SM
constexpr int kMaxSms = 256;
constexpr int kSpanCaps[3] = {24, 160, 1280};
static_assert(sizeof(SpanTable<1280>) + 64 <= 32764, "kernel parameters");
static_assert(sizeof(AdamTable<560>) + 64 <= 32764, "kernel parameters");

template <int CAP, class Launch>
int span_chunk(const rs_grad_span* s, int n, int sms, uint32_t most_rounds, Launch launch) {
  SpanTable<CAP> t;
  uint64_t total = 0;
  for (int i = 0; i < n; ++i) {
    t.e[i].ptr = s[i].grad_dev;
    t.e[i].numel = s[i].numel;
    t.e[i].dtype = s[i].dtype;
    total += s[i].numel * dtype_bytes(s[i].dtype);
  }
  t.n = n;
  t.tile_bytes = tile_rounds(total / kRoundBytes, sms, most_rounds) * kRoundBytes;
  const int rc = lay_tiles(t.e, n, [&](int i) { return (s[i].numel * dtype_bytes(s[i].dtype) + t.tile_bytes - 1) / t.tile_bytes; }, &t.n_tiles);
  if (rc != RS_OK) return rc;
  return launch(t);
}

template <class Launch>
int for_spans(const std::vector<rs_grad_span>& s, int sms, uint32_t most_rounds, Launch launch) {
  for (size_t i = 0; i < s.size(); i += kSpanCaps[2]) {
    const int n = (int)std::min<size_t>(s.size() - i, kSpanCaps[2]);
    int rc = n <= kSpanCaps[0] ? span_chunk<kSpanCaps[0]>(&s[i], n, sms, most_rounds, launch)
           : n <= kSpanCaps[1] ? span_chunk<kSpanCaps[1]>(&s[i], n, sms, most_rounds, launch)
                               : span_chunk<kSpanCaps[2]>(&s[i], n, sms, most_rounds, launch);
    if (rc != RS_OK) return rc;
  }
  return RS_OK;
}

int check_spans(const char* what, const rs_grad_span* spans, int64_t n, std::vector<rs_grad_span>* out) {
  if (n < 0 || (n > 0 && !spans)) return tfail(RS_ERR_ARG, std::string(what) + ": NULL spans");
  out->reserve((size_t)n);
  for (int64_t i = 0; i < n; ++i) {
    const rs_grad_span& s = spans[i];
    if (s.numel == 0) continue;
    if (!s.grad_dev) return tfail(RS_ERR_ARG, std::string(what) + ": span " + std::to_string(i) + " has a NULL address");
    if (!dtype_known(s.dtype)) return tfail(RS_ERR_ARG, std::string(what) + ": span " + std::to_string(i) + " has an unknown dtype");
    if (s.grad_dev % dtype_bytes(s.dtype)) return tfail(RS_ERR_ARG, std::string(what) + ": span " + std::to_string(i) + " is not aligned to its elements");
    out->push_back(s);
  }
  return RS_OK;
}

template <int CAP>
auto sumsq_small_of(const SpanTable<CAP>&) -> void (*)(SpanTable<CAP>, double*) {
  return sumsq_small_kernel<CAP>;
}

template <int CAP>
auto scale_of(const SpanTable<CAP>&) -> void (*)(SpanTable<CAP>, const double*, float, float*) {
  return scale_kernel<CAP>;
}

// The partial sums of the norm's pass, one for each CTA; *used of them.
int launch_partials(const std::vector<rs_grad_span>& s, int sms, double* partial, int* used, cudaStream_t st) {
  *used = 0;
  return for_spans(s, sms, kSumRounds, [&](const auto& t) -> int {
    const int grid = (int)std::min<uint64_t>(t.n_tiles, (uint64_t)sms * kSumCtas);
    sumsq_kernel<<<grid, kThreads, 0, st>>>(t, partial + *used);
    *used += grid;
    return tcuda(cudaGetLastError(), "the norm's launch");
  });
}
uint64_t partial_bytes(int64_t n_spans) {
  const uint64_t launches = std::max<uint64_t>(1, ((uint64_t)n_spans + kSpanCaps[2] - 1) / kSpanCaps[2]);
  return launches * kSumCtas * kMaxSms * sizeof(double);
}

// Whether two of the ranges [begin, begin + bytes) share memory. Sorts them.
bool any_overlap(std::vector<std::pair<uint64_t, uint64_t>>& r) {
  std::sort(r.begin(), r.end());
  for (size_t i = 1; i < r.size(); ++i)
    if (r[i - 1].first + r[i - 1].second > r[i].first) return true;
  return false;
}

}  // namespace

extern "C" {

int rs_grad_sumsq_workspace_bytes(int64_t n_spans, uint64_t* bytes) {
  return guarded("rs_grad_sumsq_workspace_bytes", [&]() -> int {
    if (n_spans < 0 || !bytes) return tfail(RS_ERR_ARG, "rs_grad_sumsq_workspace_bytes: bad argument");
    *bytes = partial_bytes(n_spans);
    return RS_OK;
  });
}

int rs_grad_sumsq(const rs_grad_span* spans, int64_t n, void* workspace, uint64_t workspace_bytes, double* sumsq_dev,
                  int32_t device, void* stream) {
  return guarded("rs_grad_sumsq", [&]() -> int {
    std::vector<rs_grad_span> s;
    int rc = check_spans("rs_grad_sumsq", spans, n, &s);
    if (rc != RS_OK) return rc;
    if (!sumsq_dev || misaligned(8, sumsq_dev)) return tfail(RS_ERR_ARG, "rs_grad_sumsq: NULL or misaligned result");
    uint64_t need = 0;
    rs_grad_sumsq_workspace_bytes((int64_t)s.size(), &need);
    if (!workspace || workspace_bytes < need || misaligned(8, workspace))
      return tfail(RS_ERR_CAPACITY, "rs_grad_sumsq: workspace too small or not 8-byte aligned");
    DeviceGuard guard(device);
    if (guard.err != cudaSuccess) return tcuda(guard.err, "rs_grad_sumsq: cudaSetDevice");
    const int sms = std::min(sm_count(device), kMaxSms);
    cudaStream_t st = (cudaStream_t)stream;
    uint64_t bytes = 0;
    for (const rs_grad_span& g : s) bytes += g.numel * dtype_bytes(g.dtype);
    if (bytes <= kSmallBytes && !s.empty() && s.size() <= (size_t)kSpanCaps[2])
      return for_spans(s, 1, kSmallRounds, [&](const auto& t) -> int {  // eight tiles, or of 64 KB
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(kSmallCtas);
        cfg.blockDim = dim3(kSmallThreads);
        cfg.stream = st;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = kSmallCtas;
        at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
        return tcuda(cudaLaunchKernelEx(&cfg, sumsq_small_of(t), t, sumsq_dev), "rs_grad_sumsq: launch (small)");
      });
    double* partial = (double*)workspace;
    int used = 0;
    if ((rc = launch_partials(s, sms, partial, &used, st)) != RS_OK) return rc;
    return tcuda(launch_after(sumsq_finish_kernel, 1, kFinishThreads, st, partial, used, sumsq_dev), "rs_grad_sumsq: launch (finish)");
  });
}

int rs_grad_clip(const rs_grad_span* spans, int64_t n, const double* sumsq_dev, float max_norm, float* norm_dev,
                 int32_t device, void* stream) {
  return guarded("rs_grad_clip", [&]() -> int {
    std::vector<rs_grad_span> s;
    int rc = check_spans("rs_grad_clip", spans, n, &s);
    if (rc != RS_OK) return rc;
    if (!sumsq_dev || !norm_dev) return tfail(RS_ERR_ARG, "rs_grad_clip: NULL sum of squares or norm");
    if (misaligned(8, sumsq_dev) || misaligned(4, norm_dev)) return tfail(RS_ERR_ARG, "rs_grad_clip: a misaligned sum of squares or norm");
    if (!(max_norm > 0.f)) return tfail(RS_ERR_ARG, "rs_grad_clip: max_norm must be positive");
    std::vector<std::pair<uint64_t, uint64_t>> ranges;
    ranges.reserve(s.size());
    for (const rs_grad_span& g : s) ranges.emplace_back(g.grad_dev, g.numel * dtype_bytes(g.dtype));
    if (any_overlap(ranges)) return tfail(RS_ERR_ARG, "rs_grad_clip: gradients share memory");
    DeviceGuard guard(device);
    if (guard.err != cudaSuccess) return tcuda(guard.err, "rs_grad_clip: cudaSetDevice");
    const int sms = sm_count(device);
    cudaStream_t st = (cudaStream_t)stream;
    if (s.empty()) {  // no elements here: the norm alone
      SpanTable<kSpanCaps[0]> t{};
      return tcuda(launch_after(scale_kernel<kSpanCaps[0]>, 1, kThreads, st, t, sumsq_dev, max_norm, norm_dev), "rs_grad_clip: launch");
    }
    return for_spans(s, sms, kScaleRounds, [&](const auto& t) -> int {
      return tcuda(launch_after(scale_of(t), t.n_tiles, kThreads, st, t, sumsq_dev, max_norm, norm_dev), "rs_grad_clip: launch");
    });
  });
}

int rs_adamw_workspace_bytes(int64_t n_tensors, uint64_t* bytes) {
  return guarded("rs_adamw_workspace_bytes", [&]() -> int {
    if (n_tensors < 0 || !bytes) return tfail(RS_ERR_ARG, "rs_adamw_workspace_bytes: bad argument");
    *bytes = (std::max<uint64_t>(1, (uint64_t)n_tensors) * sizeof(float4) + 255) / 256 * 256 + partial_bytes(n_tensors);
    return RS_OK;
  });
}

}  // extern "C"

namespace {

template <int CAP>
int adam_chunk(const rs_adamw_tensor* a, int n, const rs_adamw_opts& o, const double* partial, int n_partial, float* norm_out,
               float4* scal, int sms, cudaStream_t st) {
  PrepTable<CAP> p;
  AdamTable<CAP> t;
  uint64_t total = 0;
  for (int i = 0; i < n; ++i) {
    p.e[i] = {a[i].step_dev, a[i].weight_decay, 0};
    const bool vec = ((a[i].grad_dev | a[i].param_dev | a[i].master_dev | a[i].exp_avg_dev | a[i].exp_avg_sq_dev) & 15) == 0;
    t.e[i] = {a[i].grad_dev, a[i].param_dev, a[i].master_dev, a[i].exp_avg_dev, a[i].exp_avg_sq_dev, a[i].numel, 0,
              a[i].grad_dtype | a[i].param_dtype << 2 | a[i].moment_dtype << 4 | (vec ? 64u : 0u)};
    total += a[i].numel;
  }
  p.n = t.n = n;
  p.lr = o.lr; p.beta1 = o.beta1; p.beta2 = o.beta2;
  t.beta2 = (float)o.beta2;
  t.one_minus_beta1 = (float)(1.0 - o.beta1);
  t.one_minus_beta2 = (float)(1.0 - o.beta2);
  t.eps = (float)o.eps;
  t.tile = tile_rounds(total / (kThreads * 8), sms, kUpdateRounds) * kThreads * 8;
  int rc = lay_tiles(t.e, n, [&](int i) { return (a[i].numel + t.tile - 1) / t.tile; }, &t.n_tiles);
  if (rc != RS_OK) return rc;
  rc = tcuda(launch_after(prep_kernel<CAP>, 1, kThreads, st, p, partial, n_partial, (float)o.max_norm, norm_out, scal), "rs_adamw_step: launch (factors)");
  if (rc != RS_OK || t.n_tiles == 0) return rc;
  return tcuda(launch_after(adamw_kernel<CAP>, t.n_tiles, kThreads, st, t, (const float4*)scal), "rs_adamw_step: launch");
}

}  // namespace

extern "C" int rs_adamw_step(const rs_adamw_tensor* tensors, int64_t n, const rs_adamw_opts* opts, const double* sumsq_dev,
                             float* norm_dev, void* workspace, uint64_t workspace_bytes, int32_t device, void* stream) {
  return guarded("rs_adamw_step", [&]() -> int {
    if (n < 0 || (n > 0 && !tensors) || !opts) return tfail(RS_ERR_ARG, "rs_adamw_step: NULL tensors or options");
    const rs_adamw_opts& o = *opts;
    if (!(o.beta1 >= 0 && o.beta1 < 1 && o.beta2 >= 0 && o.beta2 < 1 && o.eps >= 0 && o.lr >= 0))
      return tfail(RS_ERR_ARG, "rs_adamw_step: lr, betas or eps out of range");
    if (sumsq_dev ? !(o.max_norm > 0) : !(o.max_norm >= 0)) return tfail(RS_ERR_ARG, "rs_adamw_step: max_norm must be positive");
    if (misaligned(8, sumsq_dev) || misaligned(4, norm_dev)) return tfail(RS_ERR_ARG, "rs_adamw_step: a misaligned sum of squares or norm");
    const bool norm_alone = n == 0 && norm_dev && o.max_norm > 0;  // a rank without tensors
    if (n == 0 && !norm_alone) return RS_OK;
    for (int64_t i = 0; i < n; ++i) {
      const rs_adamw_tensor& a = tensors[i];
      const std::string who = "rs_adamw_step: tensor " + std::to_string(i);
      if (!a.step_dev || a.step_dev % 4) return tfail(RS_ERR_ARG, who + " has no step, or a misaligned one");
      if (!dtype_known(a.grad_dtype) || !dtype_known(a.param_dtype) || (a.moment_dtype != RS_F32 && a.moment_dtype != RS_BF16))
        return tfail(RS_ERR_ARG, who + " has a dtype that the update does not take");
      if (a.numel == 0) continue;
      if (!a.grad_dev || !a.param_dev || !a.exp_avg_dev || !a.exp_avg_sq_dev) return tfail(RS_ERR_ARG, who + " has a NULL address");
      if (a.grad_dev % dtype_bytes(a.grad_dtype) || a.param_dev % dtype_bytes(a.param_dtype) || a.master_dev % 4 ||
          a.exp_avg_dev % dtype_bytes(a.moment_dtype) || a.exp_avg_sq_dev % dtype_bytes(a.moment_dtype))
        return tfail(RS_ERR_ARG, who + " is not aligned to its elements");
    }
    uint64_t need = 0;
    rs_adamw_workspace_bytes(n, &need);
    if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16)
      return tfail(RS_ERR_CAPACITY, "rs_adamw_step: workspace too small or not 16-byte aligned");
    DeviceGuard guard(device);
    if (guard.err != cudaSuccess) return tcuda(guard.err, "rs_adamw_step: cudaSetDevice");
    const int sms = std::min(sm_count(device), kMaxSms);
    cudaStream_t st = (cudaStream_t)stream;
    float4* scal = (float4*)workspace;
    const double* partial = sumsq_dev;
    int n_partial = sumsq_dev ? 1 : 0;
    if (!sumsq_dev && o.max_norm > 0) {  // the norm of these gradients; the factors' launch adds the partial sums
      std::vector<rs_grad_span> s;
      s.reserve((size_t)n);
      for (int64_t i = 0; i < n; ++i)
        if (tensors[i].numel) s.push_back({tensors[i].grad_dev, tensors[i].numel, tensors[i].grad_dtype, 0});
      double* sums = (double*)((char*)workspace + (need - partial_bytes(n)));
      int rc = launch_partials(s, sms, sums, &n_partial, st);
      if (rc != RS_OK) return rc;
      if (n_partial == 0) {  // no elements: the norm is 0
        if ((rc = tcuda(cudaMemsetAsync(sums, 0, sizeof(double), st), "rs_adamw_step: cudaMemsetAsync")) != RS_OK) return rc;
        n_partial = 1;
      }
      partial = sums;
    }
    if (norm_alone) return adam_chunk<16>(tensors, 0, o, partial, n_partial, norm_dev, scal, sms, st);
    for (int64_t i = 0; i < n; i += 560) {
      const int c = (int)std::min<int64_t>(n - i, 560);
      int rc = c <= 16 ? adam_chunk<16>(tensors + i, c, o, partial, n_partial, norm_dev, scal + i, sms, st)
             : c <= 96 ? adam_chunk<96>(tensors + i, c, o, partial, n_partial, norm_dev, scal + i, sms, st)
                       : adam_chunk<560>(tensors + i, c, o, partial, n_partial, norm_dev, scal + i, sms, st);
      if (rc != RS_OK) return rc;
    }
    return RS_OK;
  });
}
