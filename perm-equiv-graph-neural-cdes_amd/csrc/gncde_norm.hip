// The global norm of many tensors, and clipping to it (gncde_global_norm, gncde_clip_by_global_norm).
//
//   n = sqrt(sum_t sum_i t_i^2),  m = max_t max_i |t_i|,   out_t = t  if n < c,  else t * (c / n)
//
// the rule of optax.clip_by_global_norm (optimiser_configs.py:76-84) and of k_adamw, for tensors that stay where they
// are: fp32, bf16 and fp16 in one list, no concatenation.
//
// Two launches for every 128 tensors.  k_norm_part cuts each tensor into chunks, one workgroup a chunk, and writes one
// (sum of squares, largest magnitude) per chunk; k_norm_apply has every workgroup add up all the chunks' sums itself,
// in the same order (so no launch in between, no atomics, and the same bits from every workgroup), and scale its chunk.
// (Of very long lists k_norm_join adds them up, in that order too.)
// The tensor table travels in the kernel arguments: no copy to the device, and a captured graph keeps it.
//
// Squares and sums are held in 64 bits: an fp32 square overflows from 1.8e19 and is lost below 1e-19, and a gradient
// list may hold either.
#include "gncde_internal.h"

#include <cmath>

namespace gncde {
namespace {

constexpr int kTensors = 128;       // table entries a launch (128 * 24 + 129 * 4 bytes of 4096 of kernel arguments)
constexpr int kThreads = 256;
constexpr int kChunks = 2048;       // chunks aimed at: 8 workgroups a CU, all resident at once
// Past so many chunks (more than two thousand tensors) one workgroup adds them up first: as it is otherwise, every
// workgroup of every table's launch does, which costs the square of the tensors (clip of 5000 tensors 522 -> 447 us, 20000
// 3190 -> 2000, 100000 46 -> 13 ms; at 2000 the extra launch would gain nothing).
constexpr int kJoin = 2 * kChunks;
constexpr int64_t kMinChunk = 32768;  // bytes: one round of 8 16-byte loads for every thread
// Past what the last-level cache (256 MB) holds, a list's reads and writes go round it: 1.5e9 bf16 values clip in 1644
// instead of 1742 us (5.5 TB/s over both passes), 200 million mixed ones are summed in 83 instead of 94 us (6.4 TB/s).
// Below, the second pass finds the tensors there.
constexpr int64_t kStream = int64_t(256) << 20;

struct Entry {
  const void* in;
  void* out;
  int64_t n_dtype;  // numel * 4 + dtype
};

struct Table {
  Entry e[kTensors];
  int32_t first[kTensors + 1];  // first chunk of each entry, counted from this launch's first
  int32_t count;
  int32_t base;     // chunks of the launches before
  int64_t chunk;    // bytes, a multiple of kMinChunk
};

struct Part {
  double sum;
  float top;
  float pad;
};

typedef float f32x4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8), aligned(2)));

template <int DT>
struct Kind;
template <>
struct Kind<GNCDE_DTYPE_FP32> {
  typedef float T;
  typedef f32x4 V;
  static constexpr int N = 4;
  static __device__ __forceinline__ float get(float x) { return x; }
  static __device__ __forceinline__ float put(float x) { return x; }
};
template <>
struct Kind<GNCDE_DTYPE_BF16> {
  typedef uint16_t T;
  typedef u16x8 V;
  static constexpr int N = 8;
  static __device__ __forceinline__ float get(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }
  static __device__ __forceinline__ uint16_t put(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }
};
template <>
struct Kind<GNCDE_DTYPE_FP16> {
  typedef uint16_t T;
  typedef u16x8 V;
  static constexpr int N = 8;
  static __device__ __forceinline__ float get(uint16_t x) { return (float)__builtin_bit_cast(_Float16, x); }
  static __device__ __forceinline__ uint16_t put(float x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }
};

// Entry of this workgroup's chunk: the last whose first chunk is not past it.  Every lane looks at its entries at once:
// each step of a search would wait for a read of its own (0.2 us a launch).
__device__ __forceinline__ int entry_of(const Table& t, int chunk) {
  const int lane = threadIdx.x & 63;
  int upto = 0;
#pragma unroll
  for (int i = 0; i < kTensors; i += 64)
    upto += __popcll(__ballot(lane + i < t.count && t.first[lane + i] <= chunk));
  return __builtin_amdgcn_readfirstlane(upto - 1);
}

__device__ __forceinline__ void block_sum(double& s, float& m) {
  __shared__ double rs[kThreads / 64];
  __shared__ float rm[kThreads / 64];
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    s += __shfl_xor(s, d);
    m = fmaxf(m, __shfl_xor(m, d));
  }
  if ((threadIdx.x & 63) == 0) {
    rs[threadIdx.x >> 6] = s;
    rm[threadIdx.x >> 6] = m;
  }
  __syncthreads();
  s = rs[0];
  m = rm[0];
#pragma unroll
  for (int w = 1; w < kThreads / 64; ++w) {
    s += rs[w];
    m = fmaxf(m, rm[w]);
  }
}

template <bool STREAM, typename V>
__device__ __forceinline__ V fetch(const V* p) {
  return STREAM ? __builtin_nontemporal_load(p) : *p;
}

// The vector at x[pos..], zeros from `to` on (a zero changes neither a sum of squares nor a largest magnitude).
template <int DT>
__device__ __forceinline__ typename Kind<DT>::V load_to(const typename Kind<DT>::T* x, int64_t pos, int64_t to) {
  typedef Kind<DT> K;
  typename K::V v = {};
  if (pos + K::N <= to) {
    v = *reinterpret_cast<const typename K::V*>(x + pos);
  } else {
#pragma unroll
    for (int i = 0; i < K::N; ++i)
      if (pos + i < to) v[i] = x[pos + i];
  }
  return v;
}

constexpr int kUnroll = 8;  // 16-byte loads in flight a thread

template <int DT, bool STREAM>
__device__ __forceinline__ void part(const void* p, int64_t from, int64_t to, double& s, float& m) {
  typedef Kind<DT> K;
  const typename K::T* x = static_cast<const typename K::T*>(p);
  constexpr int64_t step = (int64_t)kThreads * K::N;
  double acc[2] = {0.0, 0.0};
  for (int64_t at = from; at < to; at += kUnroll * step) {
    typename K::V v[kUnroll];
    const int64_t pos = at + threadIdx.x * K::N;
    if (at + kUnroll * step <= to) {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) v[u] = fetch<STREAM>(reinterpret_cast<const typename K::V*>(x + pos + u * step));
    } else {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) v[u] = load_to<DT>(x, pos + u * step, to);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int i = 0; i < K::N; ++i) {
        const float f = K::get(v[u][i]);
        m = fmaxf(m, fabsf(f));
        const double d = (double)f;
        acc[i & 1] = fma(d, d, acc[i & 1]);
      }
  }
  s = acc[0] + acc[1];
}

__device__ __forceinline__ int size_of(int dt) { return dt == GNCDE_DTYPE_FP32 ? 4 : 2; }

template <bool STREAM>
__global__ void __launch_bounds__(kThreads) k_norm_part(Table t, Part* __restrict__ parts) {
  const int k = entry_of(t, blockIdx.x);
  const Entry e = t.e[k];
  const int dt = (int)(e.n_dtype & 3);
  const int64_t n = e.n_dtype >> 2, per = t.chunk / size_of(dt);
  const int64_t from = (int64_t)(blockIdx.x - t.first[k]) * per;
  const int64_t to = from + per < n ? from + per : n;
  double s = 0.0;
  float m = 0.f;
  if (dt == GNCDE_DTYPE_FP32) part<GNCDE_DTYPE_FP32, STREAM>(e.in, from, to, s, m);
  else if (dt == GNCDE_DTYPE_BF16) part<GNCDE_DTYPE_BF16, STREAM>(e.in, from, to, s, m);
  else part<GNCDE_DTYPE_FP16, STREAM>(e.in, from, to, s, m);
  block_sum(s, m);
  if (threadIdx.x == 0) parts[t.base + blockIdx.x] = Part{s, m, 0.f};
}

// All chunks' sum and largest magnitude, the same bits in every workgroup.
__device__ __forceinline__ void join(const Part* __restrict__ parts, int nparts, double& s, float& m) {
  s = 0.0;
  m = 0.f;
  for (int i = threadIdx.x; i < nparts; i += kThreads) {
    const Part p = parts[i];
    s += p.sum;
    m = fmaxf(m, p.top);
  }
  block_sum(s, m);
}

// Norm and largest magnitude from all chunks.  fmaxf passes over a NaN; the sum does not, and says so for both.
__device__ __forceinline__ void total(const Part* __restrict__ parts, int nparts, float& norm, float& top) {
  double s;
  float m;
  join(parts, nparts, s, m);
  norm = (float)sqrt(s);
  top = s != s ? norm : m;
}

__global__ void __launch_bounds__(kThreads) k_norm_join(Part* __restrict__ parts, int nparts) {
  double s;
  float m;
  join(parts, nparts, s, m);
  if (threadIdx.x == 0) parts[nparts] = Part{s, m, 0.f};
}

__global__ void __launch_bounds__(kThreads) k_norm_total(const Part* __restrict__ parts, int nparts,
                                                         float* __restrict__ stats) {
  float norm, top;
  total(parts, nparts, norm, top);
  if (threadIdx.x == 0) {
    stats[0] = norm;
    stats[1] = top;
  }
}

// t c / n as t half (c / n) half: below 2^-126 fp32 would hold few bits of c / n, or none, though t c / n is an ordinary
// value for t near n.  There half is 2^-64 (t loses nothing to it that the result would hold) and c / n taken 2^128 times.
struct Scale {
  float by, half;
  __device__ __forceinline__ Scale() {}
  __device__ __forceinline__ Scale(float norm, float c) : by(c / norm), half(1.f) {
    if (by < 0x1p-126f && norm < INFINITY) by = (c * 0x1p64f) / (norm * 0x1p-64f), half = 0x1p-64f;
  }
  __device__ __forceinline__ float operator()(float t) const { return t * half * by * half; }
};

// The chunk's first values are on their way while `scale_of`, which the whole workgroup takes part in, adds up the norm
// (200 tensors of 30 million values: 86.3 -> 84.4 us); it says false where nothing is to be written.
template <int DT, bool STREAM, typename Find>
__device__ __forceinline__ void apply(const void* p, void* q, int64_t from, int64_t to, Find scale_of) {
  typedef Kind<DT> K;
  const typename K::T* x = static_cast<const typename K::T*>(p);
  typename K::T* y = static_cast<typename K::T*>(q);
  constexpr int64_t step = (int64_t)kThreads * K::N;
  typename K::V v[kUnroll];
  const auto load = [&](int64_t at) {
    const int64_t pos = at + threadIdx.x * K::N;
    if (at + kUnroll * step <= to) {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) v[u] = fetch<STREAM>(reinterpret_cast<const typename K::V*>(x + pos + u * step));
    } else {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) v[u] = load_to<DT>(x, pos + u * step, to);
    }
  };
  load(from);
  Scale scale;
  if (!scale_of(scale)) return;
  for (int64_t at = from; at < to;) {
    const bool whole = at + kUnroll * step <= to;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
#pragma unroll
      for (int i = 0; i < K::N; ++i) v[u][i] = K::put(scale(K::get(v[u][i])));
      const int64_t w = at + threadIdx.x * K::N + u * step;
      if (whole || w + K::N <= to) {
        if (STREAM) __builtin_nontemporal_store(v[u], reinterpret_cast<typename K::V*>(y + w));
        else *reinterpret_cast<typename K::V*>(y + w) = v[u];
      } else {
#pragma unroll
        for (int i = 0; i < K::N; ++i)
          if (w + i < to) y[w + i] = v[u][i];
      }
    }
    at += kUnroll * step;
    if (at < to) load(at);
  }
}

template <bool STREAM>
__global__ void __launch_bounds__(kThreads) k_norm_apply(Table t, const Part* __restrict__ parts, int nparts,
                                                         float max_norm, float* __restrict__ stats) {
  // The chunks in reverse: what the first pass read last is still in the cache.
  const int chunk = (int)gridDim.x - 1 - (int)blockIdx.x;
  const int k = entry_of(t, chunk);
  const Entry e = t.e[k];
  const auto scale_of = [&](Scale& scale) {
    float norm, top;
    total(parts, nparts, norm, top);
    if (t.base == 0 && blockIdx.x == 0 && threadIdx.x == 0) {
      stats[0] = norm;
      stats[1] = top;
    }
    const bool keep = norm < max_norm;
    scale = keep ? Scale(1.f, 1.f) : Scale(norm, max_norm);
    return !(keep && e.in == e.out);
  };
  const int dt = (int)(e.n_dtype & 3);
  const int64_t n = e.n_dtype >> 2, per = t.chunk / size_of(dt);
  const int64_t from = (int64_t)(chunk - t.first[k]) * per;
  const int64_t to = from + per < n ? from + per : n;
  if (dt == GNCDE_DTYPE_FP32) apply<GNCDE_DTYPE_FP32, STREAM>(e.in, e.out, from, to, scale_of);
  else if (dt == GNCDE_DTYPE_BF16) apply<GNCDE_DTYPE_BF16, STREAM>(e.in, e.out, from, to, scale_of);
  else apply<GNCDE_DTYPE_FP16, STREAM>(e.in, e.out, from, to, scale_of);
}

int host_size(int dt) { return dt == GNCDE_DTYPE_FP32 ? 4 : dt == GNCDE_DTYPE_BF16 || dt == GNCDE_DTYPE_FP16 ? 2 : 0; }

int check_list(int32_t count, const GncdeTensor* ts, bool out, int64_t& bytes) {
  if (count < 0 || (count > 0 && !ts)) return GNCDE_ERR_ARG;
  bytes = 0;
  for (int i = 0; i < count; ++i) {
    const int sz = host_size(ts[i].dtype);
    if (!sz) return GNCDE_ERR_UNSUPPORTED;
    if (ts[i].numel < 0 || ts[i].numel > (int64_t(1) << 56)) return GNCDE_ERR_SHAPE;
    if (ts[i].numel > 0 && (!ts[i].in || (out && !ts[i].out))) return GNCDE_ERR_ARG;
    if (((uintptr_t)ts[i].in | (out ? (uintptr_t)ts[i].out : 0)) % sz) return GNCDE_ERR_ARG;
    bytes += ts[i].numel * sz;
    if (bytes > (int64_t(1) << 58)) return GNCDE_ERR_SHAPE;
  }
  return GNCDE_OK;
}

// Chunk size in bytes: about kChunks of them over the whole list, so the sums every workgroup adds up stay few.
int64_t chunk_bytes(int64_t bytes) {
  const int64_t c = (bytes + kChunks - 1) / kChunks;
  return c <= kMinChunk ? kMinChunk : (c + kMinChunk - 1) / kMinChunk * kMinChunk;
}

int run(int32_t count, const GncdeTensor* ts, float* stats, bool clip, float max_norm, void* workspace,
        size_t workspace_bytes, void* stream) {
  int64_t bytes = 0;
  const int rc = check_list(count, ts, clip, bytes);
  if (rc != GNCDE_OK) return rc;
  if (!stats) return GNCDE_ERR_ARG;
  if (!workspace || workspace_bytes < gncde_global_norm_workspace_bytes(count)) return GNCDE_ERR_WORKSPACE;
  hipStream_t st = static_cast<hipStream_t>(stream);
  Part* parts = static_cast<Part*>(workspace);
  const int64_t chunk = chunk_bytes(bytes);
  int nparts = 0;
  const Part* sums = parts;  // what the second pass adds up
  bool applied = false;
  for (int pass = 0; pass < (clip ? 2 : 1); ++pass) {
    Table t;
    int i = 0, base = 0;
    while (i < count) {
      t.count = 0;
      t.first[0] = 0;
      for (; i < count && t.count < kTensors; ++i) {
        if (ts[i].numel == 0) continue;
        t.e[t.count] = Entry{ts[i].in, ts[i].out, ts[i].numel * 4 + ts[i].dtype};
        const int64_t per = chunk / host_size(ts[i].dtype);
        t.first[t.count + 1] = t.first[t.count] + (int)((ts[i].numel + per - 1) / per);
        ++t.count;
      }
      if (t.count == 0) break;
      t.base = base;
      t.chunk = chunk;
      const int blocks = t.first[t.count];
      const bool stream_past = bytes > kStream;
      if (pass == 0) {
        if (stream_past) hipLaunchKernelGGL(k_norm_part<true>, dim3(blocks), dim3(kThreads), 0, st, t, parts);
        else hipLaunchKernelGGL(k_norm_part<false>, dim3(blocks), dim3(kThreads), 0, st, t, parts);
      } else {
        if (stream_past)
          hipLaunchKernelGGL(k_norm_apply<true>, dim3(blocks), dim3(kThreads), 0, st, t, sums, nparts, max_norm, stats);
        else
          hipLaunchKernelGGL(k_norm_apply<false>, dim3(blocks), dim3(kThreads), 0, st, t, sums, nparts, max_norm, stats);
        applied = true;
      }
      base += blocks;
    }
    nparts = base;
    if (clip && pass == 0 && nparts > kJoin) {
      hipLaunchKernelGGL(k_norm_join, dim3(1), dim3(kThreads), 0, st, parts, nparts);
      sums = parts + nparts, nparts = 1;
    }
  }
  if (!applied) hipLaunchKernelGGL(k_norm_total, dim3(1), dim3(kThreads), 0, st, parts, nparts, stats);
  return hipGetLastError() == hipSuccess ? GNCDE_OK : GNCDE_ERR_HIP;
}

}  // namespace
}  // namespace gncde

extern "C" {

size_t gncde_global_norm_workspace_bytes(int32_t count) {
  return count < 0 ? 0 : ((size_t)gncde::kChunks + (size_t)count + 1) * sizeof(gncde::Part);
}

int gncde_global_norm(int32_t count, const GncdeTensor* tensors, float* stats, void* workspace,
                      size_t workspace_bytes, void* stream) {
  return gncde::run(count, tensors, stats, false, 0.f, workspace, workspace_bytes, stream);
}

int gncde_clip_by_global_norm(int32_t count, const GncdeTensor* tensors, float max_norm, float* stats,
                              void* workspace, size_t workspace_bytes, void* stream) {
  if (!(max_norm > 0.f) || std::isinf(max_norm)) return GNCDE_ERR_ARG;
  return gncde::run(count, tensors, stats, true, max_norm, workspace, workspace_bytes, stream);
}

}  // extern "C"
