// Global norm of many gradients and clipping by it.
//
//   power = sum_i |g_i|^p (p = 1, 2; the largest |g_i| for infinity),  norm = scale * power^(1/p)
//   coef  = min(1, max_norm / (norm + 1e-6)),  factor = scale * coef,  g_i <- round(g_i * factor)
//
// Design (B200): multi-tensor launches, as the other elementwise kernels, with mixed types and
// any alignment. The work is cut into chunks of 16 KB that never cross a tensor; block b of G
// takes the consecutive chunks [b C / G, (b + 1) C / G), so a block touches few tensors and the
// norm of each tensor costs one block reduction per (block, tensor) pair. Those pairs lie on a
// monotone staircase, so slot b + t of the workspace belongs to one pair only and needs no
// clearing; no atomics are used and every sum has a fixed order, so results do not vary from run
// to run. Bounded by HBM: reading every gradient once; scaling reads and writes it once more.
#include "common.cuh"
#include "host_common.h"

#include <cuda_fp16.h>
#include <math.h>

#include <algorithm>
#include <utility>
#include <vector>

namespace msr {
namespace {

constexpr int GN_THREADS = 256;
constexpr int GN_VECS = 4;                            // 16-byte vectors per thread and chunk
constexpr int64_t GN_CHUNK = GN_THREADS * GN_VECS;    // vectors per chunk
constexpr int GN_BLOCKS_PER_SM = 4;
constexpr int GN_MAX_GRID = 2048;                     // slots of the workspace besides one per tensor
constexpr int GN_MAXE = 512;                          // tensors per launch
constexpr int GN_FINISH_THREADS = 1024;

struct GradArgs {
  void* ptr[GN_MAXE];
  int64_t numel[GN_MAXE];
  int64_t prefix[GN_MAXE + 1];  // exclusive prefix of the chunk counts
  uint8_t dtype[GN_MAXE];
  int count;
};

__host__ __device__ __forceinline__ int dtype_bytes(int dtype) { return dtype == MSR_FP32 ? 4 : 2; }

// A tensor as 16-byte vectors: `head` elements before the first 16-byte boundary, `vecs` whole
// vectors from there, `tail` elements after them.
struct Span {
  int64_t vecs;
  int head, tail;
};

__host__ __device__ __forceinline__ Span span_of(const void* p, int64_t n, int dtype) {
  const int es = dtype_bytes(dtype), per = 16 / es;
  int64_t head = ((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / es;
  if (head > n) head = n;
  Span s;
  s.head = static_cast<int>(head);
  s.vecs = (n - head) / per;
  s.tail = static_cast<int>((n - head) % per);
  return s;
}

// Chunks of a tensor: its vectors, and at least one where only head or tail elements exist.
__host__ __device__ __forceinline__ int64_t chunks_of(const Span& s) {
  const int64_t c = (s.vecs + GN_CHUNK - 1) / GN_CHUNK;
  return c > 0 ? c : (s.head + s.tail > 0 ? 1 : 0);
}

// First chunk of block b, and the block that holds chunk c, when `grid` blocks share `chunks`.
__host__ __device__ __forceinline__ int64_t first_chunk(int64_t b, int64_t chunks, int64_t grid) {
  return b * chunks / grid;
}
__host__ __device__ __forceinline__ int64_t block_of(int64_t c, int64_t chunks, int64_t grid) {
  return (grid * (c + 1) - 1) / chunks;
}

// ---------------------------------------------------------------------------------------
// Element access
// ---------------------------------------------------------------------------------------
template <int DT>
struct Elem;
template <>
struct Elem<MSR_BF16> {
  using type = uint16_t;
  static __device__ __forceinline__ float get(uint16_t b) { return bf16_bits_to_f32(b); }
  static __device__ __forceinline__ uint16_t put(float x) { return rne_bf16_bits(x); }
  static __device__ __forceinline__ void unpack(uint32_t w, float* x) {
    x[0] = __uint_as_float(w << 16);
    x[1] = __uint_as_float(w & 0xFFFF0000u);
  }
  static __device__ __forceinline__ uint32_t pack(const float* x) {
    return put(x[0]) | (static_cast<uint32_t>(put(x[1])) << 16);
  }
};
template <>
struct Elem<MSR_FP16> {
  using type = uint16_t;
  static __device__ __forceinline__ float get(uint16_t b) { return __half2float(__ushort_as_half(b)); }
  static __device__ __forceinline__ uint16_t put(float x) { return __half_as_ushort(__float2half_rn(x)); }
  static __device__ __forceinline__ void unpack(uint32_t w, float* x) {
    x[0] = get(static_cast<uint16_t>(w));
    x[1] = get(static_cast<uint16_t>(w >> 16));
  }
  static __device__ __forceinline__ uint32_t pack(const float* x) {
    return put(x[0]) | (static_cast<uint32_t>(put(x[1])) << 16);
  }
};
template <>
struct Elem<MSR_FP32> {
  using type = float;
  static __device__ __forceinline__ float get(float b) { return b; }
  static __device__ __forceinline__ float put(float x) { return x; }
  static __device__ __forceinline__ void unpack(uint32_t w, float* x) { x[0] = __uint_as_float(w); }
  static __device__ __forceinline__ uint32_t pack(const float* x) { return __float_as_uint(x[0]); }
};

// ---------------------------------------------------------------------------------------
// Powers. The accumulator is a double: 32 bits would lose the small terms of 10^10 elements,
// and squares of bf16 or fp32 values leave the range of fp32 at both ends.
// ---------------------------------------------------------------------------------------
__device__ __forceinline__ double positive_nan() { return __longlong_as_double(0x7FF8000000000000ll); }

template <int P>
__device__ __forceinline__ double combine(double a, double b) {
  if (P != MSR_NORM_INF) return a + b;
  return a != a || b != b ? positive_nan() : (a > b ? a : b);
}

template <int P>
__device__ __forceinline__ double power_of(float x) {
  const double d = fabs(static_cast<double>(x));
  return P == MSR_NORM_2 ? d * d : d;
}

// The power of GN_VECS vectors of one thread. Sums run in fp32 over these 16 or 32 values and
// join the double once: the conversions of every element would cost more than the loads. Where
// the fp32 sum left the range in which no term can have overflowed or lost bits that count
// (below 2^-90 a square may have underflowed: 32 terms of at most 2^-150 are 2^-55 of 2^-90),
// the same registers are summed again in double.
template <int P, int DT>
__device__ __forceinline__ double chunk_power(const uint4 (&v)[GN_VECS]) {
  constexpr int PAIR = DT == MSR_FP32 ? 1 : 2;
  const uint32_t* w = reinterpret_cast<const uint32_t*>(v);
  if (P == MSR_NORM_INF) {
    // magnitudes order as their bits do, NaN above infinity
    if (DT == MSR_FP32) {
      uint32_t m = 0u;
#pragma unroll
      for (int i = 0; i < 4 * GN_VECS; ++i) m = max(m, w[i] & 0x7FFFFFFFu);
      const float x = __uint_as_float(m);
      return x != x ? positive_nan() : static_cast<double>(x);
    }
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < 4 * GN_VECS; ++i) m = __vmaxu2(m, w[i] & 0x7FFF7FFFu);
    const uint16_t b = static_cast<uint16_t>(max(m & 0xFFFFu, m >> 16));
    const float x = DT == MSR_BF16 ? bf16_bits_to_f32(b) : __half2float(__ushort_as_half(b));
    return x != x ? positive_nan() : static_cast<double>(x);
  }
  float s[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4 * GN_VECS; ++i) {
    float x[2];
    Elem<DT>::unpack(w[i], x);
#pragma unroll
    for (int j = 0; j < PAIR; ++j) {
      float& a = s[(i * PAIR + j) & 1];
      a = P == MSR_NORM_2 ? fmaf(x[j], x[j], a) : a + fabsf(x[j]);
    }
  }
  const float sum = s[0] + s[1];
  if (sum < 0x1p126f && (P == MSR_NORM_1 || sum > 0x1p-90f)) return sum;
  uint32_t any = 0u;
#pragma unroll
  for (int i = 0; i < 4 * GN_VECS; ++i) any |= w[i];
  if ((any & (DT == MSR_FP32 ? 0x7FFFFFFFu : 0x7FFF7FFFu)) == 0u) return 0.0;
  double d = 0.0;
#pragma unroll
  for (int i = 0; i < 4 * GN_VECS; ++i) {
    float x[2];
    Elem<DT>::unpack(w[i], x);
#pragma unroll
    for (int j = 0; j < PAIR; ++j) d += power_of<P>(x[j]);
  }
  return d;
}

// The power of chunks [lo, hi) of one tensor, this thread's share.
template <int P, int DT>
__device__ __forceinline__ double span_power(const void* ptr, int64_t n, int64_t lo, int64_t hi) {
  using T = typename Elem<DT>::type;
  const Span s = span_of(ptr, n, DT);
  const T* p = static_cast<const T*>(ptr);
  const uint4* body = reinterpret_cast<const uint4*>(p + s.head);
  double acc = 0.0;
  for (int64_t c = lo; c < hi; ++c) {
    uint4 v[GN_VECS];
#pragma unroll
    for (int k = 0; k < GN_VECS; ++k) {
      const int64_t i = c * GN_CHUNK + k * GN_THREADS + threadIdx.x;
      v[k] = i < s.vecs ? body[i] : make_uint4(0u, 0u, 0u, 0u);
    }
    acc = combine<P>(acc, chunk_power<P, DT>(v));
  }
  if (lo == 0) {  // the first chunk's block also takes the elements outside the vectors
    const int t = threadIdx.x;
    if (t < s.head) acc = combine<P>(acc, power_of<P>(Elem<DT>::get(p[t])));
    if (t < s.tail) acc = combine<P>(acc, power_of<P>(Elem<DT>::get(p[n - s.tail + t])));
  }
  return acc;
}

template <int P>
__device__ __forceinline__ double warp_power(double x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x = combine<P>(x, __shfl_xor_sync(0xFFFFFFFFu, x, o));
  return x;
}

// Every thread gets the block's power; `red` holds one value per warp.
template <int P>
__device__ __forceinline__ double block_power(double x, double* red) {
  x = warp_power<P>(x);
  __syncthreads();  // red may still be read from the previous call
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = x;
  __syncthreads();
  double t = red[0];
  for (int w = 1; w < static_cast<int>(blockDim.x) / 32; ++w) t = combine<P>(t, red[w]);
  return t;
}

// EACH: one slot per (block, tensor) pair, at block + tensor; otherwise one slot per block.
template <int P, bool EACH>
__global__ __launch_bounds__(GN_THREADS, GN_BLOCKS_PER_SM) void grad_power_kernel(const __grid_constant__ GradArgs a,
                                                                                 double* slots) {
  __shared__ double red[GN_THREADS / 32];
  const int64_t chunks = a.prefix[a.count];
  int64_t c = first_chunk(blockIdx.x, chunks, gridDim.x);
  const int64_t end = first_chunk(blockIdx.x + 1, chunks, gridDim.x);
  int t = find_entry<GN_MAXE>(a.prefix, a.count, c);
  double acc = 0.0;
  while (c < end) {
    while (a.prefix[t + 1] <= c) ++t;
    const int64_t lo = c - a.prefix[t];
    const int64_t hi = min(end, a.prefix[t + 1]) - a.prefix[t];
    double x;
    if (a.dtype[t] == MSR_BF16) x = span_power<P, MSR_BF16>(a.ptr[t], a.numel[t], lo, hi);
    else if (a.dtype[t] == MSR_FP16) x = span_power<P, MSR_FP16>(a.ptr[t], a.numel[t], lo, hi);
    else x = span_power<P, MSR_FP32>(a.ptr[t], a.numel[t], lo, hi);
    if (EACH) {
      x = block_power<P>(x, red);
      if (threadIdx.x == 0) slots[blockIdx.x + t] = x;
    } else {
      acc = combine<P>(acc, x);
    }
    c = a.prefix[t] + hi;
  }
  if (!EACH) {
    acc = block_power<P>(acc, red);
    if (threadIdx.x == 0) slots[blockIdx.x] = acc;
  }
}

// ---------------------------------------------------------------------------------------
// From powers to norms and the factor
// ---------------------------------------------------------------------------------------
__device__ __forceinline__ double root(double power, int p) { return p == MSR_NORM_2 ? sqrt(power) : power; }

__device__ void write_state(msr_clip_state* st, double power, int p, double scale, double max_norm) {
  const double norm = root(power, p) * scale;
  // max_norm = infinity asks for no clipping, whatever the norm; a NaN norm makes coef NaN
  double coef = isinf(max_norm) ? 1.0 : max_norm / (norm + 1e-6);
  if (coef > 1.0) coef = 1.0;
  st->power = power;
  st->norm = static_cast<float>(norm);
  st->factor = static_cast<float>(coef * scale);
  st->active = !(coef == 1.0 && scale == 1.0);
  st->reserved = 0;
}

struct FinishArgs {
  const double* slots;
  msr_clip_state* state;
  float* each;  // norms of this launch's tensors, or NULL
  double scale, max_norm;
  int64_t grid;  // blocks of the power kernel (0: no chunks)
  int first, last;
};

template <int P>
__global__ __launch_bounds__(GN_FINISH_THREADS) void grad_finish_kernel(const __grid_constant__ GradArgs a,
                                                                       const __grid_constant__ FinishArgs f) {
  __shared__ double red[GN_FINISH_THREADS / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  double acc = 0.0;
  if (f.each) {
    const int64_t chunks = a.prefix[a.count];
    for (int t = warp; t < a.count; t += GN_FINISH_THREADS / 32) {
      double x = 0.0;
      if (a.prefix[t + 1] > a.prefix[t]) {
        const int64_t b1 = block_of(a.prefix[t + 1] - 1, chunks, f.grid);
        for (int64_t b = block_of(a.prefix[t], chunks, f.grid) + lane; b <= b1; b += 32)
          x = combine<P>(x, f.slots[b + t]);
      }
      x = warp_power<P>(x);
      if (lane == 0) {
        f.each[t] = static_cast<float>(root(x, P) * f.scale);
        acc = combine<P>(acc, x);
      }
    }
  } else {
    for (int64_t b = threadIdx.x; b < f.grid; b += GN_FINISH_THREADS) acc = combine<P>(acc, f.slots[b]);
  }
  acc = block_power<P>(acc, red);
  if (threadIdx.x == 0) {
    if (!f.first) acc = combine<P>(acc, f.state->power);
    if (f.last) write_state(f.state, acc, P, f.scale, f.max_norm);
    else f.state->power = acc;
  }
}

__global__ void grad_factor_kernel(msr_clip_state* st, int p, double scale, double max_norm) {
  write_state(st, st->power, p, scale, max_norm);
}

// ---------------------------------------------------------------------------------------
// Scaling: the same blocks over the same chunks as the power kernel, last chunk first, so that
// what that kernel read last (and L2 still holds) is read first.
// ---------------------------------------------------------------------------------------
template <int DT>
__device__ __forceinline__ void span_scale(void* ptr, int64_t n, int64_t lo, int64_t hi, float f) {
  using T = typename Elem<DT>::type;
  constexpr int PAIR = DT == MSR_FP32 ? 1 : 2;
  const Span s = span_of(ptr, n, DT);
  T* p = static_cast<T*>(ptr);
  uint4* body = reinterpret_cast<uint4*>(p + s.head);
  for (int64_t c = hi - 1; c >= lo; --c) {
    uint4 v[GN_VECS];
#pragma unroll
    for (int k = 0; k < GN_VECS; ++k) {
      const int64_t i = c * GN_CHUNK + k * GN_THREADS + threadIdx.x;
      if (i < s.vecs) v[k] = body[i];
    }
#pragma unroll
    for (int k = 0; k < GN_VECS; ++k) {
      const int64_t i = c * GN_CHUNK + k * GN_THREADS + threadIdx.x;
      if (i < s.vecs) {
        uint32_t* w = reinterpret_cast<uint32_t*>(&v[k]);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float x[2];
          Elem<DT>::unpack(w[q], x);
#pragma unroll
          for (int j = 0; j < PAIR; ++j) x[j] = __fmul_rn(x[j], f);
          w[q] = Elem<DT>::pack(x);
        }
        body[i] = v[k];
      }
    }
  }
  if (lo == 0) {
    const int t = threadIdx.x;
    if (t < s.head) p[t] = Elem<DT>::put(__fmul_rn(Elem<DT>::get(p[t]), f));
    if (t < s.tail) p[n - s.tail + t] = Elem<DT>::put(__fmul_rn(Elem<DT>::get(p[n - s.tail + t]), f));
  }
}

__global__ __launch_bounds__(GN_THREADS, GN_BLOCKS_PER_SM) void grad_scale_kernel(const __grid_constant__ GradArgs a,
                                                                                 const msr_clip_state* st) {
  if (!st->active) return;  // the norm is within the bound: the gradients stay as they are
  const float f = st->factor;
  const int64_t chunks = a.prefix[a.count];
  const int64_t begin = first_chunk(blockIdx.x, chunks, gridDim.x);
  int64_t c = first_chunk(blockIdx.x + 1, chunks, gridDim.x);
  int t = find_entry<GN_MAXE>(a.prefix, a.count, c - 1);
  while (c > begin) {
    while (a.prefix[t] >= c) --t;
    const int64_t lo = max(begin, a.prefix[t]) - a.prefix[t];
    const int64_t hi = c - a.prefix[t];
    if (a.dtype[t] == MSR_BF16) span_scale<MSR_BF16>(a.ptr[t], a.numel[t], lo, hi, f);
    else if (a.dtype[t] == MSR_FP16) span_scale<MSR_FP16>(a.ptr[t], a.numel[t], lo, hi, f);
    else span_scale<MSR_FP32>(a.ptr[t], a.numel[t], lo, hi, f);
    c = a.prefix[t] + lo;
  }
}

// ---------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------
int grid_for(int64_t chunks) {
  const int64_t cap = std::min<int64_t>(static_cast<int64_t>(sm_count()) * GN_BLOCKS_PER_SM, GN_MAX_GRID);
  return static_cast<int>(std::min<int64_t>(chunks, cap));
}

int check_entries(const msr_grad_entry* e, int count, const char* what) {
  if (count < 0 || (count > 0 && e == nullptr)) return fail(MSR_ERR_INVALID, "%s: bad entry list", what);
  for (int i = 0; i < count; ++i) {
    if (e[i].numel < 0 || (e[i].numel > 0 && !e[i].grad))
      return fail(MSR_ERR_INVALID, "%s: entry %d has a null pointer or negative numel", what, i);
    if (e[i].dtype != MSR_BF16 && e[i].dtype != MSR_FP16 && e[i].dtype != MSR_FP32)
      return fail(MSR_ERR_INVALID, "%s: entry %d has unknown dtype %d", what, i, e[i].dtype);
    if (reinterpret_cast<uintptr_t>(e[i].grad) % dtype_bytes(e[i].dtype))
      return fail(MSR_ERR_INVALID, "%s: entry %d is not aligned to its elements", what, i);
  }
  return MSR_OK;
}

int check_factor(int norm, double scale, double max_norm, const char* what) {
  if (norm != MSR_NORM_INF && norm != MSR_NORM_1 && norm != MSR_NORM_2)
    return fail(MSR_ERR_INVALID, "%s: unknown norm %d", what, norm);
  if (!(scale > 0.0) || std::isinf(scale)) return fail(MSR_ERR_INVALID, "%s: scale must be positive and finite", what);
  if (!(max_norm >= 0.0)) return fail(MSR_ERR_INVALID, "%s: max_norm must be >= 0", what);
  return MSR_OK;
}

// The table of entries [begin, begin + GN_MAXE) and its number of chunks.
int64_t fill_args(GradArgs& a, const msr_grad_entry* e, int begin, int count) {
  a.count = std::min(count - begin, GN_MAXE);
  int64_t chunks = 0;
  for (int i = 0; i < a.count; ++i) {
    const msr_grad_entry& x = e[begin + i];
    a.ptr[i] = x.grad;
    a.numel[i] = x.numel;
    a.dtype[i] = static_cast<uint8_t>(x.dtype);
    a.prefix[i] = chunks;
    if (x.numel > 0) chunks += chunks_of(span_of(x.grad, x.numel, x.dtype));
  }
  a.prefix[a.count] = chunks;
  return chunks;
}

template <int P>
int norm_launch(const msr_grad_entry* entries, int count, double scale, double max_norm, msr_clip_state* state,
                float* each, double* slots, cudaStream_t s) {
  int begin = 0;
  do {
    GradArgs a;
    const int64_t chunks = fill_args(a, entries, begin, count);
    const int grid = grid_for(chunks);
    if (grid > 0) {
      if (each) grad_power_kernel<P, true><<<grid, GN_THREADS, 0, s>>>(a, slots);
      else grad_power_kernel<P, false><<<grid, GN_THREADS, 0, s>>>(a, slots);
      if (int st = check_launch("grad_power_kernel")) return st;
    }
    FinishArgs f{slots, state, each ? each + begin : nullptr, scale, max_norm, grid, begin == 0,
                 begin + a.count >= count};
    grad_finish_kernel<P><<<1, GN_FINISH_THREADS, 0, s>>>(a, f);
    if (int st = check_launch("grad_finish_kernel")) return st;
    begin += a.count;
  } while (begin < count);
  return MSR_OK;
}

// Two entries of one scaling launch must not share memory: both would multiply it.
int check_apart(const msr_grad_entry* e, int count) {
  std::vector<std::pair<uintptr_t, uintptr_t>> r;
  r.reserve(count);
  for (int i = 0; i < count; ++i)
    if (e[i].numel > 0) {
      const uintptr_t p = reinterpret_cast<uintptr_t>(e[i].grad);
      r.emplace_back(p, p + static_cast<uintptr_t>(e[i].numel) * dtype_bytes(e[i].dtype));
    }
  std::sort(r.begin(), r.end());
  for (size_t i = 1; i < r.size(); ++i)
    if (r[i].first < r[i - 1].second) return fail(MSR_ERR_INVALID, "msr_grad_scale: two gradients overlap in memory");
  return MSR_OK;
}

}  // namespace
}  // namespace msr

using namespace msr;

extern "C" {

size_t msr_grad_norm_workspace_bytes(int count) {
  return count < 0 ? 0 : (static_cast<size_t>(GN_MAX_GRID) + std::min(count, GN_MAXE)) * sizeof(double);
}

int msr_grad_norm(const msr_grad_entry* entries, int count, int norm, double scale, double max_norm,
                  msr_clip_state* state, float* each, void* workspace, size_t workspace_bytes, msr_stream_t stream) {
  if (int st = check_entries(entries, count, "msr_grad_norm")) return st;
  if (int st = check_factor(norm, scale, max_norm, "msr_grad_norm")) return st;
  if (!state || reinterpret_cast<uintptr_t>(state) % 8)
    return fail(MSR_ERR_INVALID, "msr_grad_norm: state must be an 8-byte aligned device pointer");
  if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 8)
    return fail(MSR_ERR_INVALID, "msr_grad_norm: workspace must be an 8-byte aligned device pointer");
  if (workspace_bytes < msr_grad_norm_workspace_bytes(count))
    return fail(MSR_ERR_WORKSPACE, "msr_grad_norm: workspace of %zu bytes, %zu needed", workspace_bytes,
                msr_grad_norm_workspace_bytes(count));
  if (int st = require_sm100()) return st;
  double* slots = static_cast<double*>(workspace);
  cudaStream_t s = to_stream(stream);
  switch (norm) {
    case MSR_NORM_INF: return norm_launch<MSR_NORM_INF>(entries, count, scale, max_norm, state, each, slots, s);
    case MSR_NORM_1: return norm_launch<MSR_NORM_1>(entries, count, scale, max_norm, state, each, slots, s);
    default: return norm_launch<MSR_NORM_2>(entries, count, scale, max_norm, state, each, slots, s);
  }
}

int msr_grad_factor(msr_clip_state* state, int norm, double scale, double max_norm, msr_stream_t stream) {
  if (int st = check_factor(norm, scale, max_norm, "msr_grad_factor")) return st;
  if (!state || reinterpret_cast<uintptr_t>(state) % 8)
    return fail(MSR_ERR_INVALID, "msr_grad_factor: state must be an 8-byte aligned device pointer");
  grad_factor_kernel<<<1, 1, 0, to_stream(stream)>>>(state, norm, scale, max_norm);
  return check_launch("grad_factor_kernel");
}

int msr_grad_scale(const msr_grad_entry* entries, int count, const msr_clip_state* state, msr_stream_t stream) {
  if (int st = check_entries(entries, count, "msr_grad_scale")) return st;
  if (!state || reinterpret_cast<uintptr_t>(state) % 8)
    return fail(MSR_ERR_INVALID, "msr_grad_scale: state must be an 8-byte aligned device pointer");
  try {
    if (int st = check_apart(entries, count)) return st;
  } catch (...) {
    return fail(MSR_ERR_INVALID, "msr_grad_scale: out of host memory");
  }
  for (int begin = 0; begin < count; begin += GN_MAXE) {
    GradArgs a;
    const int64_t chunks = fill_args(a, entries, begin, count);
    if (chunks == 0) continue;
    grad_scale_kernel<<<grid_for(chunks), GN_THREADS, 0, to_stream(stream)>>>(a, state);
    if (int st = check_launch("grad_scale_kernel")) return st;
  }
  return MSR_OK;
}

}  // extern "C"
