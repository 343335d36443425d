// Global norm of many gradients and clipping by it.
//
//   power = sum_i |g_i|^p (p = 1, 2; the largest |g_i| for infinity),  norm = scale * power^(1/p)
//   coef  = min(1, max_norm / (norm + 1e-6)),  factor = scale * coef,  g_i <- round(g_i * factor)
//
// Design (B200): multi-tensor launches, as the other elementwise kernels, with mixed types and
// any alignment. The work is cut into chunks of 32 KB that never cross a tensor; block b of G
// takes the consecutive chunks [b C / G, (b + 1) C / G), so a block touches few tensors and the
// norm of each tensor costs one block reduction per (block, tensor) pair. Those pairs lie on a
// monotone staircase, so slot b + t of the workspace belongs to one pair only and needs no
// clearing; no atomics are used and every sum has a fixed order, so results do not vary from run
// to run. Bounded by HBM: reading every gradient once; scaling reads and writes it once more.
#include "common.cuh"
#include "host_common.h"

#include <cooperative_groups.h>
#include <cuda_fp16.h>
#include <float.h>
#include <math.h>

#include <algorithm>
#include <utility>
#include <vector>

namespace cg = cooperative_groups;

namespace msr {
namespace {

// The power kernel: 2 CTAs of 512 threads per SM, 4 vectors of 16 bytes per thread and chunk.
// Measured on 1.9 G bf16 elements (3.8 GB): 7.15 TB/s, against 7.0 for 4 CTAs of 256 threads,
// 6.2 for 2 vectors and 5.9 for 2 CTAs of 256 threads (too few loads in flight), 5.0 and 4.1 for
// 5 and 6 CTAs of 256 (the registers then spill).
constexpr int GN_THREADS = 512;
constexpr int GN_VECS = 4;
constexpr int GN_BLOCKS_PER_SM = 2;
constexpr int64_t GN_CHUNK = GN_THREADS * GN_VECS;    // vectors per chunk
// The scaling kernels: 2 CTAs of 256 threads per SM, 8 vectors per thread, so that each CTA
// reads and then writes a whole chunk in one go. Measured on the same elements, read + written:
// 6.3 TB/s, against 5.8 for 4 CTAs with 4 vectors, 5.7 for 3 CTAs, 5.1 for 16 vectors (spills).
constexpr int GN_SCALE_THREADS = 256;
constexpr int GN_SCALE_VECS = 8;
constexpr int GN_SCALE_BLOCKS_PER_SM = 2;
constexpr int GN_MAX_GRID = 2048;                     // slots of the workspace besides one per tensor
constexpr int GN_MAXE = 512;                          // tensors per launch
constexpr int GN_FINISH_THREADS = 1024;
// Sets of at most GN_SMALL small chunks of 16 KB, none of which spans two tensors, are one launch of
// one cluster, see grad_small_kernel.
constexpr int GN_CLUSTER = 8;
constexpr int GN_ROUNDS = 4;                          // chunks per CTA of the cluster
constexpr int GN_SMALL = GN_CLUSTER * GN_ROUNDS;
constexpr int GN_SMALL_THREADS = 1024;                // one vector per thread and chunk

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

// Chunks of `size` vectors in a tensor, at least one where only head or tail elements exist.
inline int64_t chunks_of(const Span& s, int64_t size) {
  const int64_t c = (s.vecs + size - 1) / size;
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

// The power of N vectors of one thread. Sums run in fp32 over these 4 N or 8 N values and
// join the double once: the conversions of every element would cost more than the loads. Where
// the fp32 sum left the range in which no term can have overflowed or lost bits that count
// (squares may underflow: 32 errors of at most 2^-150 are 2^-35 of 2^-110),
// the same registers are summed again in double.
template <int P, int DT, int N>
__device__ __forceinline__ double vec_power(const uint4 (&v)[N]) {
  constexpr int PAIR = DT == MSR_FP32 ? 1 : 2;
  const uint32_t* w = reinterpret_cast<const uint32_t*>(v);
  if (P == MSR_NORM_INF) {
    // magnitudes order as their bits do, NaN above infinity
    if (DT == MSR_FP32) {
      uint32_t m = 0u;
#pragma unroll
      for (int i = 0; i < 4 * N; ++i) m = max(m, w[i] & 0x7FFFFFFFu);
      const float x = __uint_as_float(m);
      return x != x ? positive_nan() : static_cast<double>(x);
    }
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < 4 * N; ++i) m = __vmaxu2(m, w[i] & 0x7FFF7FFFu);
    const uint16_t b = static_cast<uint16_t>(max(m & 0xFFFFu, m >> 16));
    const float x = DT == MSR_BF16 ? bf16_bits_to_f32(b) : __half2float(__ushort_as_half(b));
    return x != x ? positive_nan() : static_cast<double>(x);
  }
  float s[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4 * N; ++i) {
    float x[2];
    Elem<DT>::unpack(w[i], x);
#pragma unroll
    for (int j = 0; j < PAIR; ++j) {
      float& a = s[(i * PAIR + j) & 1];
      a = P == MSR_NORM_2 ? fmaf(x[j], x[j], a) : a + fabsf(x[j]);
    }
  }
  const float sum = s[0] + s[1];
  if (sum < 0x1p126f && (P == MSR_NORM_1 || sum > 0x1p-110f)) return sum;
  uint32_t any = 0u;
#pragma unroll
  for (int i = 0; i < 4 * N; ++i) any |= w[i];
  if ((any & (DT == MSR_FP32 ? 0x7FFFFFFFu : 0x7FFF7FFFu)) == 0u) return 0.0;
  double d = 0.0;
#pragma unroll
  for (int i = 0; i < 4 * N; ++i) {
    float x[2];
    Elem<DT>::unpack(w[i], x);
#pragma unroll
    for (int j = 0; j < PAIR; ++j) d += power_of<P>(x[j]);
  }
  return d;
}

// The elements of a tensor outside its vectors go with its first chunk.
template <int P, int DT>
__device__ __forceinline__ double ends_power(const typename Elem<DT>::type* p, int64_t n, const Span& s) {
  const int t = threadIdx.x;
  double acc = 0.0;
  if (t < s.head) acc = power_of<P>(Elem<DT>::get(p[t]));
  if (t < s.tail) acc = combine<P>(acc, power_of<P>(Elem<DT>::get(p[n - s.tail + t])));
  return acc;
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
    acc = combine<P>(acc, vec_power<P, DT>(v));
  }
  if (lo == 0) acc = combine<P>(acc, ends_power<P, DT>(p, n, s));
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

// Programmatic dependent launch: the finishing kernel is set up on the first SM that both CTAs of the
// power kernel have left (beside one of them its 1024 threads do not fit) while other SMs still
// sum, and reads the slots when that kernel has ended: 1 us less per norm. (The scaling kernels do
// without: their many CTAs gained nothing, 81 us either way for 90 M elements, and lost 5 us of
// 1760 on 1.9 G.)
__device__ __forceinline__ void allow_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void await_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// EACH: one slot per (block, tensor) pair, at block + tensor; otherwise one slot per block.
template <int P, bool EACH>
__global__ __launch_bounds__(GN_THREADS, GN_BLOCKS_PER_SM) void grad_power_kernel(const __grid_constant__ GradArgs a,
                                                                                 double* slots) {
  __shared__ double red[GN_THREADS / 32];
  allow_next();
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

__device__ __forceinline__ msr_clip_state state_of(double power, int p, double scale, double max_norm) {
  const double norm = root(power, p) * scale;
  // max_norm = infinity asks for no clipping, whatever the norm; a NaN norm makes coef NaN
  double coef = isinf(max_norm) ? 1.0 : max_norm / (norm + 1e-6);
  if (coef > 1.0) coef = 1.0;
  msr_clip_state st;
  st.power = power;
  st.norm = static_cast<float>(norm);
  st.factor = static_cast<float>(coef * scale);
  st.active = !(coef == 1.0 && scale == 1.0);
  st.reserved = 0;
  return st;
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
  await_previous();
  if (f.each) {
    // A warp per tensor, four tensors at once: the loads of their slots overlap, and few tensors
    // span more than 32 blocks.
    constexpr int WARPS = GN_FINISH_THREADS / 32, AT_ONCE = 4;
    const int64_t chunks = a.prefix[a.count];
    for (int t0 = warp; t0 < a.count; t0 += WARPS * AT_ONCE) {
      double x[AT_ONCE];
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) {
        const int t = t0 + u * WARPS;
        x[u] = 0.0;
        if (t < a.count && a.prefix[t + 1] > a.prefix[t]) {
          const int64_t b0 = block_of(a.prefix[t], chunks, f.grid), b1 = block_of(a.prefix[t + 1] - 1, chunks, f.grid);
          if (b0 + lane <= b1) x[u] = f.slots[b0 + lane + t];
          for (int64_t b = b0 + lane + 32; b <= b1; b += 32) x[u] = combine<P>(x[u], f.slots[b + t]);
        }
      }
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) x[u] = warp_power<P>(x[u]);
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) {
        const int t = t0 + u * WARPS;
        if (lane == 0 && t < a.count) {
          f.each[t] = static_cast<float>(root(x[u], P) * f.scale);
          acc = combine<P>(acc, x[u]);
        }
      }
    }
  } else {
    for (int64_t b = threadIdx.x; b < f.grid; b += GN_FINISH_THREADS) acc = combine<P>(acc, f.slots[b]);
  }
  acc = block_power<P>(acc, red);
  if (threadIdx.x == 0) {
    if (!f.first) acc = combine<P>(acc, f.state->power);
    if (f.last) *f.state = state_of(acc, P, f.scale, f.max_norm);
    else f.state->power = acc;
  }
}

__global__ void grad_factor_kernel(msr_clip_state* st, int p, double scale, double max_norm) {
  *st = state_of(st->power, p, scale, max_norm);
}

// ---------------------------------------------------------------------------------------
// Scaling. Blocks take groups of `group` consecutive chunks in turn, the last group of all
// first and the last chunk of a group first; with group 0, each takes one stretch, the power
// kernel's.
// ---------------------------------------------------------------------------------------
template <int DT>
__device__ __forceinline__ uint4 scaled(uint4 v, float f) {
  constexpr int PAIR = DT == MSR_FP32 ? 1 : 2;
  uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    float x[2];
    Elem<DT>::unpack(w[q], x);
#pragma unroll
    for (int j = 0; j < PAIR; ++j) x[j] = __fmul_rn(x[j], f);
    w[q] = Elem<DT>::pack(x);
  }
  return v;
}

// The elements of a tensor outside its vectors.
template <int DT>
__device__ __forceinline__ void scale_ends(typename Elem<DT>::type* p, int64_t n, const Span& s, float f) {
  const int t = threadIdx.x;
  if (t < s.head) p[t] = Elem<DT>::put(__fmul_rn(Elem<DT>::get(p[t]), f));
  if (t < s.tail) p[n - s.tail + t] = Elem<DT>::put(__fmul_rn(Elem<DT>::get(p[n - s.tail + t]), f));
}

template <int DT>
__device__ __forceinline__ void span_scale(void* ptr, int64_t n, int64_t lo, int64_t hi, float f) {
  using T = typename Elem<DT>::type;
  constexpr int STEP = GN_SCALE_THREADS * GN_SCALE_VECS;
  const Span s = span_of(ptr, n, DT);
  T* p = static_cast<T*>(ptr);
  uint4* body = reinterpret_cast<uint4*>(p + s.head);
  const int64_t first = lo * GN_CHUNK, last = min(hi * GN_CHUNK, s.vecs);
  for (int64_t at = last - STEP; at > first - STEP; at -= STEP) {
    uint4 v[GN_SCALE_VECS];
#pragma unroll
    for (int k = 0; k < GN_SCALE_VECS; ++k) {
      const int64_t i = at + k * GN_SCALE_THREADS + threadIdx.x;
      if (i >= first) v[k] = body[i];
    }
#pragma unroll
    for (int k = 0; k < GN_SCALE_VECS; ++k) {
      const int64_t i = at + k * GN_SCALE_THREADS + threadIdx.x;
      if (i >= first) __stcs(body + i, scaled<DT>(v[k], f));  // evicted before what is still to be read
    }
  }
  if (lo == 0) scale_ends<DT>(p, n, s, f);
}

__device__ __forceinline__ void scale_chunks(const GradArgs& a, int64_t group, float f) {
  const int64_t chunks = a.prefix[a.count];
  int64_t top = group ? chunks - blockIdx.x * group : first_chunk(blockIdx.x + 1, chunks, gridDim.x);
  for (; top > 0; top -= gridDim.x * group) {
    const int64_t begin = group ? max(top - group, static_cast<int64_t>(0)) : first_chunk(blockIdx.x, chunks, gridDim.x);
    int64_t c = top;
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
    if (!group) break;
  }
}

__global__ __launch_bounds__(GN_SCALE_THREADS, GN_SCALE_BLOCKS_PER_SM) void grad_scale_kernel(
    const __grid_constant__ GradArgs a, const msr_clip_state* st, int64_t group) {
  if (st->active) scale_chunks(a, group, st->factor);  // else the gradients stay as they are
}

// grad_finish_kernel and grad_scale_kernel in one: every block sums the slots of the power
// kernel (at most GN_MAX_GRID doubles, from L2) in the same order, so all blocks agree on the
// factor, and one launch and its gap are saved.
template <int P>
__global__ __launch_bounds__(GN_SCALE_THREADS, GN_SCALE_BLOCKS_PER_SM) void grad_clip_kernel(
    const __grid_constant__ GradArgs a, const __grid_constant__ FinishArgs f, int64_t group) {
  __shared__ double red[GN_SCALE_THREADS / 32];
  double acc = 0.0;
  for (int64_t b = threadIdx.x; b < f.grid; b += GN_SCALE_THREADS) acc = combine<P>(acc, f.slots[b]);
  const msr_clip_state st = state_of(block_power<P>(acc, red), P, f.scale, f.max_norm);
  if (blockIdx.x == 0 && threadIdx.x == 0) *f.state = st;
  if (st.active) scale_chunks(a, group, st.factor);
}

// ---------------------------------------------------------------------------------------
// Small sets: one cluster holds every gradient in its registers, so norm and scaling are one
// launch and one read. CTA r of the cluster takes chunks r, r + 8, r + 16, r + 24; the powers
// of the chunks meet in distributed shared memory. The host describes each chunk by itself: a
// search for the chunk's tensor would be a chain of parameter reads, each missing the cache.
// Against the two kernels, from a graph over three sets in turn, in us: norm 3.0 / 4.5 at 16 KB,
// 3.8 / 4.3 at 256 KB, 4.6 / 4.3 at 512 KB; clip 3.9 / 5.8, 4.8 / 6.4, 6.3 / 6.2; twelve tensors of
// 256 KB together 4.5 / 4.6 and 6.5 / 6.7. So the two meet where the cluster's registers end, and
// up to there its launch costs the host 4.5 us less (8.9 / 13.5 from Python's ctypes).
// ---------------------------------------------------------------------------------------
struct SmallChunk {
  char* body;  // vectors of this chunk
  char* tail;  // the elements after the tensor's last vector
  int16_t vecs;
  uint8_t head, tails;  // elements before body and at tail (first chunk of a tensor only)
  uint8_t dtype;
  uint8_t entry;
};

struct SmallArgs {
  SmallChunk c[GN_SMALL];
  int chunks, count;
};

template <int P, int DT>
__device__ __forceinline__ double small_power(const SmallChunk& c, const uint4& v) {
  using T = typename Elem<DT>::type;
  const uint4 one[1] = {v};
  double acc = vec_power<P, DT>(one);
  const int t = threadIdx.x;
  if (t < c.head) acc = combine<P>(acc, power_of<P>(Elem<DT>::get(*(reinterpret_cast<const T*>(c.body) - 1 - t))));
  if (t < c.tails) acc = combine<P>(acc, power_of<P>(Elem<DT>::get(reinterpret_cast<const T*>(c.tail)[t])));
  return acc;
}

template <int DT>
__device__ __forceinline__ void small_scale(const SmallChunk& c, const uint4& v, float f) {
  using T = typename Elem<DT>::type;
  const int t = threadIdx.x;
  if (t < c.vecs) reinterpret_cast<uint4*>(c.body)[t] = scaled<DT>(v, f);
  T* head = reinterpret_cast<T*>(c.body) - 1 - t;
  if (t < c.head) *head = Elem<DT>::put(__fmul_rn(Elem<DT>::get(*head), f));
  T* tail = reinterpret_cast<T*>(c.tail) + t;
  if (t < c.tails) *tail = Elem<DT>::put(__fmul_rn(Elem<DT>::get(*tail), f));
}

template <int P, bool SCALE>
__global__ __cluster_dims__(GN_CLUSTER, 1, 1) __launch_bounds__(GN_SMALL_THREADS, 1) void grad_small_kernel(
    const __grid_constant__ SmallArgs a, const __grid_constant__ FinishArgs f) {
  __shared__ double red[GN_ROUNDS][GN_SMALL_THREADS / 32];
  __shared__ double chunk[GN_ROUNDS];
  __shared__ double all[GN_SMALL];
  __shared__ msr_clip_state st;
  cg::cluster_group cluster = cg::this_cluster();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint4 v[GN_ROUNDS];
#pragma unroll
  for (int k = 0; k < GN_ROUNDS; ++k) {  // every load before the first use
    const int c = blockIdx.x + k * GN_CLUSTER;
    v[k] = make_uint4(0u, 0u, 0u, 0u);
    if (c < a.chunks && threadIdx.x < a.c[c].vecs) v[k] = reinterpret_cast<const uint4*>(a.c[c].body)[threadIdx.x];
  }
#pragma unroll
  for (int k = 0; k < GN_ROUNDS; ++k) {
    const int c = blockIdx.x + k * GN_CLUSTER;
    double x = 0.0;
    if (c < a.chunks) {
      if (a.c[c].dtype == MSR_BF16) x = small_power<P, MSR_BF16>(a.c[c], v[k]);
      else if (a.c[c].dtype == MSR_FP16) x = small_power<P, MSR_FP16>(a.c[c], v[k]);
      else x = small_power<P, MSR_FP32>(a.c[c], v[k]);
      x = warp_power<P>(x);
    }
    if (lane == 0) red[k][warp] = x;
  }
  __syncthreads();
  if (warp < GN_ROUNDS) {
    const double x = warp_power<P>(red[warp][lane]);
    if (lane == 0) chunk[warp] = x;
  }
  cluster.sync();
  if (warp == 0) {
    const double x = *cluster.map_shared_rank(&chunk[lane / GN_CLUSTER], lane % GN_CLUSTER);  // of chunk `lane`
    const msr_clip_state s = state_of(warp_power<P>(x), P, f.scale, f.max_norm);
    if (lane == 0) {
      st = s;
      if (blockIdx.x == 0) *f.state = s;
    }
    all[lane] = x;
  }
  __syncthreads();
  if (f.each && blockIdx.x == 0 && warp < a.count) {  // warp t: the chunks of tensor t
    const double y = warp_power<P>(lane < a.chunks && a.c[lane].entry == warp ? all[lane] : 0.0);
    if (lane == 0) f.each[warp] = static_cast<float>(root(y, P) * f.scale);
  }
  cluster.barrier_arrive();  // warp 0 has read the other CTAs' powers: they may leave
  if (SCALE && st.active) {
    const float factor = st.factor;
#pragma unroll
    for (int k = 0; k < GN_ROUNDS; ++k) {
      const int c = blockIdx.x + k * GN_CLUSTER;
      if (c >= a.chunks) break;
      if (a.c[c].dtype == MSR_BF16) small_scale<MSR_BF16>(a.c[c], v[k], factor);
      else if (a.c[c].dtype == MSR_FP16) small_scale<MSR_FP16>(a.c[c], v[k], factor);
      else small_scale<MSR_FP32>(a.c[c], v[k], factor);
    }
  }
  cluster.barrier_wait();
}

// ---------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------
int grid_for(int64_t chunks, int blocks_per_sm) {
  const int64_t cap = std::min<int64_t>(static_cast<int64_t>(sm_count()) * blocks_per_sm, GN_MAX_GRID);
  return static_cast<int>(std::min<int64_t>(chunks, cap));
}

// How the scaling kernels share out the chunks. Up to a few times the L2 cache (126 MB), every
// block takes one stretch, as in the power kernel, and begins at its end, which that kernel read
// last. Beyond, the groups of 2 of all blocks form one window that moves through memory, which DRAM
// serves better. Clipping 24 bf16 tensors, three sets in turn, stretches against groups in us:
// 64 MB 35.1 / 37.3, 180 MB 92.2 / 94.4, 256 MB 132.8 / 134.0, 400 MB 207.9 / 207.3, 600 MB
// 307 / 303, 1200 MB 601 / 585, 3840 MB 1892 / 1854.
constexpr int64_t GN_STRETCH_BYTES = int64_t(384) << 20;
struct ScaleShape {
  int grid;
  int64_t group;
};
ScaleShape scale_shape(int64_t chunks) {
  const int grid = grid_for(chunks, GN_SCALE_BLOCKS_PER_SM);
  return {grid, chunks * GN_CHUNK * 16 <= GN_STRETCH_BYTES ? 0 : 2};
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

int check_state(const msr_clip_state* state, const char* what) {
  if (!state || reinterpret_cast<uintptr_t>(state) % 8)
    return fail(MSR_ERR_INVALID, "%s: state must be an 8-byte aligned device pointer", what);
  return MSR_OK;
}

int check_factor(int norm, double scale, double max_norm, const char* what) {
  if (norm != MSR_NORM_INF && norm != MSR_NORM_1 && norm != MSR_NORM_2)
    return fail(MSR_ERR_INVALID, "%s: unknown norm %d", what, norm);
  if (!(scale >= FLT_MIN && scale <= FLT_MAX))
    return fail(MSR_ERR_INVALID, "%s: scale must be positive and within the range of fp32", what);
  if (!(max_norm >= 0.0)) return fail(MSR_ERR_INVALID, "%s: max_norm must be >= 0", what);
  return MSR_OK;
}

// The table of up to GN_MAXE entries from `begin` on and its number of chunks.
int64_t fill_table(GradArgs& a, const msr_grad_entry* e, int begin, int count) {
  a.count = std::min(count - begin, GN_MAXE);
  int64_t chunks = 0;
  for (int i = 0; i < a.count; ++i) {
    const msr_grad_entry& x = e[begin + i];
    a.ptr[i] = x.grad;
    a.numel[i] = x.numel;
    a.dtype[i] = static_cast<uint8_t>(x.dtype);
    a.prefix[i] = chunks;
    if (x.numel > 0) chunks += chunks_of(span_of(x.grad, x.numel, x.dtype), GN_CHUNK);
  }
  a.prefix[a.count] = chunks;
  return chunks;
}

// A launch that may be set up before the kernel ahead of it on the stream has ended.
template <class... Params, class... Args>
int launch_after(const char* name, void (*kernel)(Params...), int grid, int threads, cudaStream_t stream,
                 const Args&... args) {
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(grid);
  config.blockDim = dim3(threads);
  config.stream = stream;
  config.attrs = &attr;
  config.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&config, kernel, static_cast<Params>(args)...);
  if (e != cudaSuccess) return fail(MSR_ERR_CUDA, "%s: %s", name, cudaGetErrorString(e));
  return check_launch(name);
}

struct NormCall {
  const msr_grad_entry* entries;
  int count;
  double scale, max_norm;
  msr_clip_state* state;
  float* each;
  double* slots;
  cudaStream_t stream;
};

// One launch for sets that one cluster holds; false where it does not.
template <int P, bool SCALE>
bool small_launch(const NormCall& call, int* status) {
  if (call.count > GN_SMALL) return false;
  SmallArgs a;
  a.count = call.count;
  a.chunks = 0;
  for (int t = 0; t < call.count; ++t) {
    const msr_grad_entry& x = call.entries[t];
    if (x.numel == 0) continue;
    const Span s = span_of(x.grad, x.numel, x.dtype);
    const int64_t chunks = chunks_of(s, GN_SMALL_THREADS);
    if (a.chunks + chunks > GN_SMALL) return false;
    const int es = dtype_bytes(x.dtype);
    char* body = static_cast<char*>(x.grad) + s.head * es;
    for (int64_t i = 0; i < chunks; ++i) {
      SmallChunk& c = a.c[a.chunks++];
      c.body = body + i * GN_SMALL_THREADS * 16;
      c.tail = body + s.vecs * 16;
      c.vecs = static_cast<int16_t>(std::min<int64_t>(GN_SMALL_THREADS, s.vecs - i * GN_SMALL_THREADS));
      c.head = static_cast<uint8_t>(i == 0 ? s.head : 0);
      c.tails = static_cast<uint8_t>(i == 0 ? s.tail : 0);
      c.dtype = static_cast<uint8_t>(x.dtype);
      c.entry = static_cast<uint8_t>(t);
    }
  }
  FinishArgs f{nullptr, call.state, call.each, call.scale, call.max_norm, 0, 1, 1};
  grad_small_kernel<P, SCALE><<<GN_CLUSTER, GN_SMALL_THREADS, 0, call.stream>>>(a, f);
  *status = check_launch("grad_small_kernel");
  return true;
}

template <int P>
int norm_launch(const NormCall& c) {
  int status;
  if (small_launch<P, false>(c, &status)) return status;
  int begin = 0;
  do {
    GradArgs a;
    const int64_t chunks = fill_table(a, c.entries, begin, c.count);
    const int grid = grid_for(chunks, GN_BLOCKS_PER_SM);
    if (grid > 0) {
      if (c.each) grad_power_kernel<P, true><<<grid, GN_THREADS, 0, c.stream>>>(a, c.slots);
      else grad_power_kernel<P, false><<<grid, GN_THREADS, 0, c.stream>>>(a, c.slots);
      if (int st = check_launch("grad_power_kernel")) return st;
    }
    FinishArgs f{c.slots, c.state, c.each ? c.each + begin : nullptr, c.scale, c.max_norm, grid, begin == 0,
                 begin + a.count >= c.count};
    if (int st = launch_after("grad_finish_kernel", grad_finish_kernel<P>, 1, GN_FINISH_THREADS, c.stream, a, f))
      return st;
    begin += a.count;
  } while (begin < c.count);
  return MSR_OK;
}

int scale_launch(const msr_grad_entry* entries, int count, const msr_clip_state* state, cudaStream_t stream) {
  for (int begin = 0; begin < count; begin += GN_MAXE) {
    GradArgs a;
    const int64_t chunks = fill_table(a, entries, begin, count);
    if (chunks == 0) continue;
    const ScaleShape g = scale_shape(chunks);
    grad_scale_kernel<<<g.grid, GN_SCALE_THREADS, 0, stream>>>(a, state, g.group);
    if (int st = check_launch("grad_scale_kernel")) return st;
  }
  return MSR_OK;
}

template <int P>
int clip_launch(const NormCall& c) {
  int status;
  if (small_launch<P, true>(c, &status)) return status;
  if (c.count > GN_MAXE) {  // the factor needs every table's powers before the first is scaled
    if (int st = norm_launch<P>(c)) return st;
    return scale_launch(c.entries, c.count, c.state, c.stream);
  }
  GradArgs a;
  const int64_t chunks = fill_table(a, c.entries, 0, c.count);
  const int grid = grid_for(chunks, GN_BLOCKS_PER_SM);
  if (grid == 0) return norm_launch<P>(c);
  grad_power_kernel<P, false><<<grid, GN_THREADS, 0, c.stream>>>(a, c.slots);
  if (int st = check_launch("grad_power_kernel")) return st;
  FinishArgs f{c.slots, c.state, nullptr, c.scale, c.max_norm, grid, 1, 1};
  const ScaleShape g = scale_shape(chunks);
  grad_clip_kernel<P><<<g.grid, GN_SCALE_THREADS, 0, c.stream>>>(a, f, g.group);
  return check_launch("grad_clip_kernel");
}

// Two entries of one scaling launch must not share memory: both would multiply it.
int check_apart(const msr_grad_entry* e, int count, const char* what) try {
  std::vector<std::pair<uintptr_t, uintptr_t>> r;
  r.reserve(count);
  for (int i = 0; i < count; ++i)
    if (e[i].numel > 0) {
      const uintptr_t p = reinterpret_cast<uintptr_t>(e[i].grad);
      r.emplace_back(p, p + static_cast<uintptr_t>(e[i].numel) * dtype_bytes(e[i].dtype));
    }
  std::sort(r.begin(), r.end());
  for (size_t i = 1; i < r.size(); ++i)
    if (r[i].first < r[i - 1].second) return fail(MSR_ERR_INVALID, "%s: two gradients overlap in memory", what);
  return MSR_OK;
} catch (...) {
  return fail(MSR_ERR_INVALID, "%s: out of host memory", what);
}

int check_norm(const msr_grad_entry* entries, int count, int norm, double scale, double max_norm,
               const msr_clip_state* state, const void* workspace, size_t bytes, const char* what) {
  if (int st = check_entries(entries, count, what)) return st;
  if (int st = check_factor(norm, scale, max_norm, what)) return st;
  if (int st = check_state(state, what)) return st;
  if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 8)
    return fail(MSR_ERR_INVALID, "%s: workspace must be an 8-byte aligned device pointer", what);
  const size_t need = msr_grad_norm_workspace_bytes(count);
  if (bytes < need) return fail(MSR_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", what, bytes, need);
  return require_sm100();
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
  if (reinterpret_cast<uintptr_t>(each) % 4) return fail(MSR_ERR_INVALID, "msr_grad_norm: each is not 4-byte aligned");
  if (int st = check_norm(entries, count, norm, scale, max_norm, state, workspace, workspace_bytes, "msr_grad_norm"))
    return st;
  const NormCall c{entries, count, scale, max_norm, state, each, static_cast<double*>(workspace), to_stream(stream)};
  switch (norm) {
    case MSR_NORM_INF: return norm_launch<MSR_NORM_INF>(c);
    case MSR_NORM_1: return norm_launch<MSR_NORM_1>(c);
    default: return norm_launch<MSR_NORM_2>(c);
  }
}

int msr_grad_factor(msr_clip_state* state, int norm, double scale, double max_norm, msr_stream_t stream) {
  if (int st = check_factor(norm, scale, max_norm, "msr_grad_factor")) return st;
  if (int st = check_state(state, "msr_grad_factor")) return st;
  grad_factor_kernel<<<1, 1, 0, to_stream(stream)>>>(state, norm, scale, max_norm);
  return check_launch("grad_factor_kernel");
}

int msr_grad_scale(const msr_grad_entry* entries, int count, const msr_clip_state* state, msr_stream_t stream) {
  if (int st = check_entries(entries, count, "msr_grad_scale")) return st;
  if (int st = check_state(state, "msr_grad_scale")) return st;
  if (int st = check_apart(entries, count, "msr_grad_scale")) return st;
  return scale_launch(entries, count, state, to_stream(stream));
}

int msr_grad_clip(const msr_grad_entry* entries, int count, int norm, double scale, double max_norm,
                  msr_clip_state* state, void* workspace, size_t workspace_bytes, msr_stream_t stream) {
  if (int st = check_norm(entries, count, norm, scale, max_norm, state, workspace, workspace_bytes, "msr_grad_clip"))
    return st;
  if (int st = check_apart(entries, count, "msr_grad_clip")) return st;
  const NormCall c{entries, count, scale, max_norm, state, nullptr, static_cast<double*>(workspace), to_stream(stream)};
  switch (norm) {
    case MSR_NORM_INF: return clip_launch<MSR_NORM_INF>(c);
    case MSR_NORM_1: return clip_launch<MSR_NORM_1>(c);
    default: return clip_launch<MSR_NORM_2>(c);
  }
}

}  // extern "C"
