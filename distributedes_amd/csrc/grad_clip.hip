// global_norm, clip_by_global_norm: n = sqrt(sum over all tensors of g^2), and
// every g times c = max_norm / n where n > max_norm, else unchanged.  The factor
// and its products are held in 64 bits too: next to gradients of 1e38 it is
// smaller than the smallest normal fp32 number.
//
// Squares are summed in 64 bits: no finite fp32 or bf16 gradient overflows or
// vanishes in its square, and the sum loses 2^-40 of its size at most: the 32-bit
// norm is the exact one rounded, or its neighbour where the exact one lies that
// near to the middle of two.  The order of summation is fixed (a block's share, then the blocks in
// order), so equal inputs give equal bits.
#include "grad_clip.h"
#include "int8.h"

//
// Memory bound: the tensors are read for the norm and once more to be scaled,
// since no value can be written before the last is read.  Where they are large
// the second pass goes past the caches, so that they keep what the first has
// read until it is read again: 168 MB of bf16 107 us through the caches, 93 with
// stores past them, 83 with loads too, 87 backwards from the first pass's end.
#include <algorithm>

namespace {

using namespace des;

constexpr int THREADS = 256;
constexpr int SMALL = 1024;  // threads of the block that does all by itself

template <int T>
__device__ __forceinline__ double block_sum(double v, double* red) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < T / 64; ++i) s += red[i];
  return s;
}

// The tensor of share u: as many begin at or before it.  A lane looks at one of
// them (and one 64 on), which takes one memory access instead of a search's 7.
__device__ __forceinline__ int tensor_of(const DesClipTable& t, int u) {
  static_assert(DES_CLIP_TENSORS <= 128, "two tensors a lane");
  const int a = threadIdx.x & 63, b = a + 64;
  const bool at_a = a < t.count && t.first[min(a, DES_CLIP_TENSORS)] <= u;
  const bool at_b = b < t.count && t.first[min(b, DES_CLIP_TENSORS)] <= u;
  return __popcll(__ballot(at_a)) + __popcll(__ballot(at_b)) - 1;
}

// [begin, end) of a tensor, in pieces of 16 bytes at any address, four under
// way a thread
template <typename T, int N>
__device__ double share_sum(const void* in, int64_t begin, int64_t end,
                            int tid) {
  constexpr int V = 16 / sizeof(T);
  const T* p = (const T*)in;
  double s[V] = {};
  int64_t i = begin + tid * V;
  auto add = [&](const Vec<T, V>& t) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const double v = (double)to_f32(t.v[j]);
      s[j] = fma(v, v, s[j]);
    }
  };
  for (; i + 3 * N * V + V <= end; i += 4 * N * V) {
    Vec<T, V> t[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      t[u] = *reinterpret_cast<const Vec<T, V>*>(p + i + u * N * V);
#pragma unroll
    for (int u = 0; u < 4; ++u) add(t[u]);
  }
  for (; i + V <= end; i += N * V)
    add(*reinterpret_cast<const Vec<T, V>*>(p + i));
  i = end - (end - begin) % V + tid;  // what is left, a value a thread
  if (i < end) {
    const double v = (double)to_f32(p[i]);
    s[0] = fma(v, v, s[0]);
  }
  double all = 0.0;
#pragma unroll
  for (int j = 0; j < V; ++j) all += s[j];
  return all;
}

typedef __attribute__((ext_vector_type(4), aligned(2))) uint32_t u32x4_any;

template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load_past(const T* p) {
  const u32x4_any t =
      __builtin_nontemporal_load(reinterpret_cast<const u32x4_any*>(p));
  Vec<T, V> v;
  __builtin_memcpy(&v, &t, 16);
  return v;
}

template <typename T, int V>
__device__ __forceinline__ void store_past(T* p, const Vec<T, V>& v) {
  u32x4_any t;
  __builtin_memcpy(&t, &v, 16);
  __builtin_nontemporal_store(t, reinterpret_cast<u32x4_any*>(p));
}

// `factor()` joins the block for c; the first pieces are on their way meanwhile.
template <typename T, int N, bool PAST, typename F>
__device__ __forceinline__ void share_scale(const void* in, void* out,
                                            int64_t begin, int64_t end,
                                            F factor, int tid) {
  constexpr int V = 16 / sizeof(T);
  const T* p = (const T*)in;
  T* o = (T*)out;
  int64_t i = begin + tid * V;
  Vec<T, V> t[4];
  auto get = [&] {
#pragma unroll
    for (int u = 0; u < 4; ++u)
      t[u] = PAST ? load_past<T, V>(p + i + u * N * V)
                  : *reinterpret_cast<const Vec<T, V>*>(p + i + u * N * V);
  };
  bool full = i + 3 * N * V + V <= end;
  if (full) get();
  const double c = factor();
  if (c == 1.0 && in == out) return;  // in place, nothing to do
  auto put = [&](int64_t at, const Vec<T, V>& t) {
    Vec<T, V> r;
#pragma unroll
    for (int j = 0; j < V; ++j)
      r.v[j] = from_f32<T>((float)((double)to_f32(t.v[j]) * c));
    if constexpr (PAST) store_past<T, V>(o + at, r);
    else *reinterpret_cast<Vec<T, V>*>(o + at) = r;
  };
  while (full) {
#pragma unroll
    for (int u = 0; u < 4; ++u) put(i + u * N * V, t[u]);
    i += 4 * N * V;
    full = i + 3 * N * V + V <= end;
    if (full) get();
  }
  for (; i + V <= end; i += N * V)
    put(i, *reinterpret_cast<const Vec<T, V>*>(p + i));
  i = end - (end - begin) % V + tid;
  if (i < end) o[i] = from_f32<T>((float)((double)to_f32(p[i]) * c));
}

// share u of all, by N threads
template <int N>
__device__ double any_sum(const DesClipTable& t, int u, int64_t share,
                          int tid) {
  const int i = tensor_of(t, u);
  const int64_t begin = (u - t.first[i]) * share;
  const int64_t end = min(begin + share, t.numel[i]);
  if (t.elem[i] == ELEM_F32)
    return share_sum<float, N>(t.in[i], begin, end, tid);
  if (t.elem[i] == ELEM_BF16)
    return share_sum<Bf16, N>(t.in[i], begin, end, tid);
  return share_sum<_Float16, N>(t.in[i], begin, end, tid);
}

template <int N, bool PAST, typename F>
__device__ __forceinline__ void any_scale(const DesClipTable& t, int u,
                                          int64_t share, F factor, int tid) {
  const int i = tensor_of(t, u);
  const int64_t begin = (u - t.first[i]) * share;
  const int64_t end = min(begin + share, t.numel[i]);
  if (t.elem[i] == ELEM_F32)
    share_scale<float, N, PAST>(t.in[i], t.out[i], begin, end, factor, tid);
  else if (t.elem[i] == ELEM_BF16)
    share_scale<Bf16, N, PAST>(t.in[i], t.out[i], begin, end, factor, tid);
  else
    share_scale<_Float16, N, PAST>(t.in[i], t.out[i], begin, end, factor, tid);
}

__global__ __launch_bounds__(THREADS) void square_sums_kernel(
    DesClipTable t, int64_t share, double* __restrict__ sums) {
  __shared__ double red[THREADS / 64];
  const double all = block_sum<THREADS>(
      any_sum<THREADS>(t, blockIdx.x, share, threadIdx.x), red);
  if (threadIdx.x == 0) sums[blockIdx.x] = all;
}

__device__ double norm_of(const double* sums, int n, double* red) {
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += THREADS) s += sums[i];
  return sqrt(block_sum<THREADS>(s, red));
}

__global__ __launch_bounds__(THREADS) void norm_kernel(
    const double* __restrict__ sums, int n, float* __restrict__ norm) {
  __shared__ double red[THREADS / 64];
  const double v = norm_of(sums, n, red);
  if (threadIdx.x == 0) *norm = (float)v;
}

// Every block joins the sums by itself, in the same order: cheaper than a
// launch of its own for one number.
template <bool PAST>
__global__ __launch_bounds__(THREADS) void scale_kernel(
    DesClipTable t, int64_t share, const double* __restrict__ sums, int n,
    double max_norm, float* __restrict__ norm, bool write_norm) {
  __shared__ double red[THREADS / 64];
  auto factor = [&] {
    const double v = norm_of(sums, n, red);
    if (write_norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)v;
    return v > max_norm ? max_norm / v : 1.0;
  };
  any_scale<THREADS, PAST>(t, blockIdx.x, share, factor, threadIdx.x);
}

// Norm and scaling of a few small tensors by one block, a wave for each share
// (a tensor after the other took 7.3 us for six of them, by latency alone).
__global__ __launch_bounds__(SMALL) void small_kernel(DesClipTable t,
                                                      int64_t share,
                                                      double max_norm,
                                                      float* __restrict__ norm,
                                                      bool scale) {
  __shared__ double red[SMALL / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int shares = t.first[t.count];
  double s = 0.0;
  for (int u = wave; u < shares; u += SMALL / 64)
    s += any_sum<64>(t, u, share, lane);
  const double v = sqrt(block_sum<SMALL>(s, red));
  if (threadIdx.x == 0) *norm = (float)v;
  if (!scale) return;
  const double c = v > max_norm ? max_norm / v : 1.0;
  for (int u = wave; u < shares; u += SMALL / 64)
    any_scale<64, false>(t, u, share, [&] { return c; }, lane);
}

}  // namespace

extern "C" void des_launch_square_sums(const DesClipTable* t, int64_t share,
                                       double* sums, hipStream_t stream) {
  hipLaunchKernelGGL(square_sums_kernel, dim3((uint32_t)t->first[t->count]),
                     dim3(THREADS), 0, stream, *t, share, sums);
}

extern "C" void des_launch_norm(const double* sums, int n, float* norm,
                                hipStream_t stream) {
  hipLaunchKernelGGL(norm_kernel, dim3(1), dim3(THREADS), 0, stream, sums, n,
                     norm);
}

extern "C" void des_launch_clip_scale(const DesClipTable* t, int64_t share,
                                      const double* sums, int n,
                                      double max_norm, float* norm,
                                      bool write_norm, bool past,
                                      hipStream_t stream) {
  hipLaunchKernelGGL(past ? scale_kernel<true> : scale_kernel<false>,
                     dim3((uint32_t)t->first[t->count]), dim3(THREADS), 0,
                     stream, *t, share, sums, n, max_norm, norm, write_norm);
}

extern "C" void des_launch_clip_small(const DesClipTable* t, int64_t share,
                                      double max_norm, float* norm, bool scale,
                                      hipStream_t stream) {
  hipLaunchKernelGGL(small_kernel, dim3(1), dim3(SMALL), 0, stream, *t, share,
                     max_norm, norm, scale);
}
