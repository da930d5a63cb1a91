// global_norm, clip_by_global_norm: n = sqrt(sum over all tensors of g^2), and
// every g times c = max_norm / n where n > max_norm, else unchanged.  The factor
// and its products are held in 64 bits too: next to gradients of 1e38 it is
// smaller than the smallest normal fp32 number.
//
// Squares are summed in 64 bits: no finite fp32 or bf16 gradient overflows or
// vanishes in its square, and 2^53 leaves the order of summation without
// effect on the 32-bit result.  The order is fixed all the same (a block's
// share, then the blocks in order), so equal inputs give equal bits.
#include "grad_clip.h"
#include "int8.h"

namespace {

using namespace des;

constexpr int THREADS = 256;

__device__ __forceinline__ double block_sum(double v, double* red) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = 0.0;
  for (int i = 0; i < (int)blockDim.x / 64; ++i) s += red[i];
  return s;
}

// the tensor of block b
__device__ __forceinline__ int tensor_of(const DesClipTable& t, int b) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= b) lo = mid; else hi = mid - 1;
  }
  return lo;
}

template <typename T>
__device__ double share_sum(const void* in, int64_t begin, int64_t end) {
  const T* p = (const T*)in;
  double s = 0.0;
  for (int64_t i = begin + threadIdx.x; i < end; i += THREADS) {
    const double v = (double)to_f32(p[i]);
    s += v * v;
  }
  return s;
}

__global__ __launch_bounds__(THREADS) void square_sums_kernel(
    DesClipTable t, int64_t share, double* __restrict__ sums) {
  __shared__ double red[THREADS / 64];
  const int b = blockIdx.x, i = tensor_of(t, b);
  const int64_t begin = (b - t.first[i]) * share;
  const int64_t end = min(begin + share, t.numel[i]);
  const double s = t.elem[i] == ELEM_F32 ? share_sum<float>(t.in[i], begin, end)
                   : t.elem[i] == ELEM_BF16
                       ? share_sum<Bf16>(t.in[i], begin, end)
                       : share_sum<_Float16>(t.in[i], begin, end);
  const double all = block_sum(s, red);
  if (threadIdx.x == 0) sums[b] = all;
}

__device__ double norm_of(const double* sums, int n, double* red) {
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += THREADS) s += sums[i];
  return sqrt(block_sum(s, red));
}

__global__ __launch_bounds__(THREADS) void norm_kernel(
    const double* __restrict__ sums, int n, float* __restrict__ norm) {
  __shared__ double red[THREADS / 64];
  const double v = norm_of(sums, n, red);
  if (threadIdx.x == 0) *norm = (float)v;
}

template <typename T>
__device__ void share_scale(const void* in, void* out, int64_t begin,
                            int64_t end, double c) {
  const T* p = (const T*)in;
  T* o = (T*)out;
  for (int64_t i = begin + threadIdx.x; i < end; i += THREADS)
    o[i] = from_f32<T>((float)((double)to_f32(p[i]) * c));
}

// Every block joins the sums by itself, in the same order: cheaper than a
// launch of its own for one number.
__global__ __launch_bounds__(THREADS) void scale_kernel(
    DesClipTable t, int64_t share, const double* __restrict__ sums, int n,
    double max_norm, float* __restrict__ norm, bool write_norm) {
  __shared__ double red[THREADS / 64];
  const double v = norm_of(sums, n, red);
  const double c = v > max_norm ? max_norm / v : 1.0;
  const int b = blockIdx.x, i = tensor_of(t, b);
  if (write_norm && b == 0 && threadIdx.x == 0) *norm = (float)v;
  const int64_t begin = (b - t.first[i]) * share;
  const int64_t end = min(begin + share, t.numel[i]);
  if (t.elem[i] == ELEM_F32)
    share_scale<float>(t.in[i], t.out[i], begin, end, c);
  else if (t.elem[i] == ELEM_BF16)
    share_scale<Bf16>(t.in[i], t.out[i], begin, end, c);
  else
    share_scale<_Float16>(t.in[i], t.out[i], begin, end, c);
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
                                      bool write_norm, hipStream_t stream) {
  hipLaunchKernelGGL(scale_kernel, dim3((uint32_t)t->first[t->count]),
                     dim3(THREADS), 0, stream, *t, share, sums, n, max_norm,
                     norm, write_norm);
}
