// int8_matmul: y[m, n] = act(float(sum_k x[m, k] w[n, k]) * sx[m] * sw[n] + b[n])
//
// Sums of products of codes are held in 32-bit integers: exact up to
// K = 2^31 / 127^2 = 133144 (the bindings allow 131072), whatever the order.
#include "int8.h"

namespace {

using namespace des;

typedef __attribute__((ext_vector_type(4))) int v4i;

// 16 codes from any address; those at and behind `left` are 0 and not read
__device__ __forceinline__ v4i load16(const int8_t* p, int left) {
  union { v4i v; int8_t b[16]; } u;
  u.v = v4i{0, 0, 0, 0};
  if (left >= 16) {
    __builtin_memcpy(&u.v, p, 16);
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (j < left) u.b[j] = p[j];
  }
  return u.v;
}

__device__ __forceinline__ float finish(int sum, float sx, float sw, float b,
                                        int act) {
  float v = (float)sum * sx * sw + b;
  if (act == 1) v = v < 0.f ? 0.f : v;  // a NaN stays one
  if (act == 2) v = tanhf(v);
  return v;
}

template <typename T>
__device__ __forceinline__ void put(void* y, int64_t at, float v) {
  reinterpret_cast<T*>(y)[at] = from_f32<T>(v);
}

__device__ __forceinline__ void store(void* y, int elem, int64_t at, float v) {
  if (elem == ELEM_F32) put<float>(y, at, v);
  else if (elem == ELEM_BF16) put<Bf16>(y, at, v);
  else put<_Float16>(y, at, v);
}

// One wave for each 16 x 16 block of results.
__global__ __launch_bounds__(64) void product_kernel(DesInt8Product p) {
  const int lane = threadIdx.x;
  const int nt = (p.N + 15) / 16, mt = (p.M + 15) / 16;
  int64_t id = blockIdx.x;
  const int n0 = (int)(id % nt) * 16;
  id /= nt;
  const int m0 = (int)(id % mt) * 16;
  const int64_t b = id / mt;
  const int row = lane & 15, group = lane >> 4;
  const int8_t* xr = p.x + b * p.xsb + (int64_t)min(m0 + row, p.M - 1) * p.xsr;
  const int8_t* wr = p.w + b * p.wsb + (int64_t)min(n0 + row, p.N - 1) * p.wsr;
  v4i acc = {0, 0, 0, 0};
  for (int k0 = 0; k0 < p.K; k0 += 64) {
    const int k = k0 + group * 16;
    acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(
        load16(xr + k, p.K - k), load16(wr + k, p.K - k), acc, 0, 0, 0);
  }
  const int n = n0 + row;
  if (n >= p.N) return;
  const float sw = p.sw[b * p.N + n];
  const float bias = p.bias ? p.bias[b * p.N + n] : 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int m = m0 + group * 4 + i;
    if (m < p.M)
      store(p.y, p.out, (b * p.M + m) * p.N + n,
            finish(acc[i], p.sx[b * p.M + m], sw, bias, p.act));
  }
}

}  // namespace

extern "C" void des_launch_int8_product(const DesInt8Product* p,
                                        hipStream_t stream) {
  const int64_t blocks =
      p->B * ((p->M + 15) / 16) * (int64_t)((p->N + 15) / 16);
  hipLaunchKernelGGL(product_kernel, dim3((uint32_t)blocks), dim3(64), 0,
                     stream, *p);
}
