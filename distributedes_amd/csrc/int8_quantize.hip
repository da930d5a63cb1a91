// quantize_rows: float rows -> 8-bit codes and one fp32 scale a row (int8.h has
// the definition).  Memory bound: a row is read, its codes written.
#include "int8.h"

namespace {

using namespace des;

template <typename T>
__global__ __launch_bounds__(256) void quantize_rows_kernel(
    const T* __restrict__ x, int64_t xsl, int64_t xsr, int8_t* __restrict__ q,
    int64_t qsl, int64_t qsr, float* __restrict__ scale, int64_t lead,
    int64_t rows, int cols) {
  const int lane = threadIdx.x & 63;
  const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= lead * rows) return;
  const int64_t l = r / rows, i = r - l * rows;
  const T* src = x + l * xsl + i * xsr;
  int8_t* dst = q + l * qsl + i * qsr;
  uint32_t top = 0;
  for (int k = lane; k < cols; k += 64)
    top = max(top, abs_bits(to_f32(src[k])));
#pragma unroll
  for (int off = 32; off > 0; off >>= 1)
    top = max(top, (uint32_t)__shfl_xor((int)top, off));
  const RowScale rs = row_scale(top);
  for (int k = lane; k < cols; k += 64)
    dst[k] = (int8_t)row_code(to_f32(src[k]), rs);
  if (lane == 0) scale[r] = rs.scale;
}

template <typename T>
void launch(const void* x, int64_t xsl, int64_t xsr, int8_t* q, int64_t qsl,
            int64_t qsr, float* scale, int64_t lead, int64_t rows, int cols,
            hipStream_t stream) {
  const int64_t blocks = (lead * rows + 3) / 4;
  hipLaunchKernelGGL(quantize_rows_kernel<T>, dim3((uint32_t)blocks),
                     dim3(256), 0, stream, (const T*)x, xsl, xsr, q, qsl, qsr,
                     scale, lead, rows, cols);
}

}  // namespace

extern "C" void des_launch_quantize_rows(const void* x, int elem, int64_t xsl,
                                         int64_t xsr, int8_t* q, int64_t qsl,
                                         int64_t qsr, float* scale,
                                         int64_t lead, int64_t rows, int cols,
                                         hipStream_t stream) {
  if (elem == ELEM_F32)
    launch<float>(x, xsl, xsr, q, qsl, qsr, scale, lead, rows, cols, stream);
  else if (elem == ELEM_BF16)
    launch<Bf16>(x, xsl, xsr, q, qsl, qsr, scale, lead, rows, cols, stream);
  else
    launch<_Float16>(x, xsl, xsr, q, qsl, qsr, scale, lead, rows, cols,
                     stream);
}
