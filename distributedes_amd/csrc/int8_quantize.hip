// quantize_rows: float rows -> 8-bit codes and one fp32 scale a row (int8.h has
// the definition).
//
// Memory bound: a row is read once and held in registers between its maximum
// and its codes, about 6 operations a value (see row_codes).
#include <algorithm>

#include "int8.h"

namespace {

using namespace des;

struct Rows {
  const void* x;
  int8_t* q;
  float* scale;
  int64_t xsl, xsr, qsl, qsr;
  uint32_t lead, rows;
  int32_t cols;
};

template <typename T>
__device__ __forceinline__ void row_at(const Rows& p, uint32_t r,
                                       const T** src, int8_t** dst) {
  uint32_t l = 0, i = r;
  if (p.lead > 1) {
    l = r / p.rows;
    i = r - l * p.rows;
  }
  *src = (const T*)p.x + l * p.xsl + i * p.xsr;
  *dst = p.q + l * p.qsl + i * p.qsr;
}

// the V values at k, 0 behind the row, in their own type: half the registers
// for 16-bit rows, so that twice the loads are under way
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load_piece(const T* src, int k,
                                                int cols) {
  if (k + V <= cols) return *reinterpret_cast<const Vec<T, V>*>(src + k);
  Vec<T, V> t = {};
#pragma unroll
  for (int j = 0; j < V; ++j)
    if (k + j < cols) t.v[j] = src[k + j];
  return t;
}

template <typename T, int V>
__device__ __forceinline__ uint32_t top_of(const Vec<T, V>& t) {
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < V; ++j) top = max(top, abs_bits(to_f32(t.v[j])));
  return top;
}

template <typename T, int V>
__device__ __forceinline__ void store_piece(int8_t* dst, int k, int cols,
                                            const Vec<T, V>& t, RowScale rs) {
  if (k >= cols) return;
  Vec<uint8_t, V> o;
#pragma unroll
  for (int h = 0; h < V; h += 4) {
    const float four[4] = {to_f32(t.v[h]), to_f32(t.v[h + 1]),
                           to_f32(t.v[h + 2]), to_f32(t.v[h + 3])};
    const uint32_t word = row_codes(four, rs);
    __builtin_memcpy(o.v + h, &word, 4);
  }
  if (k + V <= cols) {
    *reinterpret_cast<Vec<uint8_t, V>*>(dst + k) = o;
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (k + j < cols) dst[k + j] = (int8_t)o.v[j];
  }
}

// A row to 2^lbits lanes of a wave, R pieces of 16 bytes a lane.
template <typename T, int R>
__global__ __launch_bounds__(256) void wave_rows_kernel(Rows p, int lbits) {
  constexpr int V = 16 / sizeof(T);
  const int lane = threadIdx.x & 63, L = 1 << lbits;
  const uint32_t r =
      ((blockIdx.x * 4 + (threadIdx.x >> 6)) << (6 - lbits)) + (lane >> lbits);
  const bool in = r < p.lead * p.rows;
  const T* src;
  int8_t* dst;
  row_at<T>(p, in ? r : 0, &src, &dst);
  const int cols = in ? p.cols : 0, k0 = (lane & (L - 1)) * V;
  Vec<T, V> v[R];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < R; ++i) v[i] = load_piece<T, V>(src, k0 + i * L * V, cols);
#pragma unroll
  for (int i = 0; i < R; ++i) top = max(top, top_of(v[i]));
  for (int off = L >> 1; off > 0; off >>= 1)
    top = max(top, (uint32_t)__shfl_xor((int)top, off));
  const RowScale rs = row_scale(top);
#pragma unroll
  for (int i = 0; i < R; ++i)
    store_piece(dst, k0 + i * L * V, cols, v[i], rs);
  if (in && k0 == 0) p.scale[r] = rs.scale;
}

// A row to a block: R pieces a thread in registers, what is longer is read
// again for its codes.
template <typename T, int R>
__global__ __launch_bounds__(1024) void block_rows_kernel(Rows p) {
  constexpr int V = 16 / sizeof(T);
  __shared__ uint32_t tops[16];
  const int tid = threadIdx.x, waves = blockDim.x >> 6;
  const T* src;
  int8_t* dst;
  row_at<T>(p, blockIdx.x, &src, &dst);
  const int k0 = tid * V, step = blockDim.x * V;
  Vec<T, V> v[R];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < R; ++i) v[i] = load_piece<T, V>(src, k0 + i * step, p.cols);
#pragma unroll
  for (int i = 0; i < R; ++i) top = max(top, top_of(v[i]));
  for (int k = k0 + R * step; k < p.cols; k += step) {
    top = max(top, top_of(load_piece<T, V>(src, k, p.cols)));
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1)
    top = max(top, (uint32_t)__shfl_xor((int)top, off));
  if ((tid & 63) == 0) tops[tid >> 6] = top;
  __syncthreads();
  for (int w = 0; w < waves; ++w) top = max(top, tops[w]);
  const RowScale rs = row_scale(top);
#pragma unroll
  for (int i = 0; i < R; ++i)
    store_piece(dst, k0 + i * step, p.cols, v[i], rs);
  for (int k = k0 + R * step; k < p.cols; k += step) {
    store_piece(dst, k, p.cols, load_piece<T, V>(src, k, p.cols), rs);
  }
  if (tid == 0) p.scale[blockIdx.x] = rs.scale;
}

// A launch has at most 2^32 - 1 threads; a larger one is not begun.
bool fits(int64_t blocks, int threads) {
  return blocks * threads <= 0xFFFFFFFF;
}

template <typename T, int R>
bool launch_waves(const Rows& p, int lbits, hipStream_t stream) {
  const uint32_t rows = p.lead * p.rows, per = 4u << (6 - lbits);
  if (!fits((rows + per - 1) / per, 256)) return false;
  hipLaunchKernelGGL((wave_rows_kernel<T, R>), dim3((rows + per - 1) / per),
                     dim3(256), 0, stream, p, lbits);
  return true;
}

template <typename T, int R>
bool launch_blocks(const Rows& p, int64_t threads, hipStream_t stream) {
  const uint32_t rows = p.lead * p.rows;
  const int each = (int)std::min<int64_t>(1024, (threads + 63) / 64 * 64);
  if (!fits(rows, each)) return false;
  hipLaunchKernelGGL((block_rows_kernel<T, R>), dim3(rows), dim3(each), 0,
                     stream, p);
  return true;
}

// Pieces of 16 bytes and who takes them; measured:
//  - up to 256 a row: lanes of a wave, three or four pieces each, and as many rows
//    a wave as fit. 262144 x 256 fp32 by 64 lanes 73.8 us, 32 60.0, 16 62.4, 8
//    71.0; 10000 x 376 fp32 by 64 6.1, 32 6.0, 16 6.4.
//  - longer rows: a block, four pieces a thread. 8192 x 3136 bf16 by 128 threads
//    15.1 us, 256 15.4, 448 24.6, a wave 17.5.
//  - few rows: a block, a piece a thread, for latency. 16 x 3136 bf16 by 448
//    threads 4.2 us, 256 6.1.
template <typename T>
bool choose(const Rows& p, hipStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const int64_t pieces = ((int64_t)p.cols + V - 1) / V;
  const uint32_t rows = p.lead * p.rows;
  if (pieces > 64 && rows < 512) return launch_blocks<T, 1>(p, pieces, stream);
  if (pieces > 256) return launch_blocks<T, 4>(p, (pieces + 3) / 4, stream);
  int lbits = 0;
  while (lbits < 6 && (4 << lbits) < pieces) ++lbits;
  const int64_t turns = (pieces + (1 << lbits) - 1) >> lbits;
  if (turns <= 1) return launch_waves<T, 1>(p, lbits, stream);
  if (turns <= 2) return launch_waves<T, 2>(p, lbits, stream);
  return launch_waves<T, 4>(p, lbits, stream);
}

}  // namespace

extern "C" bool des_launch_quantize_rows(const void* x, int elem, int64_t xsl,
                                         int64_t xsr, int8_t* q, int64_t qsl,
                                         int64_t qsr, float* scale,
                                         int64_t lead, int64_t rows, int cols,
                                         hipStream_t stream) {
  const Rows p = {x,   q,   scale,          xsl,            xsr,
                  qsl, qsr, (uint32_t)lead, (uint32_t)rows, cols};
  return elem == ELEM_F32    ? choose<float>(p, stream)
         : elem == ELEM_BF16 ? choose<Bf16>(p, stream)
                             : choose<_Float16>(p, stream);
}
