// int8_matmul: y[m, n] = act(float(sum_k x[m, k] w[n, k]) * sx[m] * sw[n] + b[n])
// int8_linear: the same, with x quantised on the way.
//
// Sums of products of codes are held in 32-bit integers: exact up to
// K = 2^31 / 127^2 = 133144 (the bindings allow 131072), whatever the order, so
// any split of K gives the same bits.
//
// The matrix instruction is v_mfma_i32_16x16x64_i8: a lane gives 16 neighbouring
// codes of row (lane & 15) at k = 16 * (lane >> 4), and holds the results of
// column (lane & 15) for rows 4 * (lane >> 4) .. + 3.  Weights are the first
// operand, so that a lane's four results are four neighbouring channels of one
// token: one store.
#include <algorithm>

#include "int8.h"

namespace {

using namespace des;

typedef __attribute__((ext_vector_type(4))) int v4i;
typedef __attribute__((ext_vector_type(4))) float v4f;

template <typename T, int V>
struct __attribute__((packed, aligned(sizeof(T)))) Vec { T v[V]; };

// 16 codes from any address
__device__ __forceinline__ v4i load16(const int8_t* p) {
  v4i v;
  __builtin_memcpy(&v, p, 16);
  return v;
}

// the first `left` of 16 codes, 0 behind them; `whole`: all 16 may be read
__device__ __forceinline__ v4i load_tail(const int8_t* p, int left,
                                         bool whole) {
  union { v4i v; int8_t b[16]; } u;
  u.v = v4i{0, 0, 0, 0};
  if (left <= 0) return u.v;
  if (left >= 16 || whole) {
    u.v = load16(p);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = left - 4 * j;
      u.v[j] &= n >= 4 ? -1 : n <= 0 ? 0 : (1 << (8 * n)) - 1;
    }
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

// four neighbouring channels of one token, `have` of them within the row
template <typename T>
__device__ __forceinline__ void put4(void* y, int64_t at, v4f v, int have,
                                     bool vec) {
  T* p = reinterpret_cast<T*>(y) + at;
  if (vec) {
    Vec<T, 4> o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o.v[i] = from_f32<T>(v[i]);
    *reinterpret_cast<Vec<T, 4>*>(p) = o;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < have) p[i] = from_f32<T>(v[i]);
  }
}

// results of channels n .. n + 3 for token m of member b
__device__ __forceinline__ void finish4(const DesInt8Product& p, int64_t b,
                                        int m, int n, v4i sum, float sx) {
  if (m >= p.M || n >= p.N) return;
  const int have = p.N - n;
  v4f v;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t at = b * p.N + min(n + i, p.N - 1);
    v[i] = finish(sum[i], sx, p.sw[at], p.bias ? p.bias[at] : 0.f, p.act);
  }
  const int64_t at = (b * p.M + m) * p.N + n;
  const bool vec = have >= 4;
  if (p.out == ELEM_F32) put4<float>(p.y, at, v, have, vec);
  else if (p.out == ELEM_BF16) put4<Bf16>(p.y, at, v, have, vec);
  else put4<_Float16>(p.y, at, v, have, vec);
}

// Quantises `rows` rows of K floats into shared memory, a row every `step`
// bytes with zeros up to `kpad`; a thread's slice of every row is the same, so
// one barrier joins all rows' maxima.
template <typename T>
__device__ void quantize_block(const T* x, int64_t xsr, int rows, int K,
                               int kpad, int step, int8_t* codes,
                               float* scales, uint32_t* tops, int waves) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int stride = blockDim.x * 4;
  for (int r = 0; r < rows; ++r) {
    const T* src = x + r * xsr;
    uint32_t top = 0;
    for (int k = tid * 4; k < K; k += stride) {
      if (k + 4 <= K) {
        const auto v = *reinterpret_cast<const Vec<T, 4>*>(src + k);
#pragma unroll
        for (int j = 0; j < 4; ++j) top = max(top, abs_bits(to_f32(v.v[j])));
      } else {
        for (int j = k; j < K; ++j) top = max(top, abs_bits(to_f32(src[j])));
      }
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1)
      top = max(top, (uint32_t)__shfl_xor((int)top, off));
    if (lane == 0) tops[r * waves + wave] = top;
  }
  __syncthreads();
  for (int r = 0; r < rows; ++r) {
    const T* src = x + r * xsr;
    uint32_t top = 0;
    for (int w = 0; w < waves; ++w) top = max(top, tops[r * waves + w]);
    const RowScale rs = row_scale(top);
    if (tid == 0) scales[r] = rs.scale;
    for (int k = tid * 4; k < kpad; k += stride) {
      union { int word; int8_t b[4]; } o;
      if (k + 4 <= K) {
        const auto v = *reinterpret_cast<const Vec<T, 4>*>(src + k);
#pragma unroll
        for (int j = 0; j < 4; ++j) o.b[j] = (int8_t)row_code(to_f32(v.v[j]), rs);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          o.b[j] = k + j < K ? (int8_t)row_code(to_f32(src[k + j]), rs) : 0;
      }
      *reinterpret_cast<int*>(codes + r * step + k) = o.word;
    }
  }
  __syncthreads();
}

// Few rows: weights go straight from memory into the matrix instruction's
// operands, each read once.  A wave has 16 MT tokens and 16 NT channels, a
// block wn such waves side by side times wk shares of K, joined in shared
// memory.  X: the type of float rows (MT = 1), which the block quantises into
// shared memory, or int8_t: codes, read like the weights.
template <typename X, int MT, int NT>
__global__ __launch_bounds__(1024) void stream_kernel(DesInt8Product p, int wn,
                                                      int wk) {
  extern __shared__ __align__(16) int8_t shared[];
  constexpr bool FLOATS = sizeof(X) != 1;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int row = lane & 15, group = lane >> 4;
  const int nblocks = (p.N + 16 * NT * wn - 1) / (16 * NT * wn);
  const int mblocks = (p.M + 16 * MT - 1) / (16 * MT);
  int64_t id = blockIdx.x;
  const int mb = (int)(id % mblocks);
  id /= mblocks;
  const int nb = (int)(id % nblocks);
  const int64_t b = id / nblocks;
  const int m0 = mb * 16 * MT;
  const int n0 = (nb * wn + wave % wn) * 16 * NT;
  const int steps = (p.K + 63) / 64, full = p.K / 64;
  const int xstep = steps * 64 + 16;
  const int waves = wn * wk;
  float* scales = reinterpret_cast<float*>(shared);
  int8_t* codes = shared + 64;

  if constexpr (FLOATS) {
    const int rows = min(16, p.M - m0);
    uint32_t* tops = reinterpret_cast<uint32_t*>(codes + rows * xstep);
    quantize_block((const X*)p.xf + b * p.xsb + m0 * p.xsr, p.xsr, rows, p.K,
                   steps * 64, xstep, codes, scales, tops, waves);
  }
  const int8_t* wr[NT];
  const int8_t* xr[MT];
#pragma unroll
  for (int j = 0; j < NT; ++j)
    wr[j] = p.w + b * p.wsb + (int64_t)min(n0 + 16 * j + row, p.N - 1) * p.wsr +
            group * 16;
#pragma unroll
  for (int i = 0; i < MT; ++i)
    xr[i] = FLOATS ? codes + min(row, p.M - m0 - 1) * xstep + group * 16
                   : p.x + b * p.xsb +
                         (int64_t)min(m0 + 16 * i + row, p.M - 1) * p.xsr +
                         group * 16;

  v4i acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = v4i{0, 0, 0, 0};

  const int share = wave / wn;
  const int s0 = (int)((int64_t)steps * share / wk);
  const int s1 = (int)((int64_t)steps * (share + 1) / wk);
  const int s1f = min(s1, full);
#pragma unroll 4
  for (int s = s0; s < s1f; ++s) {
    v4i a[NT], x[MT];
#pragma unroll
    for (int j = 0; j < NT; ++j) a[j] = load16(wr[j] + s * 64);
#pragma unroll
    for (int i = 0; i < MT; ++i)
      x[i] = FLOATS ? *reinterpret_cast<const v4i*>(xr[i] + s * 64)
                    : load16(xr[i] + s * 64);
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[j], x[i],
                                                          acc[i][j], 0, 0, 0);
  }
  if (s1 > full && s0 < s1) {  // the step that K ends in
    const int left = p.K - full * 64 - group * 16;
    v4i a[NT], x[MT];
#pragma unroll
    for (int j = 0; j < NT; ++j)
      a[j] = load_tail(wr[j] + full * 64, left, p.wwhole);
#pragma unroll
    for (int i = 0; i < MT; ++i)
      x[i] = FLOATS ? *reinterpret_cast<const v4i*>(xr[i] + full * 64)
                    : load_tail(xr[i] + full * 64, left, p.xwhole);
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[j], x[i],
                                                          acc[i][j], 0, 0, 0);
  }

  if (wk > 1) {
    __syncthreads();  // the codes are read for the last time
    v4i* red = reinterpret_cast<v4i*>(codes);
    const int at = (wave % wn) * 64 + lane;
    if (share > 0) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
          red[((share - 1) * MT * NT + i * NT + j) * wn * 64 + at] = acc[i][j];
    }
    __syncthreads();
    if (share > 0) return;
    for (int k = 0; k < wk - 1; ++k)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
          acc[i][j] += red[(k * MT * NT + i * NT + j) * wn * 64 + at];
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int m = m0 + 16 * i + row;
    const float sx = m >= p.M   ? 0.f
                     : FLOATS ? scales[m - m0]
                              : p.sx[b * p.M + m];
#pragma unroll
    for (int j = 0; j < NT; ++j)
      finish4(p, b, m, n0 + 16 * j + group * 4, acc[i][j], sx);
  }
}

template <typename X, int MT, int NT>
void launch_stream(const DesInt8Product& p, int wn, int wk,
                   hipStream_t stream) {
  const int64_t nblocks = (p.N + 16 * NT * wn - 1) / (16 * NT * wn);
  const int64_t mblocks = (p.M + 16 * MT - 1) / (16 * MT);
  const int rows = std::min(16, (int)p.M), waves = wn * wk;
  size_t bytes = 64;
  if (sizeof(X) != 1)
    bytes += rows * ((p.K + 63) / 64 * 64 + 16) + rows * waves * 4;
  bytes = std::max<size_t>(bytes, 64 + (size_t)(wk - 1) * wn * MT * NT * 1024);
  hipLaunchKernelGGL((stream_kernel<X, MT, NT>),
                     dim3((uint32_t)(p.B * nblocks * mblocks)),
                     dim3(64 * waves), bytes, stream, p, wn, wk);
}

// Few rows.  Many members (or channels) fill the chip with waves of 64
// channels; else a wave has 16 and K is split until about 2048 waves run.
template <typename X>
void choose_stream(const DesInt8Product& p, hipStream_t stream) {
  const int64_t groups = (p.N + 15) / 16, steps = (p.K + 63) / 64;
  const int64_t mb = (p.M + 15) / 16;
  if (p.B * mb * groups >= 4 * 2048 && groups >= 4) {
    launch_stream<X, 1, 4>(p, (int)std::min<int64_t>(4, (groups + 3) / 4), 1,
                           stream);
    return;
  }
  int wn = 1, wk = 1;
  while (wk < 16 && p.B * mb * groups * wk < 2048 && steps >= 4 * wk) wk *= 2;
  while (wn * wk < 4 && wn < groups) wn *= 2;
  launch_stream<X, 1, 1>(p, wn, wk, stream);
}

}  // namespace

extern "C" void des_launch_int8_product(const DesInt8Product* p,
                                        hipStream_t stream) {
  if (p->x) {
    if (p->M > 64 && p->N > 32)
      launch_stream<int8_t, 4, 4>(*p, 1, 1, stream);
    else
      choose_stream<int8_t>(*p, stream);
  } else if (p->xelem == ELEM_F32) {
    choose_stream<float>(*p, stream);
  } else if (p->xelem == ELEM_BF16) {
    choose_stream<Bf16>(*p, stream);
  } else {
    choose_stream<_Float16>(*p, stream);
  }
}
