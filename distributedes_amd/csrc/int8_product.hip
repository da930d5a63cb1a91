// int8_matmul: y[m, n] = act(float(sum_k x[m, k] w[n, k]) * sx[m] * sw[n] + b[n])
// int8_linear: the same, with x quantised on the way.
//
// Sums of products of codes are held in 32-bit integers: exact up to
// K = 2^31 / 127^2 = 133144 (the bindings allow 131072), whatever the order, so
// any split of K gives the same bits.
//
// Up to 4 tokens the product is a stream of weights: gemv_kernel.  Otherwise the
// matrix instruction is v_mfma_i32_16x16x64_i8: a lane gives 16 neighbouring
// codes of row (lane & 15) at k = 16 * (lane >> 4), and holds the results of
// column (lane & 15) for rows 4 * (lane >> 4) .. + 3.  Weights are the first
// operand, so that a lane's four results are four neighbouring channels of one
// token: one store.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <type_traits>

#include "int8.h"

namespace {

using namespace des;

typedef __attribute__((ext_vector_type(4))) int v4i;
typedef __attribute__((ext_vector_type(4))) float v4f;
typedef v4i v4i_any __attribute__((aligned(1)));  // at any address

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

// sum * sx * sw + b.  Sums stay below 2^31, so sum * sx stays in fp32's range for
// sx below 2^96.  Under a larger one it may leave the range where the result does
// not: 2^32 goes from sx to sw, both exactly.
__device__ __forceinline__ bool large_scale(float sx) {
  return fabsf(sx) >= 0x1p96f;
}

__device__ __forceinline__ float lowered(float sx) { return sx * 0x1p-32f; }

// A finite sw stays finite: with a sum of 0 the result is b, with any other it is
// beyond the range all the same.
__device__ __forceinline__ float lifted(float sw) {
  const float v = sw * 0x1p32f;
  return fabsf(v) == INFINITY && fabsf(sw) < INFINITY ? copysignf(FLT_MAX, sw)
                                                      : v;
}

__device__ __forceinline__ float finish(int sum, float sx, float sw, float b,
                                        int act) {
  if (large_scale(sx)) {
    sx = lowered(sx);
    sw = lifted(sw);
  }
  float v = fmaf((float)sum * sx, sw, b);
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

__device__ __forceinline__ void put1(const DesInt8Product& p, int64_t at,
                                     float v) {
  if (p.out == ELEM_F32) reinterpret_cast<float*>(p.y)[at] = v;
  else if (p.out == ELEM_BF16) reinterpret_cast<Bf16*>(p.y)[at] = from_f32<Bf16>(v);
  else reinterpret_cast<_Float16*>(p.y)[at] = from_f32<_Float16>(v);
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

template <typename T>
__device__ __forceinline__ void load_floats(const T* src, int k, int K,
                                            float (&v)[4]) {
  if (k + 4 <= K) {
    const auto t = *reinterpret_cast<const Vec<T, 4>*>(src + k);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = to_f32(t.v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = k + j < K ? to_f32(src[k + j]) : 0.f;
  }
}

// Quantises `rows` rows of K floats into shared memory, a row every `step`
// bytes with zeros up to `kpad` (a multiple of 4).  A thread's slice of every
// row is the same, so one barrier joins all rows' maxima; the slice's first
// four values of the first row are kept in between.
template <typename T>
__device__ void quantize_block(const T* x, int64_t xsr, int rows, int K,
                               int kpad, int step, int8_t* codes,
                               float* scales, uint32_t* tops, int waves) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int stride = blockDim.x * 4;
  float kept[4];
  load_floats(x, tid * 4, K, kept);
  for (int r = 0; r < rows; ++r) {
    const T* src = x + r * xsr;
    uint32_t top = 0;
    for (int k = tid * 4; k < K; k += stride) {
      float v[4];
      if (r == 0 && k == tid * 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = kept[j];
      } else {
        load_floats(src, k, K, v);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) top = max(top, abs_bits(v[j]));
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
      float v[4];
      if (r == 0 && k == tid * 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = kept[j];
      } else {
        load_floats(src, k, K, v);
      }
      *reinterpret_cast<uint32_t*>(codes + r * step + k) = row_codes(v, rs);
    }
  }
  __syncthreads();
}

// The same for rows of at most 64 NP values: 2^lbits lanes of a wave take a row,
// up to NP pieces of 4 values each, which stay in registers, so that all rows
// are read at once.  (16 rows of 40 values one after the other took 10 times
// the product that they were for.)
template <typename T, int NP>
__device__ __forceinline__ void quantize_rows_at_once(
    const T* x, int64_t xsr, int rows, int K, int kpad, int step,
    int8_t* codes, float* scales, int lbits, int waves) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int L = 1 << lbits, per = 64 >> lbits;
  const int k0 = (lane & (L - 1)) * 4;
  for (int r0 = wave * per; r0 < rows; r0 += waves * per) {
    const int r = r0 + (lane >> lbits);
    const bool in = r < rows;
    const T* src = x + (in ? r : 0) * xsr;
    float v[NP][4];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < NP; ++i)
      load_floats(src, k0 + i * L * 4, in ? K : 0, v[i]);
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) top = max(top, abs_bits(v[i][j]));
    for (int off = L >> 1; off > 0; off >>= 1)
      top = max(top, (uint32_t)__shfl_xor((int)top, off));
    const RowScale rs = row_scale(top);
    if (!in) continue;
    if (k0 == 0) scales[r] = rs.scale;
#pragma unroll
    for (int i = 0; i < NP; ++i)
      if (k0 + i * L * 4 < kpad)
        *reinterpret_cast<uint32_t*>(codes + r * step + k0 + i * L * 4) =
            row_codes(v[i], rs);
  }
  __syncthreads();
}

// A block's float rows, by the one that fits.  `tops`: rows x waves words.
template <typename T>
__device__ __forceinline__ void quantize_tokens(const T* x, int64_t xsr,
                                                int rows, int K, int kpad,
                                                int step, int8_t* codes,
                                                float* scales, uint32_t* tops,
                                                int waves) {
  // kpad may reach 64 values behind K: lanes for all of it
  int lbits = 0;
  if (kpad <= 1024) {
    while ((16 << lbits) < kpad) ++lbits;
    quantize_rows_at_once<T, 4>(x, xsr, rows, K, kpad, step, codes, scales,
                                lbits, waves);
  } else if (kpad <= 2048) {
    quantize_rows_at_once<T, 8>(x, xsr, rows, K, kpad, step, codes, scales, 6,
                                waves);
  } else {
    quantize_block(x, xsr, rows, K, kpad, step, codes, scales, tops, waves);
  }
}

// Copies rows of K codes into shared memory, a row every `step` bytes with
// zeros up to `kpad` (a multiple of 16).
__device__ void stage_block(const int8_t* x, int64_t xsr, int rows, int K,
                            int kpad, int step, int8_t* codes, bool whole) {
  for (int r = 0; r < rows; ++r)
    for (int k = threadIdx.x * 16; k < kpad; k += blockDim.x * 16)
      *reinterpret_cast<v4i*>(codes + r * step + k) =
          load_tail(x + r * xsr + k, K - k, whole);
  __syncthreads();
}

// One token to MR: memory bound, every weight is read once for 2 MR operations.
// A row of weights goes to L neighbouring lanes (1 to 64, a power of 2), so a
// wave's load is 64 / L pieces of 16 L bytes; U such loads are under way, and
// the next U begin before their products.  Products are v_dot4_i32_i8 with the
// token's codes from shared memory; L lanes' sums are joined at the row's end.
//
// The matrix instruction would want 16 rows in pieces of 64 bytes: for a layer
// of 256 x 376 for each of 10000 members that reads 3.8 TB/s (254 us), this 6.1
// (159 us; a plain read of as much: 7.0), and 2048 layers of 512 x 3136 4.6 TB/s
// (709 us) against 6.4 (511 us).
template <typename X, int MR, int U, bool ONCE>
__global__ __launch_bounds__(256) void gemv_kernel(DesInt8Product p, int lbits,
                                                   int rows_a_wave) {
  extern __shared__ __align__(16) int8_t shared[];
  constexpr bool FLOATS = sizeof(X) != 1;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int waves = blockDim.x >> 6;
  const int nblocks = (p.N + waves * rows_a_wave - 1) / (waves * rows_a_wave);
  const int64_t b = blockIdx.x / nblocks;
  const int nb = (int)(blockIdx.x - b * nblocks);
  const int kpad = (p.K + 15) / 16 * 16, step = kpad + 16;
  float* scales = reinterpret_cast<float*>(shared);
  int8_t* codes = shared + 16;
  int* sums = reinterpret_cast<int*>(codes + p.M * step);
  const int L = 1 << lbits, per = 64 >> lbits;  // lanes a row, rows a load
  const int li = lane & (L - 1), sub = lane >> lbits;
  const int kend = p.wwhole ? kpad : p.K / 16 * 16;
  const int8_t* wb = p.w + b * p.wsb;
  const int first = (nb * waves + wave) * rows_a_wave;
  const int last = min(first + rows_a_wave, p.N);

  v4i next[U];  // the next turn's weights: loads run ahead by one
  const int8_t* wr[U];
  auto rows_at = [&](int n0) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      wr[u] = wb + (int64_t)min(n0 + u * per + sub, p.N - 1) * p.wsr;
  };
  auto fetch = [&](int k) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const v4i_any* at = reinterpret_cast<const v4i_any*>(wr[u] + k);
      next[u] = k >= kend ? v4i{0, 0, 0, 0}
                : ONCE    ? __builtin_nontemporal_load(at)
                          : *at;
    }
  };
  rows_at(first);
  if (first < last) fetch(li * 16);  // under way while the token is quantised
  const int ch = first + lane;       // a wave has at most 64 channels
  float sw = 0.f, bias = 0.f;
  if (ch < last) {
    sw = p.sw[b * p.N + ch];
    if (p.bias) bias = p.bias[b * p.N + ch];
  }

  if constexpr (FLOATS) {
    uint32_t* tops = reinterpret_cast<uint32_t*>(sums + waves * 64 * MR);
    const X* xf = (const X*)p.xf + b * p.xsb;
    if constexpr (MR == 1)  // one row: all waves, and fewer registers
      quantize_block(xf, p.xsr, 1, p.K, kpad, step, codes, scales, tops, waves);
    else
      quantize_tokens(xf, p.xsr, p.M, p.K, kpad, step, codes, scales, tops,
                      waves);
  } else {
    stage_block(p.x + b * p.xsb, p.xsr, p.M, p.K, kpad, step, codes, p.xwhole);
  }

  int* mine = sums + wave * 64 * MR;
  for (int n0 = first; n0 < last; n0 += U * per) {
    if (kend == 0) rows_at(n0);  // no whole piece: the loop below has no turn
    int acc[U][MR];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int m = 0; m < MR; ++m) acc[u][m] = 0;
    auto add = [&](int k, const v4i (&w)[U]) {
#pragma unroll
      for (int m = 0; m < MR; ++m) {
        if (m > 0 && m >= p.M) break;
        const v4i x = *reinterpret_cast<const v4i*>(codes + m * step + k);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            acc[u][m] = __builtin_amdgcn_sdot4(w[u][j], x[j], acc[u][m], false);
      }
    };
    v4i tail[U];
    const bool odd = kend < p.K && li == 0;
    if (odd) {  // a row's last codes, none behind them read
#pragma unroll
      for (int u = 0; u < U; ++u)
        tail[u] = load_tail(wr[u] + kend, p.K - kend, false);
    }
    for (int k = li * 16; k - li * 16 < kend; k += L * 16) {
      v4i w[U];
#pragma unroll
      for (int u = 0; u < U; ++u) w[u] = next[u];
      if (k - li * 16 + L * 16 < kend) {
        fetch(k + L * 16);
      } else if (n0 + U * per < last) {
        rows_at(n0 + U * per);
        fetch(li * 16);
      }
      add(min(k, kpad), w);  // w = 0 behind the row
    }
    if (odd) add(kend, tail);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int m = 0; m < MR; ++m) {
        for (int off = L >> 1; off > 0; off >>= 1)
          acc[u][m] += __shfl_xor(acc[u][m], off);
        const int at = n0 - first + u * per + sub;
        if (li == 0 && at < 64) mine[m * 64 + at] = acc[u][m];
      }
  }
  __syncthreads();
  // one lane a channel: the factors were fetched at the start, and the
  // activation runs on whole waves
  if (ch < last) {
#pragma unroll
    for (int m = 0; m < MR; ++m) {
      if (m >= p.M) break;
      const float sx = FLOATS ? scales[m] : p.sx[b * p.M + m];
      put1(p, (b * p.M + m) * p.N + ch,
           finish(mine[m * 64 + lane], sx, sw, bias, p.act));
    }
  }
}

// waves of a block for parts of a member's channels: up to 4, and as even as the
// blocks that this takes allow (5 parts: 3 + 2, not 4 + 1)
int waves_for(int64_t parts) {
  const int64_t blocks = (parts + 3) / 4;
  return (int)((parts + blocks - 1) / blocks);
}

// A launch has at most 2^31 - 1 blocks and 2^32 - 1 threads; a larger one is not
// begun.
bool fits(int64_t blocks, int threads) {
  return blocks <= 0x7FFFFFFF && blocks * threads <= 0xFFFFFFFF;
}

template <typename X, int MR, int U, bool ONCE>
bool launch_gemv(const DesInt8Product& p, int lbits, int rows_a_wave,
                 hipStream_t stream) {
  const int64_t parts = (p.N + (int64_t)rows_a_wave - 1) / rows_a_wave;
  const int waves = waves_for(parts);
  const int64_t nblocks = (parts + waves - 1) / waves;
  const size_t bytes = 16 + p.M * ((p.K + 15) / 16 * 16 + 16) +
                       waves * 64 * MR * 4 + p.M * waves * 4;
  if (!fits(p.B * nblocks, 64 * waves)) return false;
  hipLaunchKernelGGL((gemv_kernel<X, MR, U, ONCE>),
                     dim3((uint32_t)(p.B * nblocks)), dim3(64 * waves), bytes,
                     stream, p, lbits, rows_a_wave);
  return true;
}

// How many lanes take a row, how many rows a wave takes, and whether its loads
// pass the caches by.  Measured over 0.5 to 1 GB of weights, M = 1:
//  - up to 32 MB: latency counts.  A row to as many lanes as it fills, one load
//    a row and turn, and as many waves as that gives, up to 8192.
//  - weights that no cache would keep (256 MB), rows that begin on lines of
//    128 bytes: past the caches, a line a turn and row.  K = 376 (rows of 384),
//    960 MB: 4 lanes 293 us, 8 163, 16 167, 32 192; 503 MB by 8 lanes 82, and
//    through the caches 90.
//  - such weights in long rows that do not: 64 lanes, so that few lines are
//    fetched in halves.  K = 3136, 3.3 GB: 509 us, 16 lanes 576, and through the
//    caches 526.
//  - all others: through the caches, which join halves of lines, and few lanes,
//    which have fewer sums to join.  503 MB, K = 300 (304): 2 lanes 223 us, 4 129,
//    8 104, 16 99; past the caches 116.  K = 48: 1 lane 139, 2 124, 4 138.
template <typename X, int MR>
bool choose_gemv_rows(const DesInt8Product& p, hipStream_t stream) {
  const int64_t bytes = p.B * (int64_t)p.N * p.K;
  auto lanes = [&](int codes, int least, int most) {  // as bits
    int bits = least;
    while (bits < most && (int64_t)codes << bits < p.K) ++bits;
    return bits;
  };
  if (bytes <= 32 << 20) {
    const int bits = lanes(16, 0, 6);
    int rows = 64 >> bits;
    while (rows < 64 && p.B * ((p.N + rows - 1) / rows) > 8192) rows *= 2;
    return launch_gemv<X, MR, 1, false>(p, bits, rows, stream);
  }
  const int rows = p.K >= 1024 ? 16 : 64;
  const bool lines =
      ((uintptr_t)p.w | (uintptr_t)p.wsr | (uintptr_t)p.wsb) % 128 == 0;
  const bool once = bytes >= 256 << 20;
  if (once && lines && p.K > 96)
    return launch_gemv<X, MR, 2, true>(p, 3, rows, stream);
  if (once && p.K >= 2048)
    return launch_gemv<X, MR, 4, true>(p, 6, rows, stream);
  return launch_gemv<X, MR, 2, false>(p, p.K <= 16 ? 0 : lanes(32, 1, 4), rows,
                                      stream);
}

template <typename X>
bool choose_gemv(const DesInt8Product& p, hipStream_t stream) {
  return p.M == 1 ? choose_gemv_rows<X, 1>(p, stream)
                  : choose_gemv_rows<X, 4>(p, stream);
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
    const X* xf = (const X*)p.xf + b * p.xsb + m0 * p.xsr;
    uint32_t* tops = reinterpret_cast<uint32_t*>(codes + rows * xstep);
    quantize_tokens(xf, p.xsr, rows, p.K, steps * 64, xstep, codes, scales,
                    tops, waves);
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
  const int s1 = n0 < p.N ? (int)((int64_t)steps * (share + 1) / wk) : s0;
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
bool launch_stream(const DesInt8Product& p, int wn, int wk,
                   hipStream_t stream) {
  const int64_t nblocks = (p.N + 16 * NT * wn - 1) / (16 * NT * wn);
  const int64_t mblocks = (p.M + 16 * MT - 1) / (16 * MT);
  const int rows = std::min(16, (int)p.M), waves = wn * wk;
  size_t bytes = 64;
  if (sizeof(X) != 1)
    bytes += rows * ((p.K + 63) / 64 * 64 + 16) + rows * waves * 4;
  bytes = std::max<size_t>(bytes, 64 + (size_t)(wk - 1) * wn * MT * NT * 1024);
  if (!fits(p.B * nblocks * mblocks, 64 * waves)) return false;
  hipLaunchKernelGGL((stream_kernel<X, MT, NT>),
                     dim3((uint32_t)(p.B * nblocks * mblocks)),
                     dim3(64 * waves), bytes, stream, p, wn, wk);
  return true;
}

// Many members fill the chip with waves of 64 channels (or, for 17 to 32
// tokens, 32 channels); else a wave has 16 channels, and 8 to 16 of them share
// K.  For one policy of 512 x 3136: 16 to 128 tokens 5.2 us, in groups of 16
// tokens; 256 tokens in groups of 32 6.8; 512 tokens in groups of 32 x 32 8.7.
template <typename X>
bool choose_stream(const DesInt8Product& p, hipStream_t stream) {
  const int64_t groups = (p.N + 15) / 16, steps = (p.K + 63) / 64;
  const int64_t blocks = p.B * ((p.M + 15) / 16) * groups;
  if (p.M <= 16 && blocks >= 4 * 2048 && groups >= 4) {
    return launch_stream<X, 1, 4>(p, waves_for((groups + 3) / 4), 1, stream);
  }
  if constexpr (sizeof(X) == 1) {
    if (p.M > 16 && p.B > 1 && blocks >= 4096) {
      return launch_stream<X, 2, 2>(p, waves_for((groups + 1) / 2), 1, stream);
    }
    if (blocks > 1024) {
      return launch_stream<X, 2, 2>(p, 1, steps >= 4 ? 4 : 1, stream);
    }
    if (blocks > 256 && p.M > 16) {
      return launch_stream<X, 2, 1>(p, 1, steps >= 8 ? 8 : steps >= 4 ? 4 : 1, stream);
    }
  }
  int wn = 1, wk = 1;
  while (wk < 8 && blocks * wk < 2048 && steps >= 2 * wk) wk *= 2;
  if (wk == 8 && blocks <= 64 && steps >= 32) wk = 16;
  while (wn * wk < 4 && wn < groups) wn *= 2;
  return launch_stream<X, 1, 1>(p, wn, wk, stream);
}

typedef __attribute__((ext_vector_type(16))) int v16i;

// memory -> shared memory without registers in between: lane l's 16 bytes go
// to `to` + 16 l
__device__ __forceinline__ void load_shared(const int8_t* from, int8_t* to) {
  __builtin_amdgcn_global_load_lds(
      (const __attribute__((address_space(1))) void*)from,
      (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}

// Until at most N of this wave's loads are under way and its reads of shared
// memory have ended, then until all waves are here.  One statement, which no
// access to memory is moved across.
template <int N>
__device__ __forceinline__ void wait_stage() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N)
               : "memory");
}

// Between writes and reads of shared memory by lanes of one wave, which the
// hardware takes in their order: the compiler has to keep it too.
__device__ __forceinline__ void wave_order() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_wave_barrier();
}

// a wave's shared memory for 32 tokens x 32 NT results of 4 bytes
constexpr int tile_room(int nt) { return 32 * (nt * 128 + 16); }

// shared memory of a tile's stages, and of its end
constexpr int tiled_room(int wn, int wm, int nt, int mt, int s) {
  return std::max(s * 32 * (wn * nt + wm * mt) * 128, wn * wm * tile_room(nt));
}

// Results of a wave's NT x MT blocks of sums.  V = 8: the results have 16 bits
// and are finished where the sums are; V = 4: floats go through shared memory,
// the activation and the type come afterwards (32 bits, or tanh, whose code is
// long and stands here once).
template <int NT, int MT, int V>
__device__ __forceinline__ void tile_end(const DesInt8Product& p, int64_t b,
                                         const v16i (&acc)[NT][MT],
                                         const float (&sx)[MT],
                                         const float* sw, const float* bias,
                                         const float* lifts, int8_t* mine,
                                         int lane, int n0, int m0) {
  constexpr int SIZE = V == 8 ? 2 : 4;            // of a value in shared memory
  constexpr int ROW = NT * 32 * SIZE + 16;        // bytes
  constexpr int LANES = NT * 32 / V, TOKENS = 64 / LANES;
  const int half = lane >> 5, row = lane & 31;
  const int n = n0 + lane % LANES * V, have = p.N - n;
  const bool relu = p.act == 1, bf16 = p.out == ELEM_BF16;
#pragma unroll 1
  for (int i = 0; i < MT; ++i) {
#pragma unroll
    for (int ii = 0; ii < MT; ++ii) {
      if (i != ii) continue;
      const bool large = large_scale(sx[ii]);
      float st = large ? lowered(sx[ii]) : sx[ii];
      asm volatile("" : "+v"(st));  // products of all i at once would spill
      const float* sc = large ? lifts : sw;
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int c = j * 32 + 8 * g + 4 * half;
          const v4f s4 = *reinterpret_cast<const v4f*>(sc + c);
          const v4f b4 = *reinterpret_cast<const v4f*>(bias + c);
          v4f v;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            v[e] = fmaf((float)acc[j][ii][4 * g + e] * st, s4[e], b4[e]);
          int8_t* to = mine + row * ROW + c * SIZE;
          if constexpr (V == 8) {
            if (relu)
#pragma unroll
              for (int e = 0; e < 4; ++e) v[e] = v[e] < 0.f ? 0.f : v[e];
            Vec<uint16_t, 4> o;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              o.v[e] = bf16 ? from_f32<Bf16>(v[e]).bits
                            : __builtin_bit_cast(uint16_t, (_Float16)v[e]);
            __builtin_memcpy(__builtin_assume_aligned(to, 8), &o, 8);
          } else {
            *reinterpret_cast<v4f*>(to) = v;
          }
        }
    }
    wave_order();
    const int8_t* from = mine + lane / LANES * ROW + lane % LANES * 16;
    int m = m0 + i * 32 + lane / LANES;
    int64_t at = (b * p.M + m) * p.N + n;
#pragma unroll 1
    for (int t = 0; t < 32; t += TOKENS) {
      const v4i got = *reinterpret_cast<const v4i*>(from + t * ROW);
      if (m < p.M && have > 0) {
        if constexpr (V == 8) {
          uint16_t* y = reinterpret_cast<uint16_t*>(p.y) + at;
          if (have >= 8) {
            __builtin_memcpy(y, &got, 16);
          } else {
            for (int e = 0; e < have; ++e) {
              const int w = e < 2 ? got[0] : e < 4 ? got[1] : e < 6 ? got[2] : got[3];
              y[e] = (uint16_t)(e & 1 ? (uint32_t)w >> 16 : w);
            }
          }
        } else {
          v4f v = __builtin_bit_cast(v4f, got);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (relu) v[e] = v[e] < 0.f ? 0.f : v[e];
            if (p.act == 2) v[e] = tanhf(v[e]);
          }
          if (have >= 4 && p.out == ELEM_F32) {
            __builtin_memcpy(reinterpret_cast<float*>(p.y) + at, &v, 16);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (e < have) put1(p, at + e, v[e]);
          }
        }
      }
      m += TOKENS;
      at += (int64_t)TOKENS * p.N;
    }
    wave_order();
  }
}

// Many rows: a block has WN x WM waves, each with NT x MT blocks of 32 x 32
// results (channels x tokens), and takes K in stages of 128 codes through
// shared memory, S stages in a ring: while one is multiplied, S - 1 are on
// their way.
//
// A stage's rows lie 128 bytes apart; the 16-byte piece c of row r is kept at
// place c ^ (r / 2 & 7), so that the 16 lanes that read together (16 rows, the
// same piece) meet all 64 banks once.  Loads write lanes' pieces next to each
// other, so the places are exchanged where the pieces are read from memory.
//
// v_mfma_i32_32x32x32_i8: a lane gives 16 codes of row (lane & 31) at
// k = 16 * (lane >> 5), and holds the results of token (lane & 31) for channels
// 8 * (i / 4) + 4 * (lane >> 5) + i % 4, i < 16.
//
// What bounds it: with 256 x 256 results a block, the reads of shared memory (192
// KB a stage at 64 bytes a clock: 3000 clocks, of which the matrix units work
// 2048) and the clock, which falls from 2.4 to 2.0 GHz: 2.1 POPS.  With fewer
// results a block, the loads of both operands (24 bytes a clock and unit) and the
// barrier of a stage; there, three stages and 8 waves hide more of them (128 x 128
// results: 4 waves 25.0 us with two stages, 20.0 with three; 8 waves 22.8 and 17.7;
// a fourth stage 18.0).  Tried without gain: 128 x 128 results a wave, K shared by
// two groups of waves in a block, stages of 64, leaving a stage before its last
// step, priorities around the products.
template <int WN, int WM, int NT, int MT, int S>
__global__ __launch_bounds__(64 * WN * WM) void tiled_kernel(
    DesInt8Product p, uint32_t nblocks, uint32_t mblocks, bool together) {
  constexpr int THREADS = 64 * WN * WM;
  constexpr int BN = 32 * WN * NT, BM = 32 * WM * MT, BK = 128;
  constexpr int PIECES = (BN + BM) * (BK / 16) / THREADS;  // a thread's
  constexpr int STAGE = (BN + BM) * BK;
  constexpr int STEPS = BK / 32;
  extern __shared__ __align__(16) int8_t shared[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = wave % WN, wm = wave / WN;
  uint32_t id = blockIdx.x;
  if (together) {  // each die takes a piece of the list (see tiles_together)
    const uint32_t each = gridDim.x / 8;
    if (id < 8 * each) id = (id & 7) * each + (id >> 3);
  }
  const int nb = id % nblocks;
  id /= nblocks;
  const int mb = id % mblocks;
  const int64_t b = id / mblocks;
  const int n0 = nb * BN, m0 = mb * BM;
  auto place = [](int r) { return r >> 1 & 7; };

  // a thread's pieces of a stage: rows of weights, then rows of tokens
  const int8_t* src[PIECES];
  int col[PIECES];
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const int at = i * THREADS + tid, r = at >> 3;
    col[i] = ((at & 7) ^ place(r)) * 16;
    src[i] = r < BN ? p.w + b * p.wsb + (int64_t)min(n0 + r, p.N - 1) * p.wsr
                    : p.x + b * p.xsb +
                          (int64_t)min(m0 + r - BN, p.M - 1) * p.xsr;
  }
  // pieces behind a row's end are read at its begin: their products are masked
  auto fetch = [&](int k0, int stage) {
    int8_t* to = shared + stage * STAGE + wave * 1024;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int k = k0 + col[i];
      load_shared(src[i] + (k < p.K ? k : 0), to + i * THREADS * 16);
    }
  };

  const int half = lane >> 5, row = lane & 31;
  // the factors: tokens' in registers, channels' in shared memory.  Loads end
  // in their order, so waiting for a stage waits for them too.
  constexpr int EACH = (BN + THREADS - 1) / THREADS;
  float sx[MT], sw[EACH], bias[EACH];
#pragma unroll
  for (int i = 0; i < MT; ++i)
    sx[i] = p.sx[b * p.M + min(m0 + (wm * MT + i) * 32 + row, p.M - 1)];
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int64_t at = b * p.N + min(n0 + i * THREADS + tid, p.N - 1);
    sw[i] = p.sw[at];
    bias[i] = p.bias ? p.bias[at] : 0.f;
  }
#pragma unroll
  for (int s = 0; s < S - 1; ++s) fetch(s * BK, s);
  float* factors = reinterpret_cast<float*>(shared + tiled_room(WN, WM, NT, MT, S));
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int c = i * THREADS + tid;
    if (c < BN) {
      factors[c] = sw[i];
      factors[BN + c] = bias[i];
      factors[2 * BN + c] = lifted(sw[i]);
    }
  }

  v16i acc[NT][MT];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[j][i][e] = 0;

  const int wrow = wn * NT * 32 + row, xrow = BN + wm * MT * 32 + row;
  // the operands of step s of a stage (32 codes of K)
  auto read = [&](const int8_t* stage, int s, v4i (&a)[NT], v4i (&x)[MT]) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int r = wrow + 32 * j;
      a[j] = *reinterpret_cast<const v4i*>(
          stage + r * BK + (((2 * s + half) ^ place(r)) << 4));
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int r = xrow + 32 * i;
      x[i] = *reinterpret_cast<const v4i*>(
          stage + r * BK + (((2 * s + half) ^ place(r)) << 4));
    }
  };
  auto multiply = [&](const v4i (&a)[NT], const v4i (&x)[MT]) {
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < MT; ++i)
        acc[j][i] = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[j], x[i], acc[j][i],
                                                          0, 0, 0);
  };

  // A turn waits for its stage's own loads, then at the barrier for all waves':
  // by then they have also read the stage before it, whose place the next loads
  // take.  Loads behind the last stage repeat row begins, to keep the count.
  // The first two steps' operands are asked for before the next stage is: 8192 x
  // 4096 x 4096 148 -> 130 us.
  int turn = 0, k0 = 0;
  for (; k0 + BK <= p.K; k0 += BK) {
    wait_stage<PIECES * (S - 2)>();
    const int8_t* stage = shared + turn * STAGE;
    v4i a[STEPS][NT], x[STEPS][MT];
#pragma unroll
    for (int s = 0; s < 2; ++s) read(stage, s, a[s], x[s]);
    fetch(k0 + (S - 1) * BK, turn == 0 ? S - 1 : turn - 1);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      if (s >= 2) read(stage, s, a[s], x[s]);
      multiply(a[s], x[s]);
    }
    turn = turn == S - 1 ? 0 : turn + 1;
  }
  if (k0 < p.K) {  // the stage that K ends in
    wait_stage<PIECES * (S - 2)>();
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      v4i a[NT], x[MT];
      read(shared + turn * STAGE, s, a, x);
      const int left = p.K - k0 - (2 * s + half) * 16;
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // tokens are 0 behind K
          const int c = left - 4 * j;
          x[i][j] &= c >= 4 ? -1 : c <= 0 ? 0 : (1 << (8 * c)) - 1;
        }
      multiply(a, x);
    }
  }
  wait_stage<0>();  // the loads behind K as well: their room is used again

  // 32 tokens x 32 NT channels at a time through the wave's own part of shared
  // memory, to store 16 bytes of a token's row a lane
  const int nw = wn * NT * 32, mw = m0 + wm * MT * 32;
  int8_t* mine = shared + wave * tile_room(NT);
  if (p.out != ELEM_F32 && p.act != 2)
    tile_end<NT, MT, 8>(p, b, acc, sx, factors + nw, factors + BN + nw,
                        factors + 2 * BN + nw, mine, lane, n0 + nw, mw);
  else
    tile_end<NT, MT, 4>(p, b, acc, sx, factors + nw, factors + BN + nw,
                        factors + 2 * BN + nw, mine, lane, n0 + nw, mw);
}

// Whether neighbouring tiles are computed on one die (blocks in turn go to 8), by
// the rows of weights and tokens that the `at` tiles read which a die computes at
// once: few of them stay in its cache.  8192 x 512 x 3136 in tiles of 128 x 64:
// 25.5 us together, 27.6 as they come; 8192 x 4096 x 4096 in such tiles 290 and
// 179.
bool tiles_together(int64_t nblocks, int64_t bn, int64_t bm, int64_t at) {
  int64_t shared = 8;  // columns of tiles that fall to one die as they come
  while (nblocks % shared) shared /= 2;
  const int64_t apart =
      std::min(nblocks / shared, at) * bn +
      std::min(at, (8 * at + nblocks - 1) / nblocks) * bm;
  const int64_t together =
      std::min(nblocks, at) * bn + (at + nblocks - 1) / nblocks * bm;
  return together < apart;
}

template <int WN, int WM, int NT, int MT, int S>
bool launch_tiled(const DesInt8Product& p, int at, hipStream_t stream) {
  constexpr int BN = 32 * WN * NT, BM = 32 * WM * MT;
  constexpr int bytes = tiled_room(WN, WM, NT, MT, S) + BN * 12;
  const uint32_t nblocks = (p.N + (int64_t)BN - 1) / BN;
  const uint32_t mblocks = (p.M + (int64_t)BM - 1) / BM;
  const int64_t blocks = p.B * (int64_t)nblocks * mblocks;
  if (!fits(blocks, 64 * WN * WM)) return false;
  auto kernel = tiled_kernel<WN, WM, NT, MT, S>;
  if (bytes > 64 * 1024)
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                              hipFuncAttributeMaxDynamicSharedMemorySize,
                              bytes);
  hipLaunchKernelGGL(kernel, dim3((uint32_t)blocks), dim3(64 * WN * WM), bytes,
                     stream, p, nblocks, mblocks,
                     tiles_together(nblocks, BN, BM, at));
  return true;
}

// The tiles that cost least, by their turns: a unit of the chip takes its tiles
// one after the other (or two at once, half as fast), each with a time for a
// stage of K and one for its end, in us.  Small tiles load more a result, large
// ones leave units without work and nothing runs beside their ends.  Measured, us:
//                        256 x 256  256 x 128  128 x 128  128 x 64  64 x 64
//   8192 x 4096 x 4096       136                   158       185       221
//   8192 x 2048 x 2048        31         37         34        45        52
//   20000 x 1024 x 1000       37         35         29        36        39
//   8192 x 1024 x 3136        52         29         34        43        53
//   8192 x 1024 x 1024        19         14         13        16        18
//   8192 x  512 x 3136        47                    18        21        22
//   4096 x  512 x 3136        39         25         17        13        13
//   1024 x  512 x 3136                              16        12         9
// Three stages of 128 x 128 fill a unit's shared memory with one block: 18 us
// instead of 23 for 8192 x 512 x 3136, a tile a unit; two blocks of two stages 34
// instead of 37 for 8192 x 1024 x 3136, two a unit.
bool choose_tiled(const DesInt8Product& p, hipStream_t stream) {
  const int stages = (p.K + 127) / 128;
  auto turns = [&](int64_t n, int64_t m) {
    const int64_t tiles = p.B * ((p.N + n - 1) / n) * ((p.M + m - 1) / m);
    return (tiles + 255) / 256;
  };
  auto cost = [&](int64_t n, int64_t m, double stage, double end) {
    return (double)turns(n, m) * (stage * stages + end);
  };
  const double by[5] = {cost(256, 256, 1.95, 5.0), cost(256, 128, 1.15, 3.5),
                        cost(128, 128, 0.70, 0.5), cost(128, 64, 0.43, 0.3),
                        cost(64, 64, 0.25, 0.2)};
  switch (std::min_element(by, by + 5) - by) {
    case 0: return launch_tiled<2, 4, 4, 2, 2>(p, 32, stream);
    case 1: return launch_tiled<2, 4, 4, 1, 3>(p, 32, stream);
    case 2:
      if (turns(128, 128) == 1) return launch_tiled<2, 4, 2, 1, 3>(p, 32, stream);
      return launch_tiled<2, 4, 2, 1, 2>(p, 64, stream);
    case 3: return launch_tiled<2, 2, 2, 1, 3>(p, 64, stream);
    default: return launch_tiled<2, 2, 1, 1, 3>(p, 64, stream);
  }
}

// codes -> rows every `step` bytes, with zeros behind them
__global__ __launch_bounds__(256) void pack_rows_kernel(
    const int8_t* __restrict__ from, int64_t sb, int64_t sr,
    int8_t* __restrict__ to, int64_t rows, int K, int step, int64_t pieces) {
  const int per = step / 16;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < pieces;
       i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / per, b = r / rows;
    const int k = (int)(i - r * per) * 16;
    reinterpret_cast<v4i*>(to)[i] =
        load_tail(from + b * sb + (r - b * rows) * sr + k, K - k, false);
  }
}

}  // namespace

extern "C" void des_launch_pack_rows(const int8_t* from, int64_t sb, int64_t sr,
                                     int8_t* to, int64_t B, int64_t rows,
                                     int K, hipStream_t stream) {
  const int step = (K + 15) / 16 * 16;
  const int64_t pieces = B * rows * (step / 16);
  if (pieces == 0) return;
  hipLaunchKernelGGL(pack_rows_kernel,
                     dim3((uint32_t)std::min<int64_t>((pieces + 255) / 256,
                                                      8192)),
                     dim3(256), 0, stream, from, sb, sr, to, rows, K, step,
                     pieces);
}

extern "C" bool des_launch_int8_product(const DesInt8Product* p,
                                        hipStream_t stream) {
  const DesInt8Product& q = *p;
  const DesInt8Plan plan = des_int8_plan(q.B, q.M, q.N, q.K);
  if (plan == DES_INT8_TILED) return choose_tiled(q, stream);
  const bool gemv = plan == DES_INT8_GEMV;
  if (q.sx)  // not x, which is null where K = 0
    return gemv ? choose_gemv<int8_t>(q, stream)
                : choose_stream<int8_t>(q, stream);
  if (q.xelem == ELEM_F32)
    return gemv ? choose_gemv<float>(q, stream)
                : choose_stream<float>(q, stream);
  if (q.xelem == ELEM_BF16)
    return gemv ? choose_gemv<Bf16>(q, stream)
                : choose_stream<Bf16>(q, stream);
  return gemv ? choose_gemv<_Float16>(q, stream)
              : choose_stream<_Float16>(q, stream);
}
