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

#include "int8.h"

namespace {

using namespace des;

typedef __attribute__((ext_vector_type(4))) int v4i;
typedef __attribute__((ext_vector_type(4))) float v4f;
typedef v4i v4i_any __attribute__((aligned(1)));  // at any address

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
      union { int word; int8_t b[4]; } o;
#pragma unroll
      for (int j = 0; j < 4; ++j) o.b[j] = (int8_t)row_code(v[j], rs);
      *reinterpret_cast<int*>(codes + r * step + k) = o.word;
    }
  }
  __syncthreads();
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
// of 256 x 376 for each of 10000 members that reads 4.2 TB/s, this 6.1 (a plain
// read of as much: 7.0), and rows of 3136 codes 5.1 against 6.3.
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
    quantize_block((const X*)p.xf + b * p.xsb, p.xsr, p.M, p.K, kpad, step,
                   codes, scales, tops, waves);
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

template <typename X, int MR, int U, bool ONCE>
void launch_gemv(const DesInt8Product& p, int lbits, int rows_a_wave,
                 hipStream_t stream) {
  const int64_t parts = (p.N + (int64_t)rows_a_wave - 1) / rows_a_wave;
  const int waves = (int)std::min<int64_t>(4, parts);
  const int64_t nblocks = (parts + waves - 1) / waves;
  const size_t bytes = 16 + p.M * ((p.K + 15) / 16 * 16 + 16) +
                       waves * 64 * MR * 4 + p.M * waves * 4;
  hipLaunchKernelGGL((gemv_kernel<X, MR, U, ONCE>),
                     dim3((uint32_t)(p.B * nblocks)), dim3(64 * waves), bytes,
                     stream, p, lbits, rows_a_wave);
}

// How many lanes take a row, how many rows a wave takes, and whether its loads
// pass the caches by.  Measured over 0.5 to 1 GB of weights, M = 1:
//  - up to 32 MB: latency counts.  A row to as many lanes as it fills, one load
//    a row and turn, and as many waves as that gives.
//  - weights that no cache would keep (256 MB), rows that begin on lines of
//    128 bytes: past the caches, a line a turn and row.  K = 376 (rows of 384):
//    4 lanes 292 us, 8 163, 16 167, 32 192; through the caches 180.
//  - such weights in long rows that do not: 64 lanes, so that few lines are
//    fetched in halves.  K = 3136: 509 us, 16 lanes 576.
//  - all others: through the caches, which join halves of lines, and few lanes,
//    which have fewer sums to join.  K = 200 (208): 2 lanes 255 us, 4 130, 8 104,
//    16 99; past the caches 150.  K = 48: 1 lane 139, 2 124, 4 138.
template <typename X, int MR>
void choose_gemv_rows(const DesInt8Product& p, hipStream_t stream) {
  const int64_t bytes = p.B * (int64_t)p.N * p.K;
  auto lanes = [&](int codes, int least, int most) {  // as bits
    int bits = least;
    while (bits < most && (int64_t)codes << bits < p.K) ++bits;
    return bits;
  };
  if (bytes <= 32 << 20) {
    const int bits = lanes(16, 0, 6);
    launch_gemv<X, MR, 1, false>(p, bits, 64 >> bits, stream);
    return;
  }
  const int rows = p.K >= 1024 ? 16 : 64;
  const bool lines =
      ((uintptr_t)p.w | (uintptr_t)p.wsr | (uintptr_t)p.wsb) % 128 == 0;
  const bool once = bytes >= 256 << 20;
  if (once && lines && p.K > 96)
    launch_gemv<X, MR, 2, true>(p, 3, rows, stream);
  else if (once && p.K >= 2048)
    launch_gemv<X, MR, 4, true>(p, 6, rows, stream);
  else
    launch_gemv<X, MR, 2, false>(p, p.K <= 16 ? 0 : lanes(32, 1, 4), rows,
                                 stream);
}

template <typename X>
void choose_gemv(const DesInt8Product& p, hipStream_t stream) {
  if (p.M == 1)
    choose_gemv_rows<X, 1>(p, stream);
  else
    choose_gemv_rows<X, 4>(p, stream);
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
  const DesInt8Product& q = *p;
  const bool gemv = q.M <= 4 && q.M * (int64_t)q.K <= 48 * 1024;
  if (q.x) {
    if (gemv)
      choose_gemv<int8_t>(q, stream);
    else if (q.M > 64 && q.N > 32)
      launch_stream<int8_t, 4, 4>(q, 1, 1, stream);
    else
      choose_stream<int8_t>(q, stream);
  } else if (q.xelem == ELEM_F32) {
    gemv ? choose_gemv<float>(q, stream) : choose_stream<float>(q, stream);
  } else if (q.xelem == ELEM_BF16) {
    gemv ? choose_gemv<Bf16>(q, stream) : choose_stream<Bf16>(q, stream);
  } else {
    gemv ? choose_gemv<_Float16>(q, stream)
         : choose_stream<_Float16>(q, stream);
  }
}
