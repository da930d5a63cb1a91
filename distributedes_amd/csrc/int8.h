// 8-bit rows: what the quantising and the product kernels share.
//
// A row x of K values is held as codes q in [-127, 127] and one fp32 scale s:
//     a = max |x_k|,  s = max(fp32(a / 127), 2^-126),
//     q_k = the whole number nearest to x_k / s, ties to even.
// The quotient is the exact one: codes do not depend on how a division rounds,
// so kernel, torch twin and a 64-bit oracle agree bit for bit.  The bound
// 2^-126 keeps the scale of rows of zeros (and of values below any use) a
// normal number, so that nothing divides by zero.  A row that holds a NaN or an
// infinity gets scale NaN and codes 0: it shows in every product.
#pragma once
#include <stdint.h>

#ifdef __HIPCC__
#include <hip/hip_runtime.h>

namespace des {

// element types of float rows and of results, as the bindings pass them
enum Elem : int { ELEM_F32 = 0, ELEM_BF16 = 1, ELEM_F16 = 2 };

struct Bf16 { uint16_t bits; };

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(_Float16 v) { return (float)v; }
__device__ __forceinline__ float to_f32(Bf16 v) {
  return __uint_as_float((uint32_t)v.bits << 16);
}

template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) {
  return v;
}
template <> __device__ __forceinline__ _Float16 from_f32<_Float16>(float v) {
  return (_Float16)v;
}
// to nearest, ties to even, a NaN stays one: v_cvt_pk_bf16_f32
template <> __device__ __forceinline__ Bf16 from_f32<Bf16>(float v) {
  return Bf16{__builtin_bit_cast(uint16_t, (__bf16)v)};
}

// |v| as bits: among floats these order like the values, infinity and NaN above
// all others, so one unsigned maximum finds both the largest and the unusable
__device__ __forceinline__ uint32_t abs_bits(float v) {
  return __float_as_uint(v) & 0x7FFFFFFFu;
}

struct RowScale {
  float scale, inv;  // inv = 0 where the row is unusable
};

__device__ __forceinline__ RowScale row_scale(uint32_t top) {
  RowScale r;
  if (top >= 0x7F800000u) {
    r.scale = __uint_as_float(0x7FC00000u);
    r.inv = 0.f;
  } else {
    r.scale = fmaxf(__uint_as_float(top) / 127.0f, 1.17549435e-38f);
    r.inv = 1.0f / r.scale;
  }
  return r;
}

// Four codes in one word.  Adding 1.5 * 2^23 rounds v * inv to a whole number,
// ties to even, which the sum's low byte holds as int8.  That is at most one
// step off, and only next to a border of two codes; the remainder v - q s has at
// most 24 bits there, so its fma is exact and tells on which side of the border
// (or on it) v lies.
__device__ __forceinline__ uint32_t row_codes(const float (&v)[4], RowScale r) {
  const float whole = 12582912.0f, border = 0.5f * r.scale;
  float t[4], rem[4];
  bool near = false;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    t[j] = fmaf(v[j], r.inv, whole);
    rem[j] = fmaf(whole - t[j], r.scale, v[j]);
    near |= fabsf(rem[j]) >= border;
  }
  // scales below 2^-125 have borders that half a scale cannot hold
  if (__builtin_expect(near || r.scale < 2.3509887e-38f, 0)) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float twice = 2.0f * fabsf(rem[j]);
      if (twice > r.scale ||
          (twice == r.scale && (__float_as_uint(t[j]) & 1)))
        t[j] += rem[j] > 0.f ? 1.0f : -1.0f;
    }
  }
  if (!(r.inv > 0.f)) return 0;
  const uint32_t low = __builtin_amdgcn_perm(
      __float_as_uint(t[1]), __float_as_uint(t[0]), 0x0c0c0400u);
  return low | __builtin_amdgcn_perm(__float_as_uint(t[3]),
                                     __float_as_uint(t[2]), 0x04000c0cu);
}

template <typename T, int V>
struct __attribute__((packed, aligned(sizeof(T)))) Vec { T v[V]; };

}  // namespace des
#endif  // __HIPCC__

// One batch of products, as the bindings pass it.  Strides in elements; the
// elements of a row are next to each other.
struct DesInt8Product {
  const int8_t* x;      // [B, M, K]
  const float* sx;      // [B, M]; null: xf is quantised on the way
  const void* xf;       // [B, M, K] float rows of type xelem
  const int8_t* w;      // [B, N, K]
  const float* sw;      // [B, N]
  const float* bias;    // nullable [B, N]
  void* y;              // [B, M, N]
  int64_t B;
  int32_t M, N, K;
  int64_t xsb, xsr, wsb, wsr;
  int32_t act;          // 0 none, 1 relu, 2 tanh
  int32_t out;          // des::Elem
  int32_t xelem;        // des::Elem
  // whether a row's last 16 codes may be read whole: the bytes behind the row
  // belong to its storage
  int32_t xwhole, wwhole;
};

enum DesInt8Plan : int {
  DES_INT8_GEMV,    // up to 4 tokens: weights as a stream
  DES_INT8_STREAM,  // few tokens, or few results for a long K
  DES_INT8_TILED    // many tokens: operands through shared memory
};

// Which kernel takes a product of M tokens, N channels and K codes for B
// members.  A stream of weights holds its tokens' codes in shared memory, the
// next kernel only those that it makes from floats (des_int8_fused).
// Tiles of 64 x 64 results leave the chip empty below about 100 of them: 128
// tokens x 512 x 3136 take 5.2 us as a stream and 10 us in tiles, 1024 tokens
// 15 and 10.7.
inline DesInt8Plan des_int8_plan(int64_t B, int64_t M, int64_t N, int64_t K) {
  if (M <= 4 && M * K <= 48 * 1024) return DES_INT8_GEMV;
  if (M <= 16 || K == 0) return DES_INT8_STREAM;
  if (M <= 32 && B > 1) return DES_INT8_STREAM;
  return B * ((M + 63) / 64) * ((N + 63) / 64) < 100 ? DES_INT8_STREAM
                                                     : DES_INT8_TILED;
}

// Whether int8_linear is one launch (every block quantises its tokens itself) or
// two: a block's 1000 values take about 0.1 us, a launch of its own 2 to 4.
inline bool des_int8_fused(int64_t M, int64_t K) {
  return M <= 4 ? M * K <= 16384 : M <= 16 && K <= 512;
}
