// Microscaled blocks (gfx950): 32 consecutive values share one power-of-two scale.
//
// Formats: kMxFp4 holds E2M1 values {0, .5, 1, 1.5, 2, 3, 4, 6} and their negatives, two codes a byte (the
// first value in the low half); kMxFp8 holds E4M3 values up to 448, one a byte.  A block's scale is
// 2^(floor(log2(max |x|)) - emax), emax = 2 or 8, held as its biased exponent in one byte (at least 1, so
// every scale is a normal float; a block of zeros has 1).  Values are x / scale rounded to nearest, ties to
// even, saturating.  A block that holds a NaN or an infinity has scale byte 255, which stands for NaN: all
// its values read back as NaN and poison what is computed from them, on the matrix cores too.
//
// The conversions are the hardware's scaled ones (one rounding, checked over all bf16 and f16 inputs against
// the definition); they overflow to NaN in E4M3, so those inputs are clamped to +-448 scales first.
#pragma once

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "common.h"

namespace mpq {

enum MxFormat : int { kMxFp4 = 0, kMxFp8 = 1 };
enum MxType : int { kMxF32 = 0, kMxBf16 = 1, kMxF16 = 2 };

constexpr int kMxBlock = 32;
constexpr int kMxRow = 256;  // matrices: rows are padded with zeros to whole 256-value pieces

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short i16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <int FMT>
struct MxTraits {
  static constexpr int kEmax = FMT == kMxFp4 ? 2 : 8;
  static constexpr int kOctet = FMT == kMxFp4 ? 4 : 8;  // bytes of eight codes
};

// 16-bit element types by their MxType.
template <int TYPE>
struct MxHalf;
template <>
struct MxHalf<kMxBf16> {
  typedef bf16x2 pair;
  typedef bf16x8 oct;
};
template <>
struct MxHalf<kMxF16> {
  typedef f16x2 pair;
  typedef f16x8 oct;
};

template <class To, class From>
__device__ __forceinline__ To bits_as(const From& f) {
  static_assert(sizeof(To) == sizeof(From), "same size");
  To t;
  __builtin_memcpy(&t, &f, sizeof(To));
  return t;
}

// Loads and stores of any alignment (the hardware takes them; rows of odd lengths start anywhere).
template <class T>
__device__ __forceinline__ T load_any(const void* p) {
  struct __attribute__((packed)) U {
    T v;
  };
  return reinterpret_cast<const U*>(p)->v;
}
template <class T>
__device__ __forceinline__ void store_any(void* p, T v) {
  struct __attribute__((packed)) U {
    T v;
  };
  reinterpret_cast<U*>(p)->v = v;
}

__device__ __forceinline__ float mx_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// Eight values of a row, as float.  `left`: values of the row from p on; those behind its end are zero.
template <int TYPE>
__device__ __forceinline__ void mx_load8(const void* __restrict__ p, int64_t left, float (&v)[8]) {
  if (left >= 8) {
    if constexpr (TYPE == kMxF32) {
      const f32x4 a = load_any<f32x4>(p), b = load_any<f32x4>(static_cast<const char*>(p) + 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = a[i];
        v[4 + i] = b[i];
      }
    } else {
      const typename MxHalf<TYPE>::oct a = load_any<typename MxHalf<TYPE>::oct>(p);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = (float)a[i];
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] = 0.f;
    if (i < left) {
      if constexpr (TYPE == kMxF32) v[i] = static_cast<const float*>(p)[i];
      if constexpr (TYPE == kMxBf16) v[i] = (float)static_cast<const __bf16*>(p)[i];
      if constexpr (TYPE == kMxF16) v[i] = (float)static_cast<const _Float16*>(p)[i];
    }
  }
}

// Largest |v| as bits: integer order is the order of magnitudes, with infinities and NaNs on top.
__device__ __forceinline__ uint32_t mx_top8(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  return m;
}

// Over the four lanes that hold a block.
__device__ __forceinline__ uint32_t mx_top_quad(uint32_t m) {
  m = max(m, (uint32_t)__shfl_xor((int)m, 1, 64));
  return max(m, (uint32_t)__shfl_xor((int)m, 2, 64));
}

template <int FMT>
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t top) {
  const int e = (int)(top >> 23);
  return e == 255 ? 255u : (uint32_t)max(e - MxTraits<FMT>::kEmax, 1);
}

// Codes of eight values under a block's scale: 4 bytes (the first of w) or 8.
template <int FMT>
__device__ __forceinline__ u32x2 mx_encode8(const float (&v)[8], uint32_t byte) {
  const float s = mx_scale(byte);
  u32x2 w = {0u, 0u};
  if constexpr (FMT == kMxFp4) {
    w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[0], v[0], v[1], s, 0);
    w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[0], v[2], v[3], s, 1);
    w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[0], v[4], v[5], s, 2);
    w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[0], v[6], v[7], s, 3);
  } else {
    const float lim = 448.f * s;
    float c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = __builtin_amdgcn_fmed3f(v[i], -lim, lim);
    i16x2 a = {0, 0}, b = {0, 0};
    a = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(a, c[0], c[1], s, false);
    a = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(a, c[2], c[3], s, true);
    b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(b, c[4], c[5], s, false);
    b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(b, c[6], c[7], s, true);
    w[0] = bits_as<uint32_t>(a);
    w[1] = bits_as<uint32_t>(b);
  }
  return w;
}

// Pair P (0..3) of the eight values of an octet's codes, in 16 bits.  Exact in bf16; in f16 as far as f16 reaches.
template <int FMT, int TYPE, int P>
__device__ __forceinline__ uint32_t mx_decode_pair(u32x2 w, float s) {
  if constexpr (FMT == kMxFp4) {
    if constexpr (TYPE == kMxBf16) return bits_as<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], s, P));
    else return bits_as<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w[0], s, P));
  } else {
    if constexpr (TYPE == kMxBf16)
      return bits_as<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[P / 2], s, P % 2 != 0));
    else return bits_as<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[P / 2], s, P % 2 != 0));
  }
}

// The eight values of an octet as one matrix-core operand.
template <int FMT, int TYPE>
__device__ __forceinline__ u32x4 mx_decode8(u32x2 w, float s) {
  u32x4 r;
  r[0] = mx_decode_pair<FMT, TYPE, 0>(w, s);
  r[1] = mx_decode_pair<FMT, TYPE, 1>(w, s);
  r[2] = mx_decode_pair<FMT, TYPE, 2>(w, s);
  r[3] = mx_decode_pair<FMT, TYPE, 3>(w, s);
  return r;
}

// Writes rows x cols values as codes (rows x padded cols) and scale bytes; the padding is zeros.  Defined in
// mx_quant.hip.
hipError_t mx_quantize_rows(const void* x, int type, int64_t rows, int64_t cols, int64_t ld, int fmt, uint8_t* codes,
                            uint8_t* scales, hipStream_t stream);

// Threads of one launch of the kernels that go over any number of rows: a launch whose threads along x pass 2^32 is cut to
// the rest without an error, so longer calls are several launches.
constexpr int64_t kMxLaunch = (int64_t)1 << 31;

__host__ __device__ inline int64_t mx_padded(int64_t cols) { return (cols + kMxRow - 1) / kMxRow * kMxRow; }
__host__ __device__ inline int64_t mx_code_bytes(int64_t padded, int fmt) { return fmt == kMxFp4 ? padded / 2 : padded; }

}  // namespace mpq
