// Quantisation of matrices into microscaled blocks and back (gfx950).
#include <algorithm>

#include "mx.h"

namespace mpq {
namespace {

// One lane holds eight values, four lanes a block: a wave reads and writes 512 consecutive values of a row at a
// time, U times.  The task (row, piece of 512 U values) is the same for a whole wave, so its division runs
// on the scalar unit.  Bound by the memory: 4096 x 14336 values of bf16 to mxfp4 in 27 us and back in 23 (149 MB each,
// 5.5 and 6.4 TB/s, part of them from the last-level cache); one row takes 2 us each way.
template <int TYPE, int FMT, int U>
__global__ __launch_bounds__(256) void quantize_kernel(const char* __restrict__ x, int64_t rows, int64_t cols,
                                                       int64_t ld, int64_t padded, uint32_t pieces,
                                                       uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  constexpr int kSize = TYPE == kMxF32 ? 4 : 2;
  const int lane = threadIdx.x & 63;
  const uint64_t task = (uint64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = (int64_t)(task / pieces);
  if (row >= rows) return;
  const int64_t c0 = (int64_t)(task % pieces) * (512 * U) + lane * 8;
  const char* src = x + row * ld * kSize;
  float v[U][8];
#pragma unroll
  for (int u = 0; u < U; ++u) mx_load8<TYPE>(src + (c0 + 512 * u) * kSize, cols - (c0 + 512 * u), v[u]);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t c = c0 + 512 * u;
    const uint32_t byte = mx_scale_byte<FMT>(mx_top_quad(mx_top8(v[u])));
    const u32x2 w = mx_encode8<FMT>(v[u], byte);
    if (c < padded) {
      if constexpr (FMT == kMxFp4) {
        *reinterpret_cast<uint32_t*>(codes + (row * padded + c) / 2) = w[0];
      } else {
        *reinterpret_cast<u32x2*>(codes + row * padded + c) = w;
      }
      if ((lane & 3) == 0) scales[(row * padded + c) / kMxBlock] = (uint8_t)byte;
    }
  }
}

template <int TYPE>
__device__ __forceinline__ void store8(void* p, int64_t left, const float (&v)[8]) {
  if constexpr (TYPE == kMxF32) {
    if (left >= 8) {
      store_any<f32x4>(p, f32x4{v[0], v[1], v[2], v[3]});
      store_any<f32x4>(static_cast<char*>(p) + 16, f32x4{v[4], v[5], v[6], v[7]});
      return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) static_cast<float*>(p)[i] = v[i];
  }
}

template <int TYPE, int FMT, int U>
__global__ __launch_bounds__(256) void dequantize_kernel(const uint8_t* __restrict__ codes,
                                                         const uint8_t* __restrict__ scales, int64_t rows, int64_t cols,
                                                         int64_t padded, uint32_t pieces, char* __restrict__ out,
                                                         int64_t ld) {
  constexpr int kSize = TYPE == kMxF32 ? 4 : 2;
  const int lane = threadIdx.x & 63;
  const uint64_t task = (uint64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = (int64_t)(task / pieces);
  if (row >= rows) return;
  const int64_t c0 = (int64_t)(task % pieces) * (512 * U) + lane * 8;
  u32x2 w[U];
  uint32_t byte[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t c = c0 + 512 * u;
    w[u] = u32x2{0u, 0u};
    byte[u] = 1u;
    if (c < cols) {  // the row is stored in whole blocks, so all eight codes are there
      if constexpr (FMT == kMxFp4) w[u][0] = *reinterpret_cast<const uint32_t*>(codes + (row * padded + c) / 2);
      else w[u] = *reinterpret_cast<const u32x2*>(codes + row * padded + c);
      byte[u] = scales[(row * padded + c) / kMxBlock];
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t c = c0 + 512 * u;
    if (c >= cols) continue;
    const float s = mx_scale(byte[u]);
    char* dst = out + (row * ld + c) * kSize;
    if constexpr (TYPE == kMxF32) {
      float v[8];
      f32x2 p;
      if constexpr (FMT == kMxFp4) {
        p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u][0], s, 0);
        v[0] = p[0], v[1] = p[1];
        p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u][0], s, 1);
        v[2] = p[0], v[3] = p[1];
        p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u][0], s, 2);
        v[4] = p[0], v[5] = p[1];
        p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u][0], s, 3);
        v[6] = p[0], v[7] = p[1];
      } else {
        p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w[u][0], s, false);
        v[0] = p[0], v[1] = p[1];
        p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w[u][0], s, true);
        v[2] = p[0], v[3] = p[1];
        p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w[u][1], s, false);
        v[4] = p[0], v[5] = p[1];
        p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w[u][1], s, true);
        v[6] = p[0], v[7] = p[1];
      }
      store8<TYPE>(dst, cols - c, v);
    } else {
      const u32x4 r = mx_decode8<FMT, TYPE>(w[u], s);
      if (cols - c >= 8) {
        store_any<u32x4>(dst, r);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i < cols - c) reinterpret_cast<uint16_t*>(dst)[i] = (uint16_t)(r[i / 2] >> (16 * (i % 2)));
      }
    }
  }
}

// Lanes take one octet each where that fills no more than the card's waves once, four where rows are plenty.
struct Shape {
  int unroll;
  uint32_t pieces;
  int64_t most;  // rows of a launch
  unsigned blocks(int64_t rows) const { return (unsigned)((rows * pieces + 3) / 4); }
};

Shape shape_of(int64_t rows, int64_t padded) {
  Shape s;
  s.unroll = rows * padded >= (int64_t)512 * 4 * 4096 ? 4 : 1;
  s.pieces = (uint32_t)((padded + 512 * s.unroll - 1) / (512 * s.unroll));
  s.most = kMxLaunch / 64 / s.pieces;
  return s;
}

template <int TYPE, int FMT>
void launch_quantize(const Shape& s, const void* x, int64_t rows, int64_t cols, int64_t ld, int64_t padded,
                     uint8_t* codes, uint8_t* scales, hipStream_t stream) {
  if (s.unroll == 4)
    hipLaunchKernelGGL((quantize_kernel<TYPE, FMT, 4>), dim3(s.blocks(rows)), dim3(256), 0, stream,
                       static_cast<const char*>(x), rows, cols, ld, padded, s.pieces, codes, scales);
  else
    hipLaunchKernelGGL((quantize_kernel<TYPE, FMT, 1>), dim3(s.blocks(rows)), dim3(256), 0, stream,
                       static_cast<const char*>(x), rows, cols, ld, padded, s.pieces, codes, scales);
}

template <int TYPE, int FMT>
void launch_dequantize(const Shape& s, const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t cols,
                       int64_t padded, void* out, int64_t ld, hipStream_t stream) {
  if (s.unroll == 4)
    hipLaunchKernelGGL((dequantize_kernel<TYPE, FMT, 4>), dim3(s.blocks(rows)), dim3(256), 0, stream, codes, scales, rows,
                       cols, padded, s.pieces, static_cast<char*>(out), ld);
  else
    hipLaunchKernelGGL((dequantize_kernel<TYPE, FMT, 1>), dim3(s.blocks(rows)), dim3(256), 0, stream, codes, scales, rows,
                       cols, padded, s.pieces, static_cast<char*>(out), ld);
}

}  // namespace

hipError_t mx_quantize_rows(const void* x, int type, int64_t rows, int64_t cols, int64_t ld, int fmt, uint8_t* codes,
                            uint8_t* scales, hipStream_t stream) {
  const int64_t padded = mx_padded(cols);
  const Shape s = shape_of(rows, padded);
  for (int64_t r = 0; r < rows; r += s.most) {
    const int64_t n = std::min(s.most, rows - r);
    const char* from = static_cast<const char*>(x) + r * ld * (type == kMxF32 ? 4 : 2);
    uint8_t *c = codes + r * mx_code_bytes(padded, fmt), *b = scales + r * (padded / kMxBlock);
#define MPQ_Q(T, F) launch_quantize<T, F>(s, from, n, cols, ld, padded, c, b, stream)
    if (fmt == kMxFp4) {
      if (type == kMxF32) MPQ_Q(kMxF32, kMxFp4);
      else if (type == kMxBf16) MPQ_Q(kMxBf16, kMxFp4);
      else MPQ_Q(kMxF16, kMxFp4);
    } else {
      if (type == kMxF32) MPQ_Q(kMxF32, kMxFp8);
      else if (type == kMxBf16) MPQ_Q(kMxBf16, kMxFp8);
      else MPQ_Q(kMxF16, kMxFp8);
    }
#undef MPQ_Q
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace mpq

extern "C" int mpq_mx_quantize(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ld, int fmt,
                               uint8_t* codes, uint8_t* scales, hipStream_t stream) {
  using namespace mpq;
  MPQ_CHECK_ARG(fmt == kMxFp4 || fmt == kMxFp8, "mpq_mx_quantize: unknown format %d", fmt);
  MPQ_CHECK_ARG(dtype >= kMxF32 && dtype <= kMxF16, "mpq_mx_quantize: unknown type %d", dtype);
  MPQ_CHECK_ARG(rows >= 0 && cols >= 1 && ld >= cols, "mpq_mx_quantize: bad shape %lld x %lld (ld %lld)",
                (long long)rows, (long long)cols, (long long)ld);
  if (rows == 0) return kOk;
  MPQ_CHECK_ARG(x && codes && scales, "mpq_mx_quantize: null pointer");
  MPQ_CHECK_ARG(cols <= ((int64_t)1 << 31) && rows <= ((int64_t)1 << 40) / mx_padded(cols),
                "mpq_mx_quantize: extent too large");
  MPQ_HIP_TRY(mx_quantize_rows(x, dtype, rows, cols, ld, fmt, codes, scales, stream));
  return kOk;
}

extern "C" int mpq_mx_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t cols, int fmt,
                                 void* out, int dtype, int64_t ld, hipStream_t stream) {
  using namespace mpq;
  MPQ_CHECK_ARG(fmt == kMxFp4 || fmt == kMxFp8, "mpq_mx_dequantize: unknown format %d", fmt);
  MPQ_CHECK_ARG(dtype >= kMxF32 && dtype <= kMxF16, "mpq_mx_dequantize: unknown type %d", dtype);
  MPQ_CHECK_ARG(rows >= 0 && cols >= 1 && ld >= cols, "mpq_mx_dequantize: bad shape %lld x %lld (ld %lld)",
                (long long)rows, (long long)cols, (long long)ld);
  if (rows == 0) return kOk;
  MPQ_CHECK_ARG(codes && scales && out, "mpq_mx_dequantize: null pointer");
  MPQ_CHECK_ARG(cols <= ((int64_t)1 << 31) && rows <= ((int64_t)1 << 40) / mx_padded(cols),
                "mpq_mx_dequantize: extent too large");
  const int64_t padded = mx_padded(cols);
  const Shape s = shape_of(rows, padded);
  for (int64_t r = 0; r < rows; r += s.most) {
    const int64_t n = std::min(s.most, rows - r);
    const uint8_t *c = codes + r * mx_code_bytes(padded, fmt), *b = scales + r * (padded / kMxBlock);
    char* to = static_cast<char*>(out) + r * ld * (dtype == kMxF32 ? 4 : 2);
#define MPQ_D(T, F) launch_dequantize<T, F>(s, c, b, n, cols, padded, to, ld, stream)
    if (fmt == kMxFp4) {
      if (dtype == kMxF32) MPQ_D(kMxF32, kMxFp4);
      else if (dtype == kMxBf16) MPQ_D(kMxBf16, kMxFp4);
      else MPQ_D(kMxF16, kMxFp4);
    } else {
      if (dtype == kMxF32) MPQ_D(kMxF32, kMxFp8);
      else if (dtype == kMxBf16) MPQ_D(kMxBf16, kMxFp8);
      else MPQ_D(kMxF16, kMxFp8);
    }
#undef MPQ_D
    MPQ_LAUNCH_CHECK();
  }
  return kOk;
}
