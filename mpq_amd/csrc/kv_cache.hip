// Writing tokens into the quantised key/value cache and reading them back (gfx950).  One pass over the data
// each: a lane holds an octet of one head of one token, four lanes a block.  Bound by the memory: 16 prompts of 500
// to 2048 tokens, 8 heads of 128, bf16 and mxfp4: written in 21 us and read in 21 (97 MB each, 4.6 TB/s).
#include <algorithm>
#include <type_traits>

#include "kv_cache.h"

namespace mpq {
namespace {

template <int TYPE, int FMT, int D>
__global__ __launch_bounds__(256) void write_kernel(const char* __restrict__ k, const char* __restrict__ v,
                                                    int64_t tokens, int64_t k_ts, int64_t k_hs, int64_t v_ts,
                                                    int64_t v_hs, const int64_t* __restrict__ slots, KvCache c) {
  typedef KvLayout<FMT, D> L;
  constexpr int kOcts = D / 8;
  const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int oct = (int)(item % kOcts);
  const int64_t pair = item / kOcts;  // (token, head)
  const int64_t t = pair / c.heads;
  const int head = (int)(pair - t * c.heads);
  if (t >= tokens) return;
  const int64_t slot = slots[t];
  if (slot < 0 || slot >= c.pages << c.shift) return;
  const int64_t row = L::row0(c, slot >> c.shift, head) + (slot & (c.page - 1));
  float a[8], b[8];
  mx_load8<TYPE>(k + (t * k_ts + head * k_hs + oct * 8) * 2, 8, a);
  mx_load8<TYPE>(v + (t * v_ts + head * v_hs + oct * 8) * 2, 8, b);
  const uint32_t sa = mx_scale_byte<FMT>(mx_top_quad(mx_top8(a)));
  const uint32_t sb = mx_scale_byte<FMT>(mx_top_quad(mx_top8(b)));
  const u32x2 ca = mx_encode8<FMT>(a, sa), cb = mx_encode8<FMT>(b, sb);
  uint8_t* kp = c.kc + row * L::kRow + oct * L::kOct;
  uint8_t* vp = c.vc + L::v_code(row, oct);
  if constexpr (FMT == kMxFp4) {
    *reinterpret_cast<uint32_t*>(kp) = ca[0];
    *reinterpret_cast<uint32_t*>(vp) = cb[0];
  } else {
    *reinterpret_cast<u32x2*>(kp) = ca;
    *reinterpret_cast<u32x2*>(vp) = cb;
  }
  if ((oct & 3) == 0) {
    c.ks[row * L::kScales + oct / 4] = (uint8_t)sa;
    c.vs[L::v_scale(row, oct / 4)] = (uint8_t)sb;
  }
}

// Tokens `first` to `total` of all sequences one after the other: starts[i] .. starts[i + 1] are those of sequence i.
template <int TYPE, int FMT, int D>
__global__ __launch_bounds__(256) void read_kernel(const int32_t* __restrict__ table, int batch, int64_t width,
                                                   const int32_t* __restrict__ starts, int64_t first, int64_t total,
                                                   KvCache c, char* __restrict__ k, char* __restrict__ v) {
  typedef KvLayout<FMT, D> L;
  constexpr int kOcts = D / 8;
  const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int oct = (int)(item % kOcts);
  const int64_t pair = first * c.heads + item / kOcts;
  const int64_t t = pair / c.heads;
  const int head = (int)(pair - t * c.heads);
  if (t >= total) return;
  int lo = 0, hi = batch;  // the last sequence that starts at or before t
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (starts[mid] <= t) lo = mid;
    else hi = mid;
  }
  u32x4 ko = {0u, 0u, 0u, 0u}, vo = {0u, 0u, 0u, 0u};
  const int64_t pos = t - starts[lo];
  if (pos >= 0 && t < starts[lo + 1] && (pos >> c.shift) < width) {
    const int64_t page = table[lo * width + (pos >> c.shift)];
    if (page >= 0 && page < c.pages) {
      const int64_t row = L::row0(c, page, head) + (pos & (c.page - 1));
      const uint8_t* kp = c.kc + row * L::kRow + oct * L::kOct;
      const uint8_t* vp = c.vc + L::v_code(row, oct);
      u32x2 kw = {0u, 0u}, vw = {0u, 0u};
      if constexpr (FMT == kMxFp4) {
        kw[0] = *reinterpret_cast<const uint32_t*>(kp);
        vw[0] = *reinterpret_cast<const uint32_t*>(vp);
      } else {
        kw = *reinterpret_cast<const u32x2*>(kp);
        vw = *reinterpret_cast<const u32x2*>(vp);
      }
      ko = mx_decode8<FMT, TYPE>(kw, mx_scale(c.ks[row * L::kScales + oct / 4]));
      vo = mx_decode8<FMT, TYPE>(vw, mx_scale(c.vs[L::v_scale(row, oct / 4)]));
    }
  }
  *reinterpret_cast<u32x4*>(k + (pair * D + oct * 8) * 2) = ko;
  *reinterpret_cast<u32x4*>(v + (pair * D + oct * 8) * 2) = vo;
}

}  // namespace
}  // namespace mpq

#define MPQ_KV_PICK(KERNEL, ...)                                                                             \
  do {                                                                                                       \
    const auto go = [&](auto type, auto f, auto d) {                                                         \
      hipLaunchKernelGGL((KERNEL<decltype(type)::value, decltype(f)::value, decltype(d)::value>), grid, dim3(256), 0, \
                         stream, __VA_ARGS__);                                                               \
    };                                                                                                       \
    const auto by_dim = [&](auto type, auto f) {                                                             \
      if (dim == 64) go(type, f, std::integral_constant<int, 64>{});                                         \
      else go(type, f, std::integral_constant<int, 128>{});                                                  \
    };                                                                                                       \
    const auto by_fmt = [&](auto type) {                                                                     \
      if (fmt == kMxFp4) by_dim(type, std::integral_constant<int, kMxFp4>{});                                \
      else by_dim(type, std::integral_constant<int, kMxFp8>{});                                              \
    };                                                                                                       \
    if (dtype == kMxBf16) by_fmt(std::integral_constant<int, kMxBf16>{});                                    \
    else by_fmt(std::integral_constant<int, kMxF16>{});                                                      \
  } while (0)

#define MPQ_KV_CHECK(NAME)                                                                                   \
  MPQ_CHECK_ARG(fmt == kMxFp4 || fmt == kMxFp8, NAME ": unknown format %d", fmt);                            \
  MPQ_CHECK_ARG(dtype == kMxBf16 || dtype == kMxF16, NAME ": unknown type %d", dtype);                       \
  MPQ_CHECK_ARG(kv_dim_ok(dim), NAME ": head size %d (64 or 128)", dim);                                     \
  MPQ_CHECK_ARG(heads >= 1 && heads <= 65535, NAME ": %d heads", heads);                                     \
  MPQ_CHECK_ARG(page >= 16 && page <= 65536 && (page & (page - 1)) == 0,                                     \
                NAME ": pages of %d tokens (a power of two from 16)", page);                                 \
  MPQ_CHECK_ARG(pages >= 1 && pages <= ((int64_t)1 << 31), NAME ": %lld pages", (long long)pages);           \
  MPQ_CHECK_ARG(k_codes && k_scales && v_codes && v_scales, NAME ": null cache")

extern "C" int mpq_kv_write(const void* k, const void* v, int dtype, int64_t tokens, int64_t k_token_stride,
                            int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride,
                            const int64_t* slots, int fmt, int heads, int dim, int page, int64_t pages,
                            uint8_t* k_codes, uint8_t* k_scales, uint8_t* v_codes, uint8_t* v_scales,
                            hipStream_t stream) {
  using namespace mpq;
  MPQ_KV_CHECK("mpq_kv_write");
  MPQ_CHECK_ARG(tokens >= 0, "mpq_kv_write: %lld tokens", (long long)tokens);
  if (tokens == 0) return kOk;
  MPQ_CHECK_ARG(k && v && slots, "mpq_kv_write: null pointer");
  MPQ_CHECK_ARG(tokens <= ((int64_t)1 << 34) / heads, "mpq_kv_write: extent too large");
  const KvCache c = {k_codes, k_scales, v_codes, v_scales, pages, heads, page, __builtin_ctz(page)};
  const int64_t most = kMxLaunch / (heads * (dim / 8));
  for (int64_t t = 0; t < tokens; t += most) {
    const int64_t n = std::min(most, tokens - t);
    const dim3 grid((unsigned)mpq_cdiv(n * heads * (dim / 8), 256));
    MPQ_KV_PICK(write_kernel, static_cast<const char*>(k) + t * k_token_stride * 2,
                static_cast<const char*>(v) + t * v_token_stride * 2, n, k_token_stride, k_head_stride, v_token_stride,
                v_head_stride, slots + t, c);
    MPQ_LAUNCH_CHECK();
  }
  return kOk;
}

extern "C" int mpq_kv_read(const int32_t* block_table, int64_t batch, int64_t table_width, const int32_t* starts,
                           int64_t total, int fmt, int heads, int dim, int page, int64_t pages,
                           const uint8_t* k_codes, const uint8_t* k_scales, const uint8_t* v_codes,
                           const uint8_t* v_scales, void* k_out, void* v_out, int dtype, hipStream_t stream) {
  using namespace mpq;
  MPQ_KV_CHECK("mpq_kv_read");
  MPQ_CHECK_ARG(batch >= 0 && batch <= (1 << 24) && table_width >= 0 && total >= 0, "mpq_kv_read: bad shape");
  if (total == 0) return kOk;
  MPQ_CHECK_ARG(batch >= 1 && starts && (block_table || table_width == 0) && k_out && v_out,
                "mpq_kv_read: null pointer or no sequence");
  MPQ_CHECK_ARG(total <= ((int64_t)1 << 34) / heads, "mpq_kv_read: extent too large");
  const KvCache c = {const_cast<uint8_t*>(k_codes), const_cast<uint8_t*>(k_scales), const_cast<uint8_t*>(v_codes),
                     const_cast<uint8_t*>(v_scales), pages, heads, page, __builtin_ctz(page)};
  const int64_t most = kMxLaunch / (heads * (dim / 8));
  for (int64_t t = 0; t < total; t += most) {
    const dim3 grid((unsigned)mpq_cdiv(std::min(most, total - t) * heads * (dim / 8), 256));
    MPQ_KV_PICK(read_kernel, block_table, (int)batch, table_width, starts, t, total, c, static_cast<char*>(k_out),
                static_cast<char*>(v_out));
    MPQ_LAUNCH_CHECK();
  }
  return kOk;
}
