// Product of a quantised linear (gfx950): out = Q(x) W^T + bias with W in mxfp4 and Q(x) in mxfp4 or mxfp8.
//
// The matrix cores take both operands as codes with one scale byte for each 32 values and apply the scales inside
// the product, so nothing is dequantised.  Accumulators are fp32; results are rounded once.  The products of two 4-bit
// values of a block span 2^8 and are summed exactly.  With an 8-bit operand the instruction cuts the terms of a block
// at 2^-13 of its largest one (measured with two terms of one block), about 1e-4 of a sum: taken all the same, since
// the format has already rounded every value to 2^-4 and the way around it, 16-bit products of dequantised
// values, runs at half the rate; between blocks nothing is cut.  Which 32 values of the
// contraction sit at which place of an instruction is free as long as both operands agree; the kernels choose the
// order in which each lane's scale bytes lie side by side in memory (one load serves 2 or 4 instructions).
//
// Rows of codes are padded with zeros to whole 256-value pieces, so no load in the contraction is conditional; rows
// outside the matrices are read from the last row and never stored.
#include <algorithm>
#include <type_traits>

#include "mx.h"

namespace mpq {
namespace {

// ---- up to 16 tokens: bound by the bytes of W ----------------------------------------------------------------
//
// A work-group owns 16 output features; its waves share the contraction in 256-value pieces and add their
// sums through LDS in wave order.  A lane's operand of two 16x16x128 products is 32 contiguous bytes of W, loaded
// straight into the registers that the matrix core reads; quantised tokens come the same way, with the W that they meet.
// One token: 4096 -> 14336 in 8.9 us (31 MB, 3.5 TB/s, the start with the token's quantisation in it).
constexpr int kFewWaves = 8;

template <int OTYPE>
__device__ __forceinline__ void store_value(void* out, int64_t at, float v) {
  if constexpr (OTYPE == kMxF32) static_cast<float*>(out)[at] = v;
  else if constexpr (OTYPE == kMxBf16) static_cast<__bf16*>(out)[at] = (__bf16)v;
  else static_cast<_Float16*>(out)[at] = (_Float16)v;
}

template <int OTYPE>
__device__ __forceinline__ uint32_t pack_pair(float a, float b) {
  if constexpr (OTYPE == kMxBf16) return bits_as<uint32_t>(bf16x2{(__bf16)a, (__bf16)b});
  else return bits_as<uint32_t>(f16x2{(_Float16)a, (_Float16)b});
}

template <int XF, int S>
__device__ __forceinline__ f32x4 mfma16(u32x4 w, uint32_t ws, u32x4 x0, u32x4 x1, uint32_t xs, f32x4 c) {
  const i32x8 a = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
  const i32x8 b = {(int)x0[0], (int)x0[1], (int)x0[2], (int)x0[3], (int)x1[0], (int)x1[1], (int)x1[2], (int)x1[3]};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, XF == kMxFp4 ? 4 : 0, S, (int)ws, S, (int)xs);
}

// FUSED: the tokens are quantised into LDS by every work-group (XTYPE values x), else xc / xs hold them.
template <int XF, bool FUSED, int XTYPE, int OTYPE>
__global__ __launch_bounds__(64 * kFewWaves) void few_kernel(const char* __restrict__ x, int64_t ldx,
                                                             const uint8_t* __restrict__ xc,
                                                             const uint8_t* __restrict__ xs, int tokens,
                                                             int64_t cols, int64_t padded,
                                                             const uint8_t* __restrict__ wc,
                                                             const uint8_t* __restrict__ wsc, int64_t rows,
                                                             const float* __restrict__ bias,
                                                             void* __restrict__ out, int64_t ldo) {
  extern __shared__ __align__(16) char smem[];
  // pieces of a wave in flight beside those being worked on
  constexpr int U = FUSED ? 2 : 1, kXParts = XF == kMxFp4 ? 1 : 2;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n16 = lane & 15, g = lane >> 4;
  const int64_t f0 = (int64_t)blockIdx.x * 16;
  const int64_t row = min(f0 + n16, rows - 1);
  const uint8_t* wp = wc + row * (padded / 2) + 32 * g;
  const uint8_t* sp = wsc + row * (padded / kMxBlock) + 2 * g;
  const int chunks = (int)(padded / kMxRow);
  const int64_t xrow = mx_code_bytes(padded, XF) + (FUSED ? 16 : 0);  // LDS rows are shifted against each other
  const int64_t srow = padded / kMxBlock;

  struct Tokens {  // operands of two products
    u32x4 x[2][kXParts];
    uint32_t s;
  };
  struct Piece {
    u32x4 w[2];
    uint32_t s;
  };
  auto load_w = [&](int c, Piece& p) {
    p.w[0] = *reinterpret_cast<const u32x4*>(wp + (int64_t)c * 128);
    p.w[1] = *reinterpret_cast<const u32x4*>(wp + (int64_t)c * 128 + 16);
    p.s = *reinterpret_cast<const uint16_t*>(sp + (int64_t)c * 8);
  };
  auto load_x = [&](const char* codes, const uint8_t* scales, int c, Tokens& p) {
    p.s = 0x7f7f;
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < kXParts; ++i) p.x[s][i] = u32x4{0u, 0u, 0u, 0u};
    if (n16 < tokens) {
      const char* from;
      if constexpr (XF == kMxFp4) from = codes + n16 * xrow + (int64_t)c * 128 + 32 * g;
      // an 8-bit operand lane holds half blocks g / 2 and g / 2 + 2: the order of its 32 bytes
      else from = codes + n16 * xrow + (int64_t)c * 256 + 64 * (g >> 1) + 16 * (g & 1);
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int i = 0; i < kXParts; ++i)
          p.x[s][i] = *reinterpret_cast<const u32x4*>(from + (XF == kMxFp4 ? 16 * s : 32 * s + 128 * i));
      p.s = *reinterpret_cast<const uint16_t*>(scales + n16 * srow + c * 8 + 2 * g);
    }
  };
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  auto multiply = [&](const Piece& w, const Tokens& x) {
    acc = mfma16<XF, 0>(w.w[0], w.s, x.x[0][0], x.x[0][kXParts - 1], x.s, acc);
    acc = mfma16<XF, 1>(w.w[1], w.s, x.x[1][0], x.x[1][kXParts - 1], x.s, acc);
  };

  Piece w[U], nw[U];
  auto load_group_w = [&](int c0, Piece(&p)[U]) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c0 + u * kFewWaves < chunks) load_w(c0 + u * kFewWaves, p[u]);
  };
  load_group_w(wave, w);
  if constexpr (FUSED) {
    char* lc = smem;
    uint8_t* ls = reinterpret_cast<uint8_t*>(smem) + tokens * xrow;
    const int octets = (int)(padded / 8), items = tokens * octets;
    for (int i = threadIdx.x; i < items; i += 64 * kFewWaves) {
      const int t = i / octets, c = (i - t * octets) * 8;
      float v[8];
      mx_load8<XTYPE>(x + ((int64_t)t * ldx + c) * (XTYPE == kMxF32 ? 4 : 2), cols - c, v);
      const uint32_t byte = mx_scale_byte<XF>(mx_top_quad(mx_top8(v)));
      const u32x2 e = mx_encode8<XF>(v, byte);
      if constexpr (XF == kMxFp4) *reinterpret_cast<uint32_t*>(lc + t * xrow + c / 2) = e[0];
      else *reinterpret_cast<u32x2*>(lc + t * xrow + c) = e;
      if ((lane & 3) == 0) ls[t * srow + c / kMxBlock] = (uint8_t)byte;
    }
    __syncthreads();
    for (int c0 = wave; c0 < chunks; c0 += U * kFewWaves) {
      load_group_w(c0 + U * kFewWaves, nw);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (c0 + u * kFewWaves < chunks) {
          Tokens t;
          load_x(lc, ls, c0 + u * kFewWaves, t);
          multiply(w[u], t);
        }
#pragma unroll
      for (int u = 0; u < U; ++u) w[u] = nw[u];
    }
  } else {
    const char* codes = reinterpret_cast<const char*>(xc);
    Tokens t[U], nt[U];
    auto load_group_x = [&](int c0, Tokens(&p)[U]) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (c0 + u * kFewWaves < chunks) load_x(codes, xs, c0 + u * kFewWaves, p[u]);
    };
    load_group_x(wave, t);
    for (int c0 = wave; c0 < chunks; c0 += U * kFewWaves) {
      load_group_w(c0 + U * kFewWaves, nw);
      load_group_x(c0 + U * kFewWaves, nt);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (c0 + u * kFewWaves < chunks) multiply(w[u], t[u]);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        w[u] = nw[u];
        t[u] = nt[u];
      }
    }
  }

  // sums of the waves: (token, feature) tiles of 16 x 16, added in wave order
  __syncthreads();
  float* red = reinterpret_cast<float*>(smem);
  *reinterpret_cast<f32x4*>(red + (wave * 16 + n16) * 16 + 4 * g) = acc;
  __syncthreads();
  if (threadIdx.x < 256) {
    const int i = threadIdx.x, token = i >> 4;
    const int64_t f = f0 + (i & 15);
    if (token >= tokens || f >= rows) return;
    float s = red[i];
#pragma unroll
    for (int v = 1; v < kFewWaves; ++v) s += red[v * 256 + i];
    if (bias) s += bias[f];
    store_value<OTYPE>(out, token * ldo + f, s);
  }
}

// ---- many tokens: bound by the matrix cores ----------------------------------------------------------------
//
// 2 x WT waves own a tile of 64 FA features x 32 TB WT tokens; a wave 32 FA x 32 TB of it, in 32x32x64
// products.  128 values of the contraction at a time go from memory straight into LDS, into a ring of stages: one is
// read while the ones after it fill.  A row's 16-byte pieces are permuted by bits of its row number, so that the reads
// of a fragment (one piece of 16 neighbouring rows at a time) fall into all 64 banks.  The scales of 512 values come
// at once, 16 bytes a row: a die's L2 serves 16 requests of up to 64 bytes a clock, and 4 bytes of each row with
// every stage took as many requests as the codes (tiles of 256 x 128 ran at 13 requests a clock, 2.7 PFLOP/s).  In LDS
// the scale words of a fragment lie 16 bytes apart and do meet in their banks: 36 k of a CU's 97 k LDS cycles.
//
// 4096 tokens of mxfp4, 4096 -> 14336: 142 to 163 us on four cards, 2.9 to 3.4 PFLOP/s; 14336 -> 4096, one round of 256
// tiles: 3.5 to 3.9.  The clock follows the power: on zeros the latter runs at 4.9 PFLOP/s, about what the
// instruction reaches with its operands from LDS and a barrier for every 128 values; with operands in
// registers it reaches 6.2 to 7.1 PFLOP/s on random data and 8.4 on zeros.  mxfp8, whose instruction reaches 3.7 PFLOP/s:
// 222 and 185 us, 2.2 and 2.6 PFLOP/s.
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef __attribute__((address_space(3))) void* lds_ptr;
typedef __attribute__((address_space(1))) const void* glb_ptr;

template <int BYTES>
__device__ __forceinline__ void to_lds(const void* from, char* to) {
  if constexpr (BYTES == 16) __builtin_amdgcn_global_load_lds((glb_ptr)from, (lds_ptr)to, 16, 0, 0);
  else __builtin_amdgcn_global_load_lds((glb_ptr)from, (lds_ptr)to, 4, 0, 0);
}

template <int XF, int FA, int TB, int WT>
struct Tile {
  static constexpr int kF = 64 * FA, kT = 32 * TB * WT, kWaves = 2 * WT;
  static constexpr int kXRow = XF == kMxFp4 ? 64 : 128, kXPieces = kXRow / 16;
  static constexpr int kX = kF * 64, kStage = kX + kT * kXRow;
  static constexpr int kSX = kF * 16, kScales = kSX + kT * 16;  // of 512 values, two buffers
  // the tiles of eight waves have a CU to themselves; of the others two work-groups share its LDS
  static constexpr int kStages = (WT == 4 ? 1 : 2) * (4 * kStage + 2 * kScales) <= 160 * 1024 ? 4 : 3;
  static constexpr int kS0 = kStages * kStage, kLds = kS0 + 2 * kScales;
  // 16-byte loads of a wave for a stage
  static constexpr int kWLoads = kF / 16 / kWaves, kXLoads = kT * kXPieces / 64 / kWaves, kLoads = kWLoads + kXLoads;
};

// All but the last N loads of this wave have arrived, and all of its reads of LDS.  (The builtin: the compiler then
// knows, and adds no wait of its own.)
template <int N>
__device__ __forceinline__ void wait_loads() {
  static_assert(N < 64, "six bits");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | ((N >> 4) << 14));
}

template <int XF, int S>
__device__ __forceinline__ f32x16 mfma32(u32x4 w, uint32_t ws, u32x4 x0, u32x4 x1, uint32_t xs, f32x16 c) {
  const i32x8 a = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
  const i32x8 b = {(int)x0[0], (int)x0[1], (int)x0[2], (int)x0[3], (int)x1[0], (int)x1[1], (int)x1[2], (int)x1[3]};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 4, XF == kMxFp4 ? 4 : 0, S, (int)ws, S, (int)xs);
}

struct TileArgs {
  const uint8_t *xc, *xs;
  int64_t tokens, padded;
  const uint8_t *wc, *wsc;
  int64_t rows;
  const float* bias;
  char* out;
  int64_t ldo;
  int ftiles, ttiles, per_xcd, whole, run;  // `whole`: of a die's tiles, the others are cut in two
};

template <int XF, int FA, int TB, int WT, int OTYPE>
__device__ __forceinline__ void tile_body(const TileArgs& args, int64_t t0, int64_t f0, char* smem) {
  typedef Tile<XF, FA, TB, WT> L;
  const uint8_t *xc = args.xc, *xs = args.xs, *wc = args.wc, *wsc = args.wsc;
  const int64_t tokens = args.tokens, padded = args.padded, rows = args.rows, ldo = args.ldo;
  const float* bias = args.bias;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r32 = lane & 31, h = lane >> 5;
  const int wf = (wave & 1) * 32 * FA, wt = (wave >> 1) * 32 * TB;
  const int64_t wrow = padded / 2, xrow = mx_code_bytes(padded, XF), srow = padded / kMxBlock;
  const int all_steps = (int)(padded / 128);
  // this work-group's run of the contraction (whole periods of scales); each run has an output of its own
  const int begin = (int)blockIdx.y * args.run, steps = min(begin + args.run, all_steps);
  char* out = args.out + (int64_t)blockIdx.y * tokens * ldo * (OTYPE == kMxF32 ? 4 : 2);

  // this lane's pieces, from the tile's first rows
  uint32_t ow[L::kWLoads], ox[L::kXLoads];
#pragma unroll
  for (int u = 0; u < L::kWLoads; ++u) {
    const int r = (wave * L::kWLoads + u) * 16 + (lane >> 2);
    ow[u] = (uint32_t)min((int64_t)r, rows - 1 - f0) * (uint32_t)wrow + (((lane & 3) ^ ((r >> 2) & 3)) * 16);
  }
#pragma unroll
  for (int u = 0; u < L::kXLoads; ++u) {
    const int r = (wave * L::kXLoads + u) * (64 / L::kXPieces) + lane / L::kXPieces;
    const int piece = (lane & (L::kXPieces - 1)) ^ (XF == kMxFp4 ? (r >> 2) & 3 : (r >> 1) & 7);
    ox[u] = (uint32_t)min((int64_t)r, tokens - 1 - t0) * (uint32_t)xrow + piece * 16;
  }
  const uint8_t *gw = wc + f0 * wrow, *gx = xc + t0 * xrow;
  // Scales of 512 values.  The last 16 bytes of a row that has an odd number of 8s reach into the next row; the last
  // row's are taken 8 bytes early.
  auto load_scales = [&](int period, char* to) {
#pragma unroll
    for (int q = 0; q < (FA + L::kT / 64 + L::kWaves - 1) / L::kWaves; ++q) {
      const int u = wave + L::kWaves * q;  // 64 rows
      if (u < FA) {
        const int64_t at = min(f0 + 64 * u + lane, rows - 1) * srow + period * 16;
        to_lds<16>(wsc + min(at, rows * srow - 16), to + u * 1024);
      } else if (u < FA + L::kT / 64) {
        const int64_t at = min(t0 + 64 * (u - FA) + lane, tokens - 1) * srow + period * 16;
        to_lds<16>(xs + min(at, tokens * srow - 16), to + u * 1024);
      }
    }
  };
  auto load_stage = [&](int k, char* stage) {
    if (k % 4 == 0) load_scales(k / 4, smem + L::kS0 + (k / 4 & 1) * L::kScales);
    const uint8_t* w = gw + (int64_t)k * 64;
    const uint8_t* x = gx + (int64_t)k * L::kXRow;
#pragma unroll
    for (int u = 0; u < L::kWLoads; ++u) to_lds<16>(w + ow[u], stage + (wave * L::kWLoads + u) * 1024);
#pragma unroll
    for (int u = 0; u < L::kXLoads; ++u) to_lds<16>(x + ox[u], stage + L::kX + (wave * L::kXLoads + u) * 1024);
  };

  f32x16 acc[FA][TB];
#pragma unroll
  for (int a = 0; a < FA; ++a)
#pragma unroll
    for (int b = 0; b < TB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[a][b][i] = 0.f;

  // where this lane's fragments lie in a stage: what is constant in a piece's number is applied last
  const int w_from = (wf + r32) * 64 + (((2 * h) ^ ((r32 >> 2) & 3)) * 16);
  const int x_from = XF == kMxFp4 ? L::kX + (wt + r32) * 64 + (((2 * h) ^ ((r32 >> 2) & 3)) * 16)
                                  : L::kX + (wt + r32) * 128 + ((h ^ ((r32 >> 1) & 7)) * 16);
  struct Frags {
    u32x4 w[FA], x0[TB], x1[TB];
  };
  struct Scales {
    uint32_t w[FA], x[TB];  // blocks 2 h and 2 h + 1 of the row in the low half
  };
  auto read = [&](const char* stage, int s, Frags& f) {
#pragma unroll
    for (int b = 0; b < TB; ++b) {
      if constexpr (XF == kMxFp4) {
        f.x0[b] = *reinterpret_cast<const u32x4*>(stage + (x_from ^ (16 * s)) + b * 2048);
        f.x1[b] = u32x4{0u, 0u, 0u, 0u};
      } else {
        // an 8-bit operand lane holds half h of blocks s and s + 2
        f.x0[b] = *reinterpret_cast<const u32x4*>(stage + (x_from ^ (32 * s)) + b * 4096);
        f.x1[b] = *reinterpret_cast<const u32x4*>(stage + (x_from ^ (32 * s + 64)) + b * 4096);
      }
    }
#pragma unroll
    for (int a = 0; a < FA; ++a) f.w[a] = *reinterpret_cast<const u32x4*>(stage + (w_from ^ (16 * s)) + a * 2048);
  };
  auto read_scales = [&](int k, Scales& s) {
    const char* from = smem + L::kS0 + (k / 4 & 1) * L::kScales + (k & 3) * 4;
#pragma unroll
    for (int a = 0; a < FA; ++a) s.w[a] = *reinterpret_cast<const uint32_t*>(from + (wf + 32 * a + r32) * 16);
#pragma unroll
    for (int b = 0; b < TB; ++b) s.x[b] = *reinterpret_cast<const uint32_t*>(from + L::kSX + (wt + 32 * b + r32) * 16);
    if ((k & ~3) + 4 > all_steps) {  // the last row's scales of a half period lie 8 bytes on
#pragma unroll
      for (int a = 0; a < FA; ++a)
        if (f0 + wf + 32 * a + r32 >= rows - 1)
          s.w[a] = *reinterpret_cast<const uint32_t*>(from + (wf + 32 * a + r32) * 16 + 8);
#pragma unroll
      for (int b = 0; b < TB; ++b)
        if (t0 + wt + 32 * b + r32 >= tokens - 1)
          s.x[b] = *reinterpret_cast<const uint32_t*>(from + L::kSX + (wt + 32 * b + r32) * 16 + 8);
    }
#pragma unroll
    for (int a = 0; a < FA; ++a) s.w[a] >>= 16 * h;
#pragma unroll
    for (int b = 0; b < TB; ++b) s.x[b] >>= 16 * h;
  };
  auto multiply = [&](const Frags& f, const Scales& c, auto s_const) {
    constexpr int s = decltype(s_const)::value;
#pragma unroll
    for (int a = 0; a < FA; ++a)
#pragma unroll
      for (int b = 0; b < TB; ++b)
        acc[a][b] = mfma32<XF, s>(f.w[a], c.w[a], f.x0[b], f.x1[b], c.x[b], acc[a][b]);
    // they stay on this side of the barrier: sunk behind it they would run one work-group-wide phase after another
#pragma unroll
    for (int a = 0; a < FA; ++a)
#pragma unroll
      for (int b = 0; b < TB; ++b) asm volatile("" : "+v"(acc[a][b]));
  };

  // A stage's 128 values are two products.  Fragments are read one product ahead, across the barrier: in the middle of
  // stage k everyone's reads of it are done, k + 1 has arrived, and stage k's place takes the one kStages on.
  constexpr int kStages = L::kStages;
#pragma unroll
  for (int k = 0; k < kStages; ++k)
    if (begin + k < steps) load_stage(begin + k, smem + k * L::kStage);
  if (begin + kStages <= steps) wait_loads<(kStages - 1) * L::kLoads>();
  else wait_loads<0>();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  Frags first, second;
  Scales scale, next_scale;
  read_scales(begin, scale);
  read(smem, 0, first);
  int now = 0;
  for (int k = begin; k + 1 < steps; ++k) {
    char* stage = smem + now * L::kStage;
    now = now + 1 == kStages ? 0 : now + 1;
    read(stage, 1, second);
    multiply(first, scale, std::integral_constant<int, 0>{});
    if (k + kStages <= steps) wait_loads<(kStages - 2) * L::kLoads>();
    else wait_loads<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (k + kStages < steps) load_stage(k + kStages, stage);
    read_scales(k + 1, next_scale);
    read(smem + now * L::kStage, 0, first);
    multiply(second, scale, std::integral_constant<int, 1>{});
    scale = next_scale;
  }
  read(smem + now * L::kStage, 1, second);
  multiply(first, scale, std::integral_constant<int, 0>{});
  multiply(second, scale, std::integral_constant<int, 1>{});

  // A lane holds 4 features in a row of one token, its partner 32 lanes on the next 4: they trade, so that each has 8 in
  // a row.  Through LDS (a part of each wave's own, once everyone is done with the stages) a wave then stores 32 FA
  // features of a token side by side: on 117 MB 32-byte stores straight from the registers took 30 us more, and stores
  // that stay in L2 17 us more, where they drive out the codes that the next tiles share.
  constexpr int kSize = OTYPE == kMxF32 ? 4 : 2, kWords = OTYPE == kMxF32 ? 4 : 2;
  constexpr int kRow = 32 * FA * kSize + 16;          // 16 rows fall into all banks
  constexpr int kLanes = 2 * FA * kSize, kPer = 16 / kSize;  // lanes that store a row, features of each
  static_assert(L::kWaves * 32 * kRow <= L::kLds, "fits the stages");
  wait_loads<0>();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  char* mine = smem + wave * 32 * kRow;
  const bool whole = t0 + L::kT <= tokens && f0 + L::kF <= rows;
#pragma unroll
  for (int b = 0; b < TB; ++b) {
#pragma unroll
    for (int a = 0; a < FA; ++a) {
      const int64_t fa = f0 + wf + 32 * a;
      if (bias) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int64_t f = fa + 8 * q + 4 * h;
          f32x4 v = {0.f, 0.f, 0.f, 0.f};
          if (f + 4 <= rows) {
            v = load_any<f32x4>(bias + f);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (f + i < rows) v[i] = bias[f + i];
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[a][b][4 * q + i] += v[i];
        }
      }
#pragma unroll
      for (int q = 0; q < 4; q += 2) {
        uint32_t lo[kWords], hi[kWords];  // this lane's 4 features of groups q and q + 1
        if constexpr (OTYPE == kMxF32) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            lo[i] = __float_as_uint(acc[a][b][4 * q + i]);
            hi[i] = __float_as_uint(acc[a][b][4 * q + 4 + i]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            lo[i] = pack_pair<OTYPE>(acc[a][b][4 * q + 2 * i], acc[a][b][4 * q + 2 * i + 1]);
            hi[i] = pack_pair<OTYPE>(acc[a][b][4 * q + 4 + 2 * i], acc[a][b][4 * q + 4 + 2 * i + 1]);
          }
        }
        uint32_t v[2 * kWords];
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
          const auto r = __builtin_amdgcn_permlane32_swap(lo[i], hi[i], false, false);
          v[i] = r[0];
          v[kWords + i] = r[1];
        }
        // the lower lanes have group q, the upper ones q + 1
        char* to = mine + r32 * kRow + (32 * a + 8 * (q + h)) * kSize;
#pragma unroll
        for (int i = 0; i < 2 * kWords; i += 4)
          *reinterpret_cast<u32x4*>(to + 4 * i) = u32x4{v[i], v[i + 1], v[i + 2], v[i + 3]};
      }
    }
    const int f = (lane % kLanes) * kPer;
    const int64_t left = rows - (f0 + wf + f);
#pragma unroll
    for (int r0 = 0; r0 < 32; r0 += 64 / kLanes) {
      const int r = r0 + lane / kLanes;
      const int64_t token = t0 + wt + 32 * b + r;
      const u32x4 v = *reinterpret_cast<const u32x4*>(mine + r * kRow + f * kSize);
      char* dst = out + (token * ldo + f0 + wf + f) * kSize;
      if (whole && FA == 4) {
        __builtin_nontemporal_store(v, reinterpret_cast<u32x4_any*>(dst));  // 256 bytes a row: nothing to join in L2
      } else if (whole || (token < tokens && left >= kPer)) {
        store_any<u32x4>(dst, v);
      } else if (token < tokens) {
#pragma unroll
        for (int i = 0; i < kPer; ++i)
          if (i < left) {
            if constexpr (kSize == 4) reinterpret_cast<uint32_t*>(dst)[i] = v[i];
            else reinterpret_cast<uint16_t*>(dst)[i] = (uint16_t)(v[i / 2] >> (16 * (i % 2)));
          }
      }
    }
  }
}

// Consecutive blocks go to the 8 dies in turn: each die takes a run of tiles, four token tiles deep, so that its L2
// holds the rows that its tiles share.  The largest tiles take a CU each; where half of the CUs or more would idle in
// the last round, its tiles are cut into halves of their features (codes given, 4096 tokens: 4096 -> 4608 69 -> 60 us,
// 2048 -> 5000 47 -> 41, 4096 -> 14336 167 -> 163).  Whole tiles taken one after another by a work-group a CU, the next
// one's first stages loaded ahead of the stores, changed nothing: the power rules.
template <int XF, int FA, int TB, int WT, int OTYPE>
__global__ __launch_bounds__(128 * WT, 2) void tile_kernel(TileArgs args) {
  extern __shared__ __align__(16) char smem[];
  typedef Tile<XF, FA, TB, WT> L;
  const int at = (int)(blockIdx.x / 8), cut = max(at - args.whole, 0);
  const int t = (int)(blockIdx.x % 8) * args.per_xcd + at - (cut + 1) / 2;
  if (t >= args.ftiles * args.ttiles) return;
  const int group = t / (4 * args.ftiles), deep = min(4, args.ttiles - 4 * group), in = t - group * 4 * args.ftiles;
  const int64_t t0 = (int64_t)(4 * group + in % deep) * L::kT, f0 = (int64_t)(in / deep) * L::kF;
  if constexpr (FA == 4) {
    if (at >= args.whole) {
      const int64_t half = f0 + (cut & 1) * (L::kF / 2);
      if (half < args.rows) tile_body<XF, FA / 2, TB, WT, OTYPE>(args, t0, half, smem);
      return;
    }
  }
  tile_body<XF, FA, TB, WT, OTYPE>(args, t0, f0, smem);
}

// Sums of the runs, in their order.
template <int OTYPE>
__global__ __launch_bounds__(256) void join_kernel(const float* __restrict__ part, int runs, int64_t tokens,
                                                   int64_t rows, const float* __restrict__ bias,
                                                   void* __restrict__ out, int64_t ldo) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= tokens * rows) return;
  float s = sum_splits(part, runs, tokens * rows, i);
  const int64_t t = i / rows, f = i - t * rows;
  if (bias) s += bias[f];
  store_value<OTYPE>(out, t * ldo + f, s);
}

// ---- choice and launch ------------------------------------------------------------------------------------

constexpr int kFewTokens = 16;  // above, tiles: at 8 tokens those take 1 to 2 us more, at 24 they take less
// Up to here every work-group quantises the tokens itself, in so much LDS: saves a launch and the codes' way
// through memory (two tokens 4096 -> 14336: 15.8 -> 10.7 us a call; 8 tokens in 8 work-group waves would lose 3 us).
constexpr int kFusedTokens = 4;
constexpr int64_t kFusedBytes = 64 * 1024;

constexpr int kCus = 256;

struct Args {
  const void* x;
  int xtype;
  int64_t ldx;
  const uint8_t *xc, *xs;
  int64_t tokens, cols, padded;
  const uint8_t *wc, *ws;
  int64_t rows;
  const float* bias;
  void* out;
  int64_t ldo;
  float* part;  // of split contractions
  hipStream_t stream;
};

// The contraction of few tiles is split into runs of whole 512-value periods, eight stages at least, until every CU has a
// work-group: 64 tokens of mxfp8, 14336 -> 4096, 42 -> 18 us; twice as many runs take 1 to 4 us more.
struct Split {
  int runs, run;  // run: stages of 128 values
};

int64_t tiles_of(int64_t rows, int64_t tokens, int f, int t) { return mpq_cdiv(rows, f) * mpq_cdiv(tokens, t); }

Split split_of(int64_t rows, int64_t tokens, int64_t padded) {
  const int steps = (int)(padded / 128);
  const int64_t tiles = tiles_of(rows, tokens, 64, 64);
  int64_t runs = std::min<int64_t>({256 / std::max<int64_t>(tiles, 1), steps / 8, kMaxSplits});
  if (tokens <= kFewTokens || runs < 2) return {1, steps};
  const int run = (int)(mpq_cdiv(mpq_cdiv(steps, runs), 4) * 4);
  return {(int)mpq_cdiv(steps, run), run};
}

int64_t fused_bytes(int64_t tokens, int64_t padded, int xf) {
  return tokens * (mx_code_bytes(padded, xf) + 16 + padded / kMxBlock);
}

bool fuses(int64_t tokens, int64_t padded, int xf) {
  return tokens <= kFusedTokens && fused_bytes(tokens, padded, xf) <= kFusedBytes;
}

template <class K>
hipError_t allow_lds(K kernel, int bytes) {
  if (bytes <= 64 * 1024) return hipSuccess;
  return hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

template <int XF, bool FUSED, int XTYPE, int OTYPE>
hipError_t launch_few(const Args& a) {
  constexpr int red = kFewWaves * 256 * 4;
  const int lds = FUSED ? (int)std::max<int64_t>(red, fused_bytes(a.tokens, a.padded, XF)) : red;
  auto kernel = few_kernel<XF, FUSED, XTYPE, OTYPE>;
  if (hipError_t e = allow_lds(kernel, lds); e != hipSuccess) return e;
  constexpr int64_t most = kMxLaunch / (64 * kFewWaves) * 16;
  for (int64_t f = 0; f < a.rows; f += most) {
    const int64_t n = std::min(most, a.rows - f);
    hipLaunchKernelGGL(kernel, dim3((unsigned)mpq_cdiv(n, 16)), dim3(64 * kFewWaves), lds, a.stream,
                       static_cast<const char*>(a.x), a.ldx, a.xc, a.xs, (int)a.tokens, a.cols, a.padded,
                       a.wc + f * (a.padded / 2), a.ws + f * (a.padded / kMxBlock), n, a.bias ? a.bias + f : nullptr,
                       static_cast<char*>(a.out) + f * (OTYPE == kMxF32 ? 4 : 2), a.ldo);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <int XF, int FA, int TB, int WT, int OTYPE>
hipError_t launch_tile(const Args& a, Split split, void* out, int64_t ldo, const float* bias) {
  typedef Tile<XF, FA, TB, WT> L;
  auto kernel = tile_kernel<XF, FA, TB, WT, OTYPE>;
  if (hipError_t e = allow_lds(kernel, L::kLds); e != hipSuccess) return e;
  const int64_t ft = mpq_cdiv(a.rows, L::kF), tt = mpq_cdiv(a.tokens, L::kT), per = mpq_cdiv(ft * tt, 8);
  const int64_t left = FA == 4 ? per % (kCus / 8) : 0;
  const int64_t halves = left <= kCus / 16 ? left : 0;
  const TileArgs args = {a.xc, a.xs, a.tokens, a.padded, a.wc, a.ws, a.rows, bias, static_cast<char*>(out), ldo,
                         (int)ft, (int)tt, (int)per, (int)(per - halves), split.run};
  hipLaunchKernelGGL(kernel, dim3((unsigned)((per + halves) * 8), (unsigned)split.runs), dim3(64 * L::kWaves), L::kLds,
                     a.stream, args);
  return hipGetLastError();
}

template <int XF, int OTYPE>
hipError_t run_linear(const Args& a, bool fused) {
  if (fused) {
    if (a.xtype == kMxF32) return launch_few<XF, true, kMxF32, OTYPE>(a);
    if (a.xtype == kMxBf16) return launch_few<XF, true, kMxBf16, OTYPE>(a);
    return launch_few<XF, true, kMxF16, OTYPE>(a);
  }
  if (a.tokens <= kFewTokens) return launch_few<XF, false, kMxF32, OTYPE>(a);
  if (a.rows * a.padded < 16 * kMxBlock) {  // a single row of 8 scale bytes: tiles load 16
    Args part = a;
    for (int64_t t = 0; t < a.tokens; t += kFewTokens) {
      part.tokens = std::min<int64_t>(kFewTokens, a.tokens - t);
      part.xc = a.xc + t * mx_code_bytes(a.padded, XF);
      part.xs = a.xs + t * (a.padded / kMxBlock);
      part.out = static_cast<char*>(a.out) + t * a.ldo * (OTYPE == kMxF32 ? 4 : 2);
      if (hipError_t e = launch_few<XF, false, kMxF32, OTYPE>(part); e != hipSuccess) return e;
    }
    return hipSuccess;
  }
  const Split split = split_of(a.rows, a.tokens, a.padded);
  if (split.runs > 1) {
    if (hipError_t e = launch_tile<XF, 1, 1, 2, kMxF32>(a, split, a.part, a.rows, nullptr); e != hipSuccess) return e;
    const int64_t n = a.tokens * a.rows;
    hipLaunchKernelGGL(join_kernel<OTYPE>, dim3((unsigned)mpq_cdiv(n, 256)), dim3(256), 0, a.stream, a.part, split.runs,
                       a.tokens, a.rows, a.bias, a.out, a.ldo);
    return hipGetLastError();
  }
  // The largest tile that keeps most CUs at work (codes given, us).  256 x 256 of mxfp4 from 96 on, where up to 128 are
  // cut in two: 224 tiles (1000 tokens, 4096 -> 14336) 42 against 61 in 128 x 128, 96 (700, 4096 -> 8000) 24 and 27,
  // 64 (1000, 4096 -> 4096) 24 and 19.  Of mxfp8 from 192 on: 896 (4096, 4096 -> 14336) 222 and 243 in 256 x 128, 192
  // (2048, 4096 -> 6144) 55 and 55, 128 (1024, 4096 -> 8192) 35 and 33; 320 (4096, 2048 -> 5000) 53 and 51.
  if (tiles_of(a.rows, a.tokens, 256, 256) >= (XF == kMxFp4 ? 96 : 192))
    return launch_tile<XF, 4, 2, 4, OTYPE>(a, split, a.out, a.ldo, a.bias);
  // 128 tiles (1000, 4096 -> 4096): 23 and 24 in 128 x 128
  if constexpr (XF == kMxFp8)
    if (tiles_of(a.rows, a.tokens, 256, 128) >= 128)
      return launch_tile<XF, 4, 1, 4, OTYPE>(a, split, a.out, a.ldo, a.bias);
  // 192 tiles (300, 4096 -> 8192): 16 and 20 in 64 x 64; 128 (512, 4096 -> 4096): 16 and 15
  if (tiles_of(a.rows, a.tokens, 128, 128) >= 192)
    return launch_tile<XF, 2, 2, 2, OTYPE>(a, split, a.out, a.ldo, a.bias);
  return launch_tile<XF, 1, 1, 2, OTYPE>(a, split, a.out, a.ldo, a.bias);
}

// x's codes, their scales, the partial sums.
struct Layout {
  int64_t scales, part, bytes;
};

Layout layout_of(int64_t tokens, int64_t rows, int64_t padded, int xf) {
  Layout l;
  l.scales = tokens * mx_code_bytes(padded, xf);
  l.part = mpq_cdiv(l.scales + tokens * (padded / kMxBlock), 256) * 256;
  const Split s = split_of(rows, tokens, padded);
  l.bytes = l.part + (s.runs > 1 ? s.runs * tokens * rows * (int64_t)sizeof(float) : 0);
  return l;
}

}  // namespace
}  // namespace mpq

extern "C" int64_t mpq_mx_linear_workspace_size(int64_t tokens, int64_t cols, int64_t rows, int x_fmt) {
  using namespace mpq;
  if (tokens <= 0 || cols <= 0 || rows <= 0 || (x_fmt != kMxFp4 && x_fmt != kMxFp8)) return 0;
  const int64_t padded = mx_padded(cols);
  if (fuses(tokens, padded, x_fmt)) return 0;
  return layout_of(tokens, rows, padded, x_fmt).bytes;
}

extern "C" int mpq_mx_linear(const void* x, int dtype, int64_t ldx, const uint8_t* x_codes, const uint8_t* x_scales,
                             int x_fmt, int64_t tokens, int64_t cols, const uint8_t* w_codes, const uint8_t* w_scales,
                             int64_t rows, const float* bias, void* out, int out_dtype, int64_t ldo, void* workspace,
                             int64_t workspace_bytes, hipStream_t stream) {
  using namespace mpq;
  MPQ_CHECK_ARG(x_fmt == kMxFp4 || x_fmt == kMxFp8, "mpq_mx_linear: unknown format %d", x_fmt);
  MPQ_CHECK_ARG(dtype >= kMxF32 && dtype <= kMxF16 && out_dtype >= kMxF32 && out_dtype <= kMxF16,
                "mpq_mx_linear: unknown type %d / %d", dtype, out_dtype);
  MPQ_CHECK_ARG(tokens >= 0 && rows >= 0 && cols >= 1, "mpq_mx_linear: bad shape %lld x %lld x %lld",
                (long long)tokens, (long long)rows, (long long)cols);
  if (tokens == 0 || rows == 0) return kOk;
  const bool given = x_codes != nullptr;
  MPQ_CHECK_ARG(given ? x_scales != nullptr : (x != nullptr && ldx >= cols), "mpq_mx_linear: no tokens given");
  MPQ_CHECK_ARG(w_codes && w_scales && out && ldo >= rows, "mpq_mx_linear: null pointer or short output rows");
  // (the tiles of a launch of 512 threads each: more results than the card holds)
  MPQ_CHECK_ARG(cols <= (1 << 23) && tokens <= (1 << 30) && rows <= (1 << 30) &&
                    mpq_cdiv(tokens, 256) * mpq_cdiv(rows, 256) <= (1 << 23) - 256,
                "mpq_mx_linear: extent too large");
  const int64_t padded = mx_padded(cols);
  Args a = {x, dtype, ldx, x_codes, x_scales, tokens, cols, padded, w_codes, w_scales, rows, bias, out, ldo, nullptr,
            stream};
  const bool fused = !given && fuses(tokens, padded, x_fmt);
  const Layout l = layout_of(tokens, rows, padded, x_fmt);
  if (!fused && (!given || l.bytes > l.part)) {
    MPQ_CHECK_ARG(workspace && workspace_bytes >= l.bytes && reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
                  "mpq_mx_linear: workspace of %lld bytes, %lld needed (16-byte aligned)", (long long)workspace_bytes,
                  (long long)l.bytes);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    a.part = reinterpret_cast<float*>(ws + l.part);
    if (!given) {
      MPQ_HIP_TRY(mx_quantize_rows(x, dtype, tokens, cols, ldx, x_fmt, ws, ws + l.scales, stream));
      a.xc = ws;
      a.xs = ws + l.scales;
    }
  }
  hipError_t e;
#define MPQ_L(F)                                                          \
  (out_dtype == kMxF32 ? run_linear<F, kMxF32>(a, fused)                  \
                       : out_dtype == kMxBf16 ? run_linear<F, kMxBf16>(a, fused) : run_linear<F, kMxF16>(a, fused))
  e = x_fmt == kMxFp4 ? MPQ_L(kMxFp4) : MPQ_L(kMxFp8);
#undef MPQ_L
  MPQ_HIP_TRY(e);
  return kOk;
}
