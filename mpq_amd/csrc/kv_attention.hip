// Attention of new tokens over the quantised, paged key/value cache (gfx950).
//
//   o_r = sum_p softmax_p(scale q_r . k_p) v_p over the positions p that row r sees.
//
// Rows are (new token, query head) pairs; the query heads that share a key/value head are rows of one tile, so
// the cache is read once for all of them.  One pass over the keys with the running maximum and sum of the
// softmax, in fp32 and base 2.  Scores are formed transposed, S^T = K Q^T: a lane then holds several
// keys of one row, the row's statistics are per lane, and after exp2 the lane's values are, as they stand, its
// operand of O^T = V^T P^T: the order of the keys in that product is free, and V^T is loaded in the order in which
// S^T leaves them.  K and V become 16-bit operands (exact for what was written from that type), P is rounded to 16
// bits for the product while its sum is kept in fp32.  The maximum that p is taken against is moved only when a tile
// exceeds it by more than 2^8: the result does not depend on it, sums and products stay within range, and sums are
// rarely rescaled.
//
// Positions that a row does not see get -inf; a row that sees nothing is 0 (lse -inf).  Memory behind a sequence's
// end may hold anything: its scores are replaced and its values read as zeros.  A value block that stands for NaN
// (scale byte 255) poisons exactly the rows that see it.  NaN codes of mxfp8 under another scale byte, which the write
// kernel never stores, would reach every row of their tile; a search for them in each tile took 1 % of chunks over a long
// context and 12 % of whole prompts (8 of 2048: 465 -> 521 us), so caches must not hold any.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "kv_cache.h"

namespace mpq {
namespace {

struct AttnArgs {
  const char* q;
  int64_t q_ts, q_hs;
  int64_t total_q;
  int q_heads, group, batch, max_q;
  const int32_t* table;
  int64_t width;
  const int32_t *kv_lens, *q_starts;
  float scale2;  // scale * log2(e)
  int causal;
  int split_len, splits;
  char* out;
  float* lse;
  float *part_o, *part_ml;  // (row, split, D) unnormalised sums and (row, split, 2) maximum and sum
  KvCache c;
};

constexpr float kLn2 = 0.69314718055994531f;

template <int TYPE>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (TYPE == kMxBf16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(bits_as<bf16x8>(a), bits_as<bf16x8>(b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(bits_as<f16x8>(a), bits_as<f16x8>(b), c, 0, 0, 0);
}

template <int TYPE>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (TYPE == kMxBf16) return bits_as<uint32_t>(bf16x2{(__bf16)a, (__bf16)b});
  else return bits_as<uint32_t>(f16x2{(_Float16)a, (_Float16)b});
}

// Exchanges within the vector unit: the larger of a lane's and its partner's value, 32 (16) lanes on.
__device__ __forceinline__ float max32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

__device__ __forceinline__ float max16(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

__device__ __forceinline__ float group_sum(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

// A sequence as a work-group sees it; lengths from device memory are brought into range first.
struct Seq {
  int q0, q_len, kv_len;
  // (new token, query head) pairs of a key/value head
  __device__ int rows(const AttnArgs& a) const { return min(q_len, a.max_q) * a.group; }
  __device__ Seq(const AttnArgs& a, int b) {
    const int64_t s = min((int64_t)max(a.q_starts[b], 0), a.total_q);
    q0 = (int)s;
    q_len = (int)(min(max((int64_t)a.q_starts[b + 1], s), a.total_q) - s);
    kv_len = (int)min((int64_t)max(a.kv_lens[b], 0), a.width << a.c.shift);
  }
  __device__ int last_seen(const AttnArgs& a, int t) const { return a.causal ? kv_len - q_len + t : kv_len - 1; }
};

// Rows of this key/value head that no tile holds see nothing: tokens before the first sequence or behind the last one (a
// batch padded to a captured size has such) and those of a sequence behind max_q.  By one work-group of each
// sequence and head (`mine`).
template <int D>
__device__ __forceinline__ void clear_unheld(const AttnArgs& a, const Seq& seq, int head, int b, bool mine) {
  const auto clear = [&](int from, int to) {
    const int pieces = a.group * (D / 8);  // of 16 bytes; the query heads of a token lie side by side
    for (int t = from; t < to; ++t) {
      const int64_t at = (int64_t)t * a.q_heads + head * a.group;
      for (int i = threadIdx.x; i < pieces; i += blockDim.x)
        store_any<u32x4>(a.out + at * (D * 2) + (int64_t)i * 16, u32x4{0u, 0u, 0u, 0u});
      if (a.lse)
        for (int i = threadIdx.x; i < a.group; i += blockDim.x) a.lse[at + i] = -INFINITY;
    }
  };
  const int end = seq.q0 + seq.q_len;
  const int from = b == 0 ? 0 : seq.q0, to = b == a.batch - 1 ? (int)a.total_q : end, held = min(end, seq.q0 + a.max_q);
  if (__builtin_expect(mine & ((from != seq.q0) | (held != to)), 0)) {
    clear(from, seq.q0);
    clear(held, to);
  }
}

// The run of keys of a work-group.  Consecutive work-groups go to the 8 dies in turn: unrotated, 4 or 8 runs would give
// each die the same run of every sequence, and the later runs of short sequences are empty (64 sequences of 512 to
// 8192 positions: 95 -> 79 us).
__device__ __forceinline__ int split_of(const AttnArgs& a, int x, int head, int b) {
  return (int)((uint32_t)(x + head + b) % (uint32_t)a.splits);
}

// The sign of the scale goes into q, and a scale of 0 is q = 0: the maximum of the scores is that of the products.
struct QSign {
  float scale2;
  uint32_t flip, keep;
  __device__ QSign(const AttnArgs& a)
      : scale2(a.scale2 == 0.f ? 1.f : fabsf(a.scale2)),
        flip(a.scale2 < 0.f ? 0x80008000u : 0u),
        keep(a.scale2 == 0.f ? 0u : 0xffffffffu) {}
  __device__ u32x4 operator()(u32x4 q) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = (q[i] ^ flip) & keep;
    return q;
  }
};

// ---- 16 rows a wave ----------------------------------------------------------------------------------------
//
// For few rows: bound by the cache's bytes.  A work-group owns 16 rows of one key/value head and a run of keys; its
// waves take 32 keys at a time in turn, each with statistics of its own, joined in LDS at the end.  The codes go from
// memory straight into LDS, kAhead tiles of each wave ahead of the one it works on; a lane reads back what it
// fetched itself (16 bytes for its part of 16 keys, two in mxfp8), so LDS is a queue without bank conflicts and
// without barriers, and the bytes on their way take no registers.  64 sequences of 512 to 8192 positions, 32 query and
// 8 key/value heads of 128, mxfp4, 318 MB: 64 us, 4.9 TB/s, and 5 for the join; 32 key/value heads: 252 us, 5.0 TB/s.
constexpr int kWaves = 4;

// What a lane holds of a tile of two runs of 16 keys.
template <int TYPE, int FMT, int D>
struct KeyTile {
  static constexpr int kKBytes = D / 4 * MxTraits<FMT>::kOctet / 8;  // a lane's quarter of a key's codes
  static constexpr int kKWords = kKBytes / 4;
  static constexpr int kVd = D / 16;                                 // values of D a lane holds of each key
  static constexpr int kVWords = FMT == kMxFp4 ? 1 : kVd / 4;        // words of a key
  uint32_t k[2][kKWords], ks[2];
  uint32_t v[2][4][kVWords], vs[2];
};

// A wave's place for a tile's bytes.
template <int FMT, int D>
struct Queue {
  static constexpr int kKBytes = D / 4 * MxTraits<FMT>::kOctet / 8;
  static constexpr int kKSize = kKBytes < 16 ? 4 : 16, kKOps = kKBytes / kKSize;  // loads of 4 or 16 bytes
  static constexpr int kVOps = FMT == kMxFp4 ? 1 : 2;
  static constexpr int kV = 2 * kKOps * kKSize * 64, kKs = kV + 2 * kVOps * 1024, kVs = kKs + 512, kTile = kVs + 512;
  static constexpr int kOps = 2 * (kKOps + kVOps + 2);
  // many waves hide more than deep queues: four work-groups a CU where they fit (the batch below: 3 tiles ahead and two
  // work-groups 103 us, 2 and four 88; in mxfp8 with heads of 64 2 and three 96 us, 1 and four 85)
  static constexpr int kAhead = kWaves * 2 * kTile <= 40 * 1024 ? 2 : 1;
  static constexpr int kJoin = kWaves * 16 * (D + 4) * 4 + kWaves * 16 * 2 * 4;
  static constexpr int kBytes = kWaves * kAhead * kTile > kJoin ? kWaves * kAhead * kTile : kJoin;
};

typedef __attribute__((address_space(3))) void* lds_ptr;
typedef __attribute__((address_space(1))) const void* glb_ptr;

template <int BYTES>
__device__ __forceinline__ void to_lds(const void* from, char* to) {
  if constexpr (BYTES == 16) __builtin_amdgcn_global_load_lds((glb_ptr)from, (lds_ptr)to, 16, 0, 0);
  else __builtin_amdgcn_global_load_lds((glb_ptr)from, (lds_ptr)to, 4, 0, 0);
}

// All but the last N loads of this wave have arrived (the builtin: the compiler counts along).
template <int N>
__device__ __forceinline__ void wait_loads() {
  static_assert(N < 64, "six bits");
  __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (15 << 8) | ((N >> 4) << 14));
  asm volatile("" ::: "memory");
}

template <int TYPE, int FMT, int D>
__global__ __launch_bounds__(64 * kWaves, 2) void rows16_kernel(AttnArgs a) {
  typedef KvLayout<FMT, D> L;
  typedef KeyTile<TYPE, FMT, D> T;
  typedef Queue<FMT, D> Q;
  constexpr int kJ = D / 32;  // products of S^T
  constexpr int kVd = T::kVd;
  extern __shared__ __align__(16) char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n16 = lane & 15, g = lane >> 4;
  const int tile = blockIdx.x / a.splits, head = blockIdx.y, b = blockIdx.z;
  const int split = split_of(a, blockIdx.x % a.splits, head, b);
  const Seq seq(a, b);
  clear_unheld<D>(a, seq, head, b, blockIdx.x == 0 && a.splits == 1);
  const int rows = seq.rows(a);
  if (tile * 16 >= rows) return;
  const int r = tile * 16 + n16;
  const bool real = r < rows;
  const int t = real ? r / a.group : 0;
  const int qh = head * a.group + (real ? r - t * a.group : 0);
  const int lim = real ? seq.last_seen(a, t) : -1;
  const int end_seen = seq.last_seen(a, (min(tile * 16 + 15, rows - 1)) / a.group) + 1;
  const int begin = (int)min((int64_t)split * a.split_len, (int64_t)0x7fffffff - 64);
  if (a.splits > 1 && begin >= end_seen) return;  // the join does not look at this run
  // the last run takes what is left: a sequence may be longer than the caller's estimate
  const int end = split + 1 < a.splits ? (int)min((int64_t)begin + a.split_len, (int64_t)end_seen) : end_seen;
  const int all_seen = min(seq.last_seen(a, tile * 16 / a.group) + 1, end);  // every row sees the positions below

  // Pages of a tile's two runs of keys, -1 for none; looked up on the scalar unit a tile ahead of the codes.
  constexpr int kStep = 32 * kWaves, kAhead = Q::kAhead;
  const __attribute__((address_space(4))) int32_t* table =
      (const __attribute__((address_space(4))) int32_t*)(a.table + b * a.width);
  int page[2];
  auto look = [&](int pos) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      page[s] = -1;
      if (pos + 16 * s < end) page[s] = table[(pos + 16 * s) >> a.c.shift];
    }
  };
  // Brings a tile; without a page the bytes are those of the first one, and the two bits say so.
  char* const mine = lds + wave * (kAhead * Q::kTile);
  auto bring = [&](int pos, char* to) {
    uint32_t there = 0;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const bool ok = page[s] >= 0 && page[s] < a.c.pages;
      there |= ok ? 1u << s : 0u;
      const int64_t row = L::row0(a.c, ok ? page[s] : 0, head) + ((pos + 16 * s) & (a.c.page - 1));
      const uint8_t* kp = a.c.kc + (row + n16) * L::kRow + g * T::kKBytes;
#pragma unroll
      for (int i = 0; i < Q::kKOps; ++i)
        to_lds<Q::kKSize>(kp + i * Q::kKSize, to + (s * Q::kKOps + i) * (64 * Q::kKSize));
      const uint8_t* vp = a.c.vc + L::v_code(row + 4 * g, n16 * kVd / 8);
#pragma unroll
      for (int i = 0; i < Q::kVOps; ++i) to_lds<16>(vp + 16 * i, to + Q::kV + (s * Q::kVOps + i) * 1024);
      to_lds<4>(a.c.ks + (((row + n16) * L::kScales) & ~(int64_t)3), to + Q::kKs + s * 256);
      to_lds<4>(a.c.vs + L::v_scale(row + 4 * g, n16 * kVd / kMxBlock), to + Q::kVs + s * 256);
    }
    return there;
  };
  auto take = [&](const char* from, T& x) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int i = 0; i < Q::kKOps; ++i) {
        const char* p = from + (s * Q::kKOps + i) * (64 * Q::kKSize) + lane * Q::kKSize;
        if constexpr (Q::kKSize == 16) {
          const u32x4 w = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
          for (int j = 0; j < 4; ++j) x.k[s][4 * i + j] = w[j];
        } else {
          x.k[s][i] = *reinterpret_cast<const uint32_t*>(p);
        }
      }
      const uint32_t ks = *reinterpret_cast<const uint32_t*>(from + Q::kKs + s * 256 + lane * 4);
      x.ks[s] = (ks >> (8 * (((n16 * L::kScales) & 3) + g * (D / 4) / kMxBlock))) & 255u;
      x.vs[s] = *reinterpret_cast<const uint32_t*>(from + Q::kVs + s * 256 + lane * 4);
      const u32x4 w0 = *reinterpret_cast<const u32x4*>(from + Q::kV + s * Q::kVOps * 1024 + lane * 16);
      if constexpr (FMT == kMxFp4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x.v[s][i][0] = D == 128 ? w0[i] : w0[i] >> (16 * (n16 & 1));
      } else {
        const u32x4 w1 = *reinterpret_cast<const u32x4*>(from + Q::kV + (s * Q::kVOps + 1) * 1024 + lane * 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t lo = i < 2 ? w0[2 * i] : w1[2 * i - 4], hi = i < 2 ? w0[2 * i + 1] : w1[2 * i - 3];
          if constexpr (D == 128) {
            x.v[s][i][0] = lo;
            x.v[s][i][T::kVWords - 1] = hi;
          } else {
            x.v[s][i][0] = n16 & 1 ? hi : lo;
          }
        }
      }
    }
  };

  int pos = begin + 32 * wave;
  look(pos);
  const QSign sign(a);
  const float scale2 = sign.scale2;
  u32x4 q[kJ];
#pragma unroll
  for (int j = 0; j < kJ; ++j) {
    q[j] = u32x4{0u, 0u, 0u, 0u};
    if (real) q[j] = sign(load_any<u32x4>(a.q + ((seq.q0 + t) * a.q_ts + qh * a.q_hs + g * (D / 4) + 8 * j) * 2));
  }

  uint32_t queue = 0;  // two bits a tile, the next one lowest
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    if (pos + i * kStep < end) {
      queue |= bring(pos + i * kStep, mine + i * Q::kTile) << (2 * i);
      look(pos + (i + 1) * kStep);
    }

  f32x4 o[kVd];
#pragma unroll
  for (int j = 0; j < kVd; ++j) o[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;

  // `all`: every row sees all of these keys
  auto compute = [&](int pos, T& x, uint32_t there, auto all) {
    constexpr bool kAll = decltype(all)::value;
    f32x4 s[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      s[u] = f32x4{0.f, 0.f, 0.f, 0.f};
      const float scale = mx_scale(x.ks[u]);
#pragma unroll
      for (int j = 0; j < kJ; ++j) {
        u32x2 w = {0u, 0u};
        if constexpr (FMT == kMxFp4) w[0] = x.k[u][j];
        else w = u32x2{x.k[u][2 * j], x.k[u][2 * j + 1]};
        s[u] = mfma16<TYPE>(mx_decode8<FMT, TYPE>(w, scale), q[j], s[u]);
      }
    }
    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (!kAll) {
          const bool seen = (there >> u & 1u) && pos + 16 * u + 4 * g + i <= lim;
          s[u][i] = seen ? s[u][i] : -INFINITY;
        }
        top = fmaxf(top, s[u][i]);
      }
    top = max16(max32(top)) * scale2;
    if (__any(top > m + 8.f)) {
      const float to = top > m + 8.f ? top : m;
      const float alpha = to == m ? 1.f : exp2f(m - to);
      m = to;
      l *= alpha;
#pragma unroll
      for (int j = 0; j < kVd; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[j][i] *= alpha;
    }
    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[u][i] = __builtin_amdgcn_exp2f(fmaf(s[u][i], scale2, -base));
        l += s[u][i];
      }
    u32x4 p;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      p[2 * u] = pack2<TYPE>(s[u][0], s[u][1]);
      p[2 * u + 1] = pack2<TYPE>(s[u][2], s[u][3]);
    }

    // scales of this lane's keys: zeros behind the end, and zeros of a finite scale for NaN blocks (byte 255: the byte of
    // ~vs is 0; in mxfp8 their codes may be NaN under every scale)
    uint32_t vs[2] = {x.vs[0], x.vs[1]};
    if constexpr (!kAll) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int left = there >> u & 1u ? seq.kv_len - (pos + 16 * u + 4 * g) : 0;  // keys of the group that there are
        vs[u] = left >= 4 ? vs[u] : left <= 0 ? 0u : vs[u] & ((1u << (8 * left)) - 1u);
      }
    }
    const uint32_t full0 = (~vs[0] - 0x01010101u) & vs[0] & 0x80808080u;
    const uint32_t full1 = (~vs[1] - 0x01010101u) & vs[1] & 0x80808080u;
    if (__any((full0 | full1) != 0u)) {
      uint32_t nan = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t at = 0xffu << (8 * (e & 3));
        if ((vs[e >> 2] & at) == at) {
          nan |= 1u << e;
          vs[e >> 2] &= ~at;
          if constexpr (FMT == kMxFp8)
#pragma unroll
            for (int i = 0; i < T::kVWords; ++i) x.v[e >> 2][e & 3][i] = 0u;
        }
      }
      float poison = 0.f;
      const int block = g * (D / 4) / kMxBlock;  // of the sums that this lane holds
#pragma unroll 1
      for (int sg = 0; sg < 4; ++sg) {
        const uint32_t f = (uint32_t)__shfl((int)nan, sg * 16 + block * (kMxBlock / kVd), 64);
#pragma unroll 1
        for (int e = 0; e < 8; ++e)
          if ((f >> e & 1u) && pos + 16 * (e >> 2) + 4 * sg + (e & 3) <= lim) poison = NAN;
      }
#pragma unroll
      for (int j = 0; j < kVd; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[j][i] += poison;
    }
    float vscale[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) vscale[e] = mx_scale((vs[e >> 2] >> (8 * (e & 3))) & 255u);
    const auto pair = [&](auto p_const) {  // values 2 P and 2 P + 1 of each of the eight keys
      constexpr int P = decltype(p_const)::value;
      uint32_t c[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        u32x2 w = {x.v[e >> 2][e & 3][0], x.v[e >> 2][e & 3][T::kVWords - 1]};
        if constexpr (!kAll) {
          const bool drop = !(there >> (e >> 2) & 1u) || pos + 16 * (e >> 2) + 4 * g + (e & 3) >= seq.kv_len;
          const uint32_t keep = drop ? 0u : 0xffffffffu;
          w &= keep;
        }
        c[e] = mx_decode_pair<FMT, TYPE, P>(w, vscale[e]);
      }
      u32x4 lo, hi;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        lo[e] = __builtin_amdgcn_perm(c[2 * e + 1], c[2 * e], 0x05040100u);
        hi[e] = __builtin_amdgcn_perm(c[2 * e + 1], c[2 * e], 0x07060302u);
      }
      o[2 * P] = mfma16<TYPE>(lo, p, o[2 * P]);
      o[2 * P + 1] = mfma16<TYPE>(hi, p, o[2 * P + 1]);
    };
    pair(std::integral_constant<int, 0>{});
    pair(std::integral_constant<int, 1>{});
    if constexpr (kVd == 8) {
      pair(std::integral_constant<int, 2>{});
      pair(std::integral_constant<int, 3>{});
    }
  };

  int slot = 0;
  for (; pos < end; pos += kStep) {
    if (pos + (kAhead - 1) * kStep < end) wait_loads<(kAhead - 1) * Q::kOps>();
    else wait_loads<0>();
    char* at = mine + slot * Q::kTile;
    T x;
    take(at, x);
    const uint32_t there = queue & 3u;
    queue >>= 2;
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the tile is in registers, its place is free
    asm volatile("" ::: "memory");
    if (pos + kAhead * kStep < end) {
      queue |= bring(pos + kAhead * kStep, at) << (2 * (kAhead - 1));
      look(pos + (kAhead + 1) * kStep);
    }
    if (pos + 32 <= all_seen && there == 3u) compute(pos, x, there, std::true_type{});
    else compute(pos, x, there, std::false_type{});
    slot = slot + 1 == kAhead ? 0 : slot + 1;
  }

  // join the waves: lane (n16, g) holds values kVd (4 g + i) + j of row n16
  l = group_sum(l);
  __syncthreads();  // everyone is done with the queues
  float(*red_o)[16][D + 4] = reinterpret_cast<float(*)[16][D + 4]>(lds);
  float(*red_ml)[16][2] = reinterpret_cast<float(*)[16][2]>(lds + kWaves * 16 * (D + 4) * 4);
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < kVd; j += 4)
      *reinterpret_cast<f32x4*>(&red_o[wave][n16][kVd * (4 * g + i) + j]) =
          f32x4{o[j][i], o[j + 1][i], o[j + 2][i], o[j + 3][i]};
  if (g == 0) {
    red_ml[wave][n16][0] = m;
    red_ml[wave][n16][1] = l;
  }
  __syncthreads();
  const int row = threadIdx.x >> 4, r2 = tile * 16 + row;
  if (r2 >= rows) return;
  float top = -INFINITY;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) top = fmaxf(top, red_ml[w][row][0]);
  const float base = top == -INFINITY ? 0.f : top;
  float f[kWaves], sum = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    f[w] = exp2f(red_ml[w][row][0] - base);
    sum += f[w] * red_ml[w][row][1];
  }
  const int t2 = r2 / a.group;
  const int64_t at = (int64_t)(seq.q0 + t2) * a.q_heads + head * a.group + (r2 - t2 * a.group);
  const int d0 = (threadIdx.x & 15) * (D / 16);
  float v[D / 16];
#pragma unroll
  for (int d = 0; d < D / 16; ++d) {
    v[d] = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) v[d] += f[w] * red_o[w][row][d0 + d];
  }
  if (a.splits > 1) {
    float* po = a.part_o + (at * a.splits + split) * D + d0;
#pragma unroll
    for (int d = 0; d < D / 16; d += 4) *reinterpret_cast<f32x4*>(po + d) = f32x4{v[d], v[d + 1], v[d + 2], v[d + 3]};
    if ((threadIdx.x & 15) == 0) {
      a.part_ml[(at * a.splits + split) * 2] = top;
      a.part_ml[(at * a.splits + split) * 2 + 1] = sum;
    }
    return;
  }
  const float inv = sum == 0.f ? 1.f : 1.f / sum;
  char* dst = a.out + (at * D + d0) * 2;
#pragma unroll
  for (int d = 0; d < D / 16; d += 2)
    *reinterpret_cast<uint32_t*>(dst + d * 2) = pack2<TYPE>(v[d] * inv, v[d + 1] * inv);
  if (a.lse && (threadIdx.x & 15) == 0) a.lse[at] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
}

// ---- 32 rows a wave, 128 or 256 a work-group --------------------------------------------------------------------
//
// For chunks of prompts: bound by the matrix cores.  Each wave of the work-group turns 16 keys of a tile into 16-bit
// operands for all of them, in LDS: K as rows of D, V transposed as rows of 64 keys in the order of S^T's lanes, so
// that one 16-byte read is one operand of a 32x32x16 product.  16-byte pieces are permuted by the low bits of
// their row, which keeps these reads free of bank conflicts.  While a tile is worked on, the next one goes into the
// other buffer and the codes of the one after it are on their way: one barrier a tile.
//
// Two chunks of 2048 over 12000 to 16384 positions, 32 query and 8 key/value heads of 128, mxfp8: 990 to 1050 us on three
// cards, 940 to 1000 TFLOP/s, where one large bf16 product reaches 1223.  The matrix cores are busy 40 % of the time, the
// vector units (softmax, operands) 45 %, LDS 31 %: the two waves of a SIMD run beside each other only in part.  Put a
// phase apart by barriers (products of one beside the softmax of the other) they take 4 % more: the products of four
// waves at once need all that LDS gives.
template <int TYPE>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (TYPE == kMxBf16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(bits_as<bf16x8>(a), bits_as<bf16x8>(b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(bits_as<f16x8>(a), bits_as<f16x8>(b), c, 0, 0, 0);
}

template <int D, int WAVES>
struct TileLds {
  static constexpr int kKeys = 16 * WAVES, kPanels = kKeys / 64;
  static constexpr int kKPanel = 64 * D * 2, kVPanel = D * 128;  // K and V^T of 64 keys
  static constexpr int kV = kPanels * kKPanel, kStage = kV + kPanels * kVPanel;  // a power of two
  static constexpr int kNan = 2 * kStage, kOk = kNan + 2 * kKeys, kBytes = kOk + 2 * 4 * WAVES;
};

template <int TYPE, int FMT, int D, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2) void tile_kernel(AttnArgs a) {
  typedef KvLayout<FMT, D> L;
  typedef TileLds<D, WAVES> S;
  constexpr int kRows = 32 * WAVES;
  constexpr int kOcts = D / 8;
  constexpr int kKWords = D / 4 * L::kOct / 8 / 4;  // of a quarter of a key
  constexpr int kVWords = L::kOct;                  // of an octet of four keys
  extern __shared__ __align__(16) char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r32 = lane & 31, h = lane >> 5;
  const int tile = blockIdx.x / a.splits, head = blockIdx.y, b = blockIdx.z;
  const int split = split_of(a, blockIdx.x % a.splits, head, b);
  const Seq seq(a, b);
  clear_unheld<D>(a, seq, head, b, blockIdx.x == 0 && a.splits == 1);
  const int rows = seq.rows(a), row0 = tile * kRows;
  if (row0 >= rows) return;
  const int end_seen = seq.last_seen(a, (min(row0 + kRows, rows) - 1) / a.group) + 1;
  const int begin = (int)min((int64_t)split * a.split_len, (int64_t)0x7fffffff - 512);
  if (a.splits > 1 && begin >= end_seen) return;
  const int end = split + 1 < a.splits ? (int)min((int64_t)begin + a.split_len, (int64_t)end_seen) : end_seen;
  const int all_seen = seq.last_seen(a, row0 / a.group) + 1;  // every row sees the positions below

  const int r = row0 + wave * 32 + r32;
  const bool real = r < rows;
  const int t = real ? r / a.group : 0, qh = head * a.group + (real ? r - t * a.group : 0);
  const int lim = real ? seq.last_seen(a, t) : -1;
  const QSign sign(a);
  const float scale2 = sign.scale2;
  u32x4 q[D / 16];
#pragma unroll
  for (int j = 0; j < D / 16; ++j) {
    q[j] = u32x4{0u, 0u, 0u, 0u};
    if (real) q[j] = sign(load_any<u32x4>(a.q + ((seq.q0 + t) * a.q_ts + qh * a.q_hs + 16 * j + 8 * h) * 2));
  }
  // the last position that a row of this wave sees
  const int wave_row = min(row0 + (wave + 1) * 32, rows) - 1;
  const int wave_end = row0 + wave * 32 < rows ? seq.last_seen(a, wave_row / a.group) + 1 : 0;

  // (constant memory: behind the stores above the compiler would look pages up on the vector unit; 8 prompts of 2048:
  // 466 -> 519 us)
  const __attribute__((address_space(4))) int32_t* table =
      (const __attribute__((address_space(4))) int32_t*)(a.table + b * a.width);
  // this wave brings 16 keys of each tile: a lane a quarter of one key, and an octet of four keys' values
  uint32_t kw[kKWords], ks, vw[kVWords], vs;
  bool ok = false;
  const int vo = lane & 15, vg = lane >> 4;
  auto fetch = [&](int pos) {
    const int p0 = pos + 16 * wave;
    int page = -1;
    if (p0 < end) page = table[p0 >> a.c.shift];
    page = __builtin_amdgcn_readfirstlane(page);
    ok = page >= 0 && page < a.c.pages;
    ks = 1u;
    vs = 0u;
#pragma unroll
    for (int i = 0; i < kKWords; ++i) kw[i] = 0u;
#pragma unroll
    for (int i = 0; i < kVWords; ++i) vw[i] = 0u;
    if (!ok) return;
    const int64_t row = L::row0(a.c, page, head) + (p0 & (a.c.page - 1));
    const uint8_t* kp = a.c.kc + (row + (lane >> 2)) * L::kRow + (lane & 3) * (kKWords * 4);
    __builtin_memcpy(kw, __builtin_assume_aligned(kp, kKWords >= 4 ? 16 : 8), kKWords * 4);
    ks = a.c.ks[(row + (lane >> 2)) * L::kScales + (lane & 3) * (D / 4) / kMxBlock];
    if (vo < kOcts) {
      const uint8_t* vp = a.c.vc + L::v_code(row + 4 * vg, vo);
      __builtin_memcpy(vw, __builtin_assume_aligned(vp, 16), kVWords * 4);
      vs = *reinterpret_cast<const uint32_t*>(a.c.vs + L::v_scale(row + 4 * vg, vo / 4));
    }
  };
  // Addresses in LDS: the permutation of a row's pieces is an exclusive or of the piece with the row, and what is
  // constant in a piece's number can be applied last.
  const int key = 16 * wave + (lane >> 2);
  const int k_to = key * (D * 2) + ((((lane & 3) * (D / 32)) ^ (key & (kOcts - 1))) * 16);
  const int v_group = 4 * (wave & 3) + vg;  // of the panel
  const int v_to = S::kV + (wave >> 2) * S::kVPanel + vo * 1024 +
                   (((2 * (v_group >> 2) + (v_group & 1)) ^ (vo & 7)) * 16) + ((v_group >> 1) & 1) * 8;
  const int k_from = r32 * (D * 2) + ((h ^ (r32 & (kOcts - 1))) * 16);
  const int v_from = S::kV + r32 * 128 + ((h ^ ((r32 ^ (r32 >> 3)) & 7)) * 16);
  auto store = [&](int pos, int stage) {
    char* at = lds + stage * S::kStage;
    const float kscale = mx_scale(ks);
#pragma unroll
    for (int o = 0; o < D / 32; ++o) {
      u32x2 w = {0u, 0u};
      if constexpr (FMT == kMxFp4) w[0] = kw[o];
      else w = u32x2{kw[2 * o], kw[2 * o + 1]};
      *reinterpret_cast<u32x4*>(at + (k_to ^ (o * 16))) = mx_decode8<FMT, TYPE>(w, kscale);
    }
    uint32_t nan = 0;
    u32x2 w[4];
    float vscale[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      uint32_t byte = (vs >> (8 * e)) & 255u;
      if constexpr (FMT == kMxFp4) w[e] = u32x2{vw[e], 0u};
      else w[e] = u32x2{vw[2 * e], vw[2 * e + 1]};
      if (pos + 16 * wave + 4 * vg + e >= seq.kv_len) {
        byte = 0u;
        w[e] = u32x2{0u, 0u};
      }
      if (byte == 255u) {  // in mxfp8 the codes may be NaN under every scale
        nan |= 1u << e;
        byte = 0u;
        if constexpr (FMT == kMxFp8) w[e] = u32x2{0u, 0u};
      }
      vscale[e] = mx_scale(byte);
    }
    if (vo < kOcts) {
      const auto pair = [&](auto p_const) {
        constexpr int P = decltype(p_const)::value;
        uint32_t c[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) c[e] = mx_decode_pair<FMT, TYPE, P>(w[e], vscale[e]);
        const u32x2 lo = {__builtin_amdgcn_perm(c[1], c[0], 0x05040100u), __builtin_amdgcn_perm(c[3], c[2], 0x05040100u)};
        const u32x2 hi = {__builtin_amdgcn_perm(c[1], c[0], 0x07060302u), __builtin_amdgcn_perm(c[3], c[2], 0x07060302u)};
        *reinterpret_cast<u32x2*>(at + (v_to ^ (32 * P)) + 256 * P) = lo;
        *reinterpret_cast<u32x2*>(at + (v_to ^ (32 * P + 16)) + 256 * P + 128) = hi;
      };
      pair(std::integral_constant<int, 0>{});
      pair(std::integral_constant<int, 1>{});
      pair(std::integral_constant<int, 2>{});
      pair(std::integral_constant<int, 3>{});
      if ((vo & 3) == 0) lds[S::kNan + stage * S::kKeys + (4 * wave + vg) * 4 + vo / 4] = (char)nan;
    }
    // what the readers have to know of these 16 keys: 1: there are none, 2: some value block is NaN
    const uint32_t state = (ok ? 0u : 1u) | (__any(nan) ? 2u : 0u);
    if (lane == 0) *reinterpret_cast<uint32_t*>(lds + S::kOk + (stage * WAVES + wave) * 4) = state;
  };

  f32x16 o[D / 32];
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.f;

  // 64 keys: scores, softmax, product with V
  auto compute = [&](int pos, int stage, auto panel_const) {
    constexpr int panel = decltype(panel_const)::value;
    const char* from = lds + stage * S::kStage;
    f32x16 s[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[u][i] = 0.f;
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        const u32x4 k = *reinterpret_cast<const u32x4*>(from + (k_from ^ (32 * j)) + panel * S::kKPanel + u * (64 * D));
        s[u] = mfma32<TYPE>(k, q[j], s[u]);
      }
    }
    const u32x4 state = *reinterpret_cast<const u32x4*>(lds + S::kOk + stage * (4 * WAVES) + panel * 16);
    const uint32_t any = __builtin_amdgcn_readfirstlane(state[0] | state[1] | state[2] | state[3]);
    if (pos + 64 > all_seen || (any & 1u)) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const bool seen = !(state[2 * u + i / 8] & 1u) && pos + 32 * u + 8 * (i / 4) + 4 * h + i % 4 <= lim;
          s[u][i] = seen ? s[u][i] : -INFINITY;
        }
    }
    float x = -INFINITY;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) x = fmaxf(x, s[u][i]);
    const float top = max32(x) * scale2;
    if (__any(top > m + 8.f)) {
      const float to = top > m + 8.f ? top : m;
      const float alpha = to == m ? 1.f : exp2f(m - to);
      m = to;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] *= alpha;
    }
    if (any & 2u) {
#pragma unroll
      for (int d = 0; d < D / 32; ++d) {
        float poison = 0.f;
#pragma unroll 1
        for (int g = 0; g < 16; ++g) {
          const uint32_t f = (uint8_t)lds[S::kNan + stage * S::kKeys + (16 * panel + g) * 4 + d];
#pragma unroll 1
          for (int e = 0; e < 4; ++e)
            if ((f >> e & 1u) && pos + 4 * g + e <= lim) poison = NAN;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] += poison;
      }
    }
    const float base = m == -INFINITY ? 0.f : m;
    u32x4 p[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      float e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        e[i] = __builtin_amdgcn_exp2f(fmaf(s[c / 2][8 * (c % 2) + i], scale2, -base));
        l += e[i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) p[c][i] = pack2<TYPE>(e[2 * i], e[2 * i + 1]);
    }
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int d = 0; d < D / 32; ++d) {
        const u32x4 v = *reinterpret_cast<const u32x4*>(from + (v_from ^ (32 * (c ^ (2 * (d & 1))))) + panel * S::kVPanel +
                                                        d * 4096);
        o[d] = mfma32<TYPE>(v, p[c], o[d]);
      }
  };

  if (begin < end) {
    fetch(begin);
    store(begin, 0);
    fetch(begin + S::kKeys);
    __syncthreads();
    int stage = 0;
    const int last = min(end, wave_end);
    for (int pos = begin; pos < end; pos += S::kKeys) {
      if (pos + S::kKeys < end) {
        store(pos + S::kKeys, stage ^ 1);
        fetch(pos + 2 * S::kKeys);
      }
      if (pos < last) compute(pos, stage, std::integral_constant<int, 0>{});
      if constexpr (S::kPanels == 2)
        if (pos + 64 < last) compute(pos + 64, stage, std::integral_constant<int, 1>{});
      __syncthreads();
      stage ^= 1;
    }
  }

  const float sum = l + __shfl_xor(l, 32, 64);
  if (!real) return;
  const int64_t at = (int64_t)(seq.q0 + t) * a.q_heads + qh;
  if (a.splits > 1) {
    float* po = a.part_o + (at * a.splits + split) * D;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<f32x4*>(po + 32 * d + 8 * i + 4 * h) =
            f32x4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
    if (h == 0) {
      a.part_ml[(at * a.splits + split) * 2] = m;
      a.part_ml[(at * a.splits + split) * 2 + 1] = sum;
    }
    return;
  }
  const float inv = sum == 0.f ? 1.f : 1.f / sum;
  char* dst = a.out + at * (D * 2);
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<u32x2*>(dst + (32 * d + 8 * i + 4 * h) * 2) =
          u32x2{pack2<TYPE>(o[d][4 * i] * inv, o[d][4 * i + 1] * inv),
                pack2<TYPE>(o[d][4 * i + 2] * inv, o[d][4 * i + 3] * inv)};
  if (a.lse && h == 0) a.lse[at] = sum == 0.f ? -INFINITY : (m + log2f(sum)) * kLn2;
}

// Joins the runs of keys: a work-group a row, 16 lanes for a run's sums, 16 runs at a time; the runs of a group and
// then the groups are added in order.
template <int TYPE, int D>
__global__ __launch_bounds__(256) void join_kernel(AttnArgs a) {
  __shared__ float red_m[4];
  __shared__ __align__(16) float red_o[16][D + 4];
  __shared__ float red_l[16];
  const int head = blockIdx.y, b = blockIdx.z, r = blockIdx.x;
  const Seq seq(a, b);
  clear_unheld<D>(a, seq, head, b, r == 0);
  if (r >= seq.rows(a)) return;
  const int t = r / a.group;
  const int64_t at = (int64_t)(seq.q0 + t) * a.q_heads + head * a.group + (r - t * a.group);
  // runs that hold a position this row sees
  const int seen = seq.last_seen(a, t) + 1;
  const int n = seen <= 0 ? 0 : min((seen - 1) / a.split_len + 1, a.splits);
  const float* ml = a.part_ml + at * a.splits * 2;
  float top = -INFINITY;
  for (int s = threadIdx.x; s < n; s += 256) top = fmaxf(top, ml[2 * s]);
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
  if ((threadIdx.x & 63) == 0) red_m[threadIdx.x >> 6] = top;
  __syncthreads();
  top = fmaxf(fmaxf(red_m[0], red_m[1]), fmaxf(red_m[2], red_m[3]));
  const float base = top == -INFINITY ? 0.f : top;
  const int part = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * (D / 16);
  float v[D / 16], sum = 0.f;
#pragma unroll
  for (int d = 0; d < D / 16; ++d) v[d] = 0.f;
#pragma unroll 4
  for (int s = part; s < n; s += 16) {
    const float f = exp2f(ml[2 * s] - base);
    sum += f * ml[2 * s + 1];
    const float* po = a.part_o + (at * a.splits + s) * D + d0;
#pragma unroll
    for (int d = 0; d < D / 16; d += 4) {
      const f32x4 w = *reinterpret_cast<const f32x4*>(po + d);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[d + i] += f * w[i];
    }
  }
#pragma unroll
  for (int d = 0; d < D / 16; d += 4)
    *reinterpret_cast<f32x4*>(&red_o[part][d0 + d]) = f32x4{v[d], v[d + 1], v[d + 2], v[d + 3]};
  if ((threadIdx.x & 15) == 0) red_l[part] = sum;
  __syncthreads();
  if (threadIdx.x >= D / 2) return;
  float total = red_l[0], x = red_o[0][2 * threadIdx.x], y = red_o[0][2 * threadIdx.x + 1];
#pragma unroll
  for (int p = 1; p < 16; ++p) {
    total += red_l[p];
    x += red_o[p][2 * threadIdx.x];
    y += red_o[p][2 * threadIdx.x + 1];
  }
  const float inv = total == 0.f ? 1.f : 1.f / total;
  *reinterpret_cast<uint32_t*>(a.out + (at * D + 2 * threadIdx.x) * 2) = pack2<TYPE>(x * inv, y * inv);
  if (a.lse && threadIdx.x == 0) a.lse[at] = total == 0.f ? -INFINITY : (top + log2f(total)) * kLn2;
}

// ---- choice and launch ------------------------------------------------------------------------------------

struct Plan {
  int all_rows;  // of the longest sequence
  int rows;      // of a work-group: 16, 128 or 256
  int tiles, splits, split_len;
};

// Runs of keys of at least 256, as many as make 3072 work-groups of 16 rows (three rounds of four a CU: a third to a
// half of them find a run that their sequence does not reach) or 512 of more rows.  64 sequences of 512 to 8192
// positions, 8 key/value heads, mxfp4: 93 us with 1024 work-groups, 80 with 2048, 77 with 4096; 256 sequences of 100 to
// 2000: 68 us with up to 3072, 94 with 4096, which split them.  Up to 1024 positions of few rows are one run: what the join
// and its launch take (4 us, 18.2 against 14.5 us a call for one token of 16 query and 8 key/value heads) is more than
// what more work-groups save.
//
// Rows of a work-group: up to 64 rows (new tokens x query heads of a key/value head) the cache's bytes rule, and reading
// it four times is cheaper than 128 rows that are half empty (16 sequences of up to 8192 positions, 16 new tokens, four
// query heads to one: 76 against 88 us).  256 rows turn K and V into operands half as often as 128 and win over a long
// context (2 chunks of 2048 over 12000 to 16384 positions: 1027 against 1107 us); where the new tokens are most of
// the positions their waves wait for the one that sees the most (8 prompts of 2048: 577 against 475 us).
Plan plan_of(int64_t batch, int heads, int group, int64_t max_q, int64_t max_kv) {
  Plan p;
  const int64_t rows = max_q * group;
  p.all_rows = (int)rows;
  p.rows = rows <= 64 ? 16 : max_kv < 4 * max_q || batch * heads * mpq_cdiv(rows, 256) < 256 ? 128 : 256;
  p.tiles = (int)mpq_cdiv(rows, p.rows);
  const int64_t have = batch * heads * p.tiles;
  const int64_t most = std::max<int64_t>(1, mpq_cdiv(max_kv, 256));
  const int64_t groups = (p.rows == 16 ? 3072 : 512) / std::max<int64_t>(have, 1);
  const int64_t want = p.rows == 16 && max_kv <= 1024 ? 1 : std::min(most, std::max<int64_t>(1, groups));
  p.split_len = (int)(mpq_cdiv(mpq_cdiv(std::max<int64_t>(max_kv, 1), want), 128) * 128);
  p.splits = (int)std::max<int64_t>(1, mpq_cdiv(max_kv, p.split_len));
  return p;
}

template <class K>
hipError_t allow_lds(K kernel, int bytes) {
  if (bytes <= 64 * 1024) return hipSuccess;
  return hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

template <int TYPE, int FMT, int D, int WAVES>
hipError_t launch_tile(const AttnArgs& a, dim3 grid, hipStream_t stream) {
  constexpr int bytes = TileLds<D, WAVES>::kBytes;
  auto kernel = tile_kernel<TYPE, FMT, D, WAVES>;
  if (hipError_t e = allow_lds(kernel, bytes); e != hipSuccess) return e;
  hipLaunchKernelGGL(kernel, grid, dim3(64 * WAVES), bytes, stream, a);
  return hipSuccess;
}

template <int TYPE, int FMT, int D>
hipError_t run_attention(const AttnArgs& a, const Plan& p, int64_t batch, hipStream_t stream) {
  const dim3 grid((unsigned)(p.tiles * p.splits), (unsigned)a.c.heads, (unsigned)batch);
  if (p.rows == 16) {
    constexpr int bytes = Queue<FMT, D>::kBytes;
    auto kernel = rows16_kernel<TYPE, FMT, D>;
    if (hipError_t e = allow_lds(kernel, bytes); e != hipSuccess) return e;
    hipLaunchKernelGGL(kernel, grid, dim3(64 * kWaves), bytes, stream, a);
  } else if (p.rows == 128) {
    if (hipError_t e = launch_tile<TYPE, FMT, D, 4>(a, grid, stream); e != hipSuccess) return e;
  } else {
    if (hipError_t e = launch_tile<TYPE, FMT, D, 8>(a, grid, stream); e != hipSuccess) return e;
  }
  if (p.splits > 1)
    hipLaunchKernelGGL((join_kernel<TYPE, D>),
                       dim3((unsigned)p.all_rows, (unsigned)a.c.heads, (unsigned)batch), dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace
}  // namespace mpq

extern "C" int64_t mpq_kv_attend_workspace_size(int64_t total_q, int64_t batch, int64_t max_q, int64_t max_kv,
                                                int q_heads, int heads, int dim) {
  using namespace mpq;
  if (total_q <= 0 || batch <= 0 || max_q <= 0 || heads <= 0 || q_heads <= 0 || q_heads % heads || !kv_dim_ok(dim) ||
      max_q > (1 << 24) || max_kv < 0 || max_kv > 0x7ffff000)
    return 0;
  const Plan p = plan_of(batch, heads, q_heads / heads, max_q, max_kv);
  return p.splits == 1 ? 0 : total_q * q_heads * p.splits * (dim + 2) * (int64_t)sizeof(float);
}

extern "C" int mpq_kv_attend(const void* q, int dtype, int64_t total_q, int64_t q_token_stride, int64_t q_head_stride,
                             int q_heads, int64_t batch, const int32_t* block_table, int64_t table_width,
                             const int32_t* kv_lens, const int32_t* q_starts, int64_t max_q, int64_t max_kv, int fmt,
                             int heads, int dim, int page, int64_t pages, const uint8_t* k_codes,
                             const uint8_t* k_scales, const uint8_t* v_codes, const uint8_t* v_scales, float scale,
                             int causal, void* out, float* lse, void* workspace, int64_t workspace_bytes,
                             hipStream_t stream) {
  using namespace mpq;
  MPQ_CHECK_ARG(fmt == kMxFp4 || fmt == kMxFp8, "mpq_kv_attend: unknown format %d", fmt);
  MPQ_CHECK_ARG(dtype == kMxBf16 || dtype == kMxF16, "mpq_kv_attend: unknown type %d", dtype);
  MPQ_CHECK_ARG(kv_dim_ok(dim), "mpq_kv_attend: head size %d (64 or 128)", dim);
  MPQ_CHECK_ARG(heads >= 1 && heads <= 65535 && q_heads >= heads && q_heads % heads == 0 && q_heads <= (1 << 20),
                "mpq_kv_attend: %d query heads over %d key/value heads", q_heads, heads);
  MPQ_CHECK_ARG(page >= 16 && page <= 65536 && (page & (page - 1)) == 0,
                "mpq_kv_attend: pages of %d tokens (a power of two from 16)", page);
  MPQ_CHECK_ARG(pages >= 1 && pages <= ((int64_t)1 << 31), "mpq_kv_attend: %lld pages", (long long)pages);
  MPQ_CHECK_ARG(total_q >= 0 && total_q <= (1 << 30) && batch >= 0 && batch <= 65535 && max_q >= 0 &&
                    max_q <= (1 << 24) / (q_heads / heads) && table_width >= 0,
                "mpq_kv_attend: bad shape (%lld tokens, %lld sequences, up to %lld new tokens)", (long long)total_q,
                (long long)batch, (long long)max_q);
  MPQ_CHECK_ARG(std::isfinite(scale), "mpq_kv_attend: scale is not finite");
  MPQ_CHECK_ARG(total_q * (q_heads / heads) <= 0x7ffffff0, "mpq_kv_attend: extent too large");
  MPQ_CHECK_ARG(table_width <= 0x7ffff000 / page && max_kv >= 0 && max_kv <= table_width * page,
                "mpq_kv_attend: up to %lld positions, the table holds %lld pages of %d", (long long)max_kv,
                (long long)table_width, page);
  if (total_q == 0) return kOk;
  MPQ_CHECK_ARG(batch >= 1 && max_q >= 1, "mpq_kv_attend: %lld tokens do not fit %lld sequences of up to %lld",
                (long long)total_q, (long long)batch, (long long)max_q);
  MPQ_CHECK_ARG(q && kv_lens && q_starts && out && (block_table || table_width == 0), "mpq_kv_attend: null pointer");
  MPQ_CHECK_ARG(k_codes && k_scales && v_codes && v_scales, "mpq_kv_attend: null cache");
  const Plan p = plan_of(batch, heads, q_heads / heads, max_q, max_kv);
  MPQ_CHECK_ARG((int64_t)p.tiles * p.splits <= 0x7fffffff, "mpq_kv_attend: extent too large");
  const int64_t need = mpq_kv_attend_workspace_size(total_q, batch, max_q, max_kv, q_heads, heads, dim);
  MPQ_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0),
                "mpq_kv_attend: workspace of %lld bytes, %lld needed (16-byte aligned)", (long long)workspace_bytes,
                (long long)need);
  AttnArgs a;
  a.q = static_cast<const char*>(q);
  a.q_ts = q_token_stride;
  a.q_hs = q_head_stride;
  a.total_q = total_q;
  a.q_heads = q_heads;
  a.group = q_heads / heads;
  a.batch = (int)batch;
  a.max_q = (int)max_q;
  a.table = block_table;
  a.width = table_width;
  a.kv_lens = kv_lens;
  a.q_starts = q_starts;
  a.scale2 = scale * 1.44269504088896341f;
  a.causal = causal;
  a.split_len = p.split_len;
  a.splits = p.splits;
  a.out = static_cast<char*>(out);
  a.lse = lse;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = a.part_o + total_q * q_heads * p.splits * dim;
  a.c = KvCache{const_cast<uint8_t*>(k_codes), const_cast<uint8_t*>(k_scales), const_cast<uint8_t*>(v_codes),
                const_cast<uint8_t*>(v_scales), pages, heads, page, __builtin_ctz(page)};
  hipError_t e;
#define MPQ_A(T, F) (dim == 64 ? run_attention<T, F, 64>(a, p, batch, stream) : run_attention<T, F, 128>(a, p, batch, stream))
  if (dtype == kMxBf16) e = fmt == kMxFp4 ? MPQ_A(kMxBf16, kMxFp4) : MPQ_A(kMxBf16, kMxFp8);
  else e = fmt == kMxFp4 ? MPQ_A(kMxF16, kMxFp4) : MPQ_A(kMxF16, kMxFp8);
#undef MPQ_A
  MPQ_HIP_TRY(e);
  return kOk;
}
