// Single-token attention over a paged cache in bf16 or 4 bits, with grouped heads: per sequence b and query head h,
//   y = softmax(scale q k_t) v_t  over the cached tokens t < lengths[b],  kv head h / G,  G = H / kv_heads;
// zeros where a sequence has no token.
//
// Bound by the cache's bytes, so each row is read once for all G query heads of its kv head (groups of 16), straight into
// registers.  A wavefront walks its own range of tokens in tiles of 32 (two runs of 16, each within one page) with an online
// softmax of its own; nothing is shared until the ranges are joined, first the workgroup's wavefronts through LDS, then, where few
// sequences leave compute units idle, the splits of a sequence by a second launch.  A tile's keys are loaded behind the scores of
// the tile before, its values behind that one's value products, each into the registers just read, so that three wavefronts
// fit a SIMD, and it is their number that hides the latency (two sets of registers, two wavefronts: 48 sequences in 4 bits 80
// against 73 us, before the second term below).  bf16 reaches 4.7 to 5.1 TB/s (a copy 5.1).  4 bits reach 3.0 to 4.2, bound by the
// latency of the loads: by the counters of those 48 sequences a wavefront waits for loads in 53% of its time and for its turn
// to issue in 15%, and vector instructions, some 320 a tile, fill 63% of a SIMD's cycles (a third less of them, before the second
// term, gained nothing, 73 against 72 us): more bytes would have to be under way than one tile a wavefront.
//
// Products on v_mfma_f32_16x16x32 with the tokens (then the dims) as M and up to 16 query heads as N.  S = K Q^T: a lane
// (r, g) loads token r's dims and receives tokens 4 g .. 4 g + 3 of query r.  O^T = V^T P^T: a lane loads the 8 tokens that its
// own probabilities belong to, HD / 16 dims r HD / 16 .. of each, so 16 lanes read a row, and one v_perm per pair of tokens
// turns them into operands: dim r HD / 16 + i of the 8 tokens for product i.
//
// 4 bits: a row is lo + step * code, code 0 .. 15.  Codes become fp16 or bf16 by their bits alone (0x4300 | code is 128 + code of
// bf16, exactly), and step and lo act on sums:  q k = step (q (n + c) - n sum q) + lo sum q,  the accumulator starting from -n
// sum q,  and  sum_t p_t v_t = sum_t p'_t (128 + c_t) - 135.5 sum_t p'_t + sum_t p_t (lo_t + 7.5 step_t)  with p' = p step,
// whose sum is taken of the same rounded values on the matrix cores: a rounding acts on step (c - 7.5), a value's distance from
// its row's middle.  fp32 sums; the n cost 2^-20 of a sum.
//
// Probabilities (p') go into the products as two bf16 terms, a value and what its rounding left, 16 bits together: with one the
// result's error is 1.3 to 1.5 times that of its own rounding to bf16, so 1.0.  The products beside it cost bf16 rows nothing and
// 4-bit rows 5% (48 sequences 68 -> 71 us).
#include <algorithm>

#include "lm_paged.h"

namespace smlm {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 32;          // tokens of a wavefront's step
constexpr int kMaxSplits = 256;

template <int J>
__device__ __forceinline__ float xor_lane_f(float v) { return __uint_as_float(xor_lane<J>(__float_as_uint(v))); }

struct DecodeArgs {
  const uint16_t *q;
  int64_t q_stride;                // elements between sequences (H x HD dense)
  const int *table;
  int64_t table_stride;
  int max_pages;
  const int *lengths;
  uint16_t *y;                     // (B, H, HD), written where splits == 1
  float *parts, *stats;            // (B H, splits, HD) sums and (B H, splits, 2) maximum (log2) and sum of the exponentials
  int H, G, groups, splits;
  float scale_log2;
};

// 16 rows of one page and head as a buffer: a load's address is the descriptor's (uniform), a lane's offset that stays the same
// for the whole walk and an immediate.
struct Run {
  __amdgpu_buffer_rsrc_t r;
  __device__ __forceinline__ Run(const void *base, int bytes)
      : r(__builtin_amdgcn_make_buffer_rsrc((void *)base, (short)0, bytes, 0x00020000)) {}
  template <int BYTES>
  __device__ __forceinline__ void load(int offset, uint32_t *o) const {
    if constexpr (BYTES == 16) {
      const uint4 w = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, offset, 0, 0));
      o[0] = w.x, o[1] = w.y, o[2] = w.z, o[3] = w.w;
    } else if constexpr (BYTES == 8) {
      const uint2 w = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(r, offset, 0, 0));
      o[0] = w.x, o[1] = w.y;
    } else if constexpr (BYTES == 4) {
      o[0] = __builtin_amdgcn_raw_buffer_load_b32(r, offset, 0, 0);
    } else if constexpr (BYTES == 2) {
      o[0] = __builtin_amdgcn_raw_buffer_load_b16(r, offset, 0, 0);
    } else {
      o[0] = __builtin_amdgcn_raw_buffer_load_b8(r, offset, 0, 0);
    }
  }
};

template <int HD, bool Q4>
struct Tile {
  static constexpr int KS = HD / 32, ROWB = Q4 ? HD / 2 : HD * 2, VB = ROWB / 16;    // VB: bytes of a value row that a lane reads
  uint32_t k[2][KS * (Q4 ? 1 : 4)];
  uint32_t v[8][VB >= 4 ? VB / 4 : 1];
  uint32_t ks[2][4], vs[2][4];     // steps and lowest values of tokens 4 g .. 4 g + 3 of each run

  // keys and values of run kt from row `row` of the pages
  __device__ __forceinline__ void load_keys(const KVPages &P, int kt, int64_t row, int r, int g) {
    const Run kr((const char *)P.k + row * ROWB, 16 * ROWB);
    if constexpr (Q4) {
      kr.load<KS * 4>(r * ROWB + g * (KS * 4), k[kt]);
      Run((const char *)P.k_scale + row * 4, 64).load<16>(16 * g, ks[kt]);
    } else {
#pragma unroll
      for (int s = 0; s < KS; ++s) kr.load<16>(r * ROWB + 16 * g + 64 * s, k[kt] + 4 * s);
    }
  }
  __device__ __forceinline__ void load_values(const KVPages &P, int kt, int64_t row, int r, int g) {
    const Run vr((const char *)P.v + row * ROWB, 16 * ROWB);
    if constexpr (Q4) Run((const char *)P.v_scale + row * 4, 64).load<16>(16 * g, vs[kt]);
#pragma unroll
    for (int e = 0; e < 4; ++e) vr.load<VB>(4 * g * ROWB + r * VB + e * ROWB, v[4 * kt + e]);
  }
};

template <int HD, bool Q4, int NW>
__global__ void __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(NW == 8 ? 2 : 3)))
    paged_attention_kernel(DecodeArgs A, KVPages P) {
  constexpr int KS = HD / 32, MT = HD / 16;
  using T = Tile<HD, Q4>;
  extern __shared__ __align__(16) float smem[];     // [NW][16][HD] sums, then [NW][16][2] statistics

  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, r = lane & 15, g = lane >> 4;
  const int split = blockIdx.x % A.splits, rest = blockIdx.x / A.splits;
  const int hg = rest % A.groups, bk = rest / A.groups, kh = bk % P.kv_heads, b = bk / P.kv_heads;
  const int h0 = kh * A.G + hg * 16, nq = min(16, A.G - hg * 16);      // this workgroup's query heads
  const int64_t cap = (int64_t)A.max_pages << P.page_shift;
  const int len = (int)min((int64_t)max(A.lengths[b], 0), cap);
  const int tiles = (len + kTile - 1) / kTile, ranges = A.splits * NW, at = split * NW + wave;
  const int t0 = (int)((int64_t)tiles * at / ranges), t1 = (int)((int64_t)tiles * (at + 1) / ranges);

  // The queries as B fragments; dims as the keys' lanes hold them.  4 bits: in fp16, whose 10 bits of mantissa take a nibble at
  // bit 2 as 256 + code and at bit 6 as 16 + code, two nibbles of a half word for one shift; a word's dims 0 4, 1 5, 2 6 and 3 7
  // share registers, 1 5 and 3 7 in the upper place.  Scaled by a power of two to below 2: what fp16 then drops is below 2^-25
  // of the largest.
  bf16x8 bq[KS];
  [[maybe_unused]] float sum_q = 0.f, bias = 0.f, unscale = 1.f;
  {
    const uint16_t *row = A.q + b * A.q_stride + (h0 + min(r, nq - 1)) * HD;
    uint4 w[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) w[s] = *(const uint4 *)(row + (Q4 ? 8 * (g * KS + s) : 32 * s + 8 * g));
    if constexpr (Q4) {
      uint32_t top = 0;                  // the largest magnitude's bits
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const uint32_t u[4] = {w[s].x, w[s].y, w[s].z, w[s].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) top = max(top, max(u[i] & 0x7FFFu, u[i] >> 16 & 0x7FFFu));
      }
      top = max(top, xor_lane<16>(top));
      top = max(top, xor_lane<32>(top));
      const int e = min(max((int)(top >> 7), 27), 227);          // its exponent
      const float down = __uint_as_float((uint32_t)(254 - e) << 23);
      unscale = __uint_as_float((uint32_t)e << 23);
      float low_place = 0.f, high_place = 0.f;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const uint32_t u[4] = {w[s].x, w[s].y, w[s].z, w[s].w};
        _Float16 x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float f = __uint_as_float(i % 2 ? u[i / 2] & 0xFFFF0000u : u[i / 2] << 16) * down;
          x[i] = (_Float16)f;
          (i % 2 ? high_place : low_place) += (float)x[i];
        }
        typedef _Float16 half8 __attribute__((ext_vector_type(8)));
        bq[s] = __builtin_bit_cast(bf16x8, half8{x[0], x[4], x[1], x[5], x[2], x[6], x[3], x[7]});
      }
      low_place += xor_lane_f<16>(low_place);
      low_place += xor_lane_f<32>(low_place);
      high_place += xor_lane_f<16>(high_place);
      high_place += xor_lane_f<32>(high_place);
      bias = -256.f * low_place - 16.f * high_place;
      sum_q = low_place + high_place;
    } else {
#pragma unroll
      for (int s = 0; s < KS; ++s) bq[s] = __builtin_bit_cast(bf16x8, w[s]);
    }
  }
  const float scale = Q4 ? A.scale_log2 * unscale : A.scale_log2;

  // page ids, 64 at a time, one a lane
  const int *table = A.table + b * A.table_stride;
  int window = -1, ids = 0;
  const int64_t head_row = (int64_t)kh << P.page_shift;
  T x;
  int64_t rows[2];                     // where the runs of the tile that is loaded last lie, and how many tokens they hold
  int next[2], valid[2];
  auto load_keys = [&](int t) __attribute__((always_inline)) {
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const int tok = t * kTile + 16 * kt, page = tok >> P.page_shift;
      if (window < 0 || page >= window + 64) {       // uniform
        window = page;
        const int i = window + lane;
        ids = i < A.max_pages ? table[i] : -1;
      }
      const int id = __builtin_amdgcn_readlane(ids, page - window);
      const bool good = id >= 0 && id < P.num_pages;
      next[kt] = good ? min(max(len - tok, 0), 16) : 0;
      rows[kt] = (((int64_t)(good ? id : 0) * P.kv_heads) << P.page_shift) + head_row + (tok & ((1 << P.page_shift) - 1));
      x.load_keys(P, kt, rows[kt], r, g);
    }
  };
  auto load_values = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) x.load_values(P, kt, rows[kt], r, g);
  };

  const floatx4 zero4 = {0.f, 0.f, 0.f, 0.f};
  float m = -3.0e38f, l = 0.f, low = 0.f;
  floatx4 oacc[MT], pacc = zero4;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) oacc[mt] = zero4;
  const bf16x8 ones = __builtin_bit_cast(bf16x8, uint4{0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u});

  // (masks in registers: a bitwise and-or takes one constant of its own at most)
  uint32_t low4 = 0x000F000Fu, at2 = 0x003C003Cu, at6 = 0x03C003C0u;
  asm volatile("" : "+v"(low4), "+v"(at2), "+v"(at6));

  auto compute = [&](int t) __attribute__((always_inline)) {
    valid[0] = next[0], valid[1] = next[1];
    floatx4 sc[2];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      if constexpr (Q4) {
        typedef _Float16 half8 __attribute__((ext_vector_type(8)));
        sc[kt] = floatx4{bias, bias, bias, bias};
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          const uint32_t w = x.k[kt][s] << 2, v = x.k[kt][s] >> 6;
          const uint4 a{(w & at2) | 0x5C005C00u, (w & at6) | 0x4C004C00u, (v & at2) | 0x5C005C00u, (v & at6) | 0x4C004C00u};
          sc[kt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, bq[s]), sc[kt], 0,
                                                          0, 0);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t w = x.ks[kt][i];
          const float step = __uint_as_float(w << 16);
          // (a key that is not finite has an infinite step: its lowest value as NaN, or the infinities might add up to -infinity)
          sc[kt][i] = step * sc[kt][i] + __builtin_fmaf(step, 0.f, __uint_as_float(w & 0xFFFF0000u)) * sum_q;
        }
      } else {
        sc[kt] = zero4;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          const uint4 a{x.k[kt][4 * s], x.k[kt][4 * s + 1], x.k[kt][4 * s + 2], x.k[kt][4 * s + 3]};
          sc[kt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), bq[s], sc[kt], 0, 0, 0);
        }
      }
    }
    if (t + 1 < t1) load_keys(t + 1);        // (into the registers that the scores were read from)
    uint32_t vs[2][4];
    if constexpr (Q4) {
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) vs[kt][i] = x.vs[kt][i];
    }
    const bool full = valid[0] == 16 && valid[1] == 16;
    if (!full) {
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (4 * g + i >= valid[kt]) {
            sc[kt][i] = -__builtin_inff();
            if constexpr (Q4) vs[kt][i] = 0;
          }
    }
    // Online softmax per query (lane) in the log2 domain, with a reference point m that moves, to 2^8 above a tile's maximum, only
    // when an exponential reaches 2 (one of the group's heads: all whose maximum is as near to it, 2^0.99, move theirs).
    float p[8];
    auto exponentials = [&]() __attribute__((always_inline)) {
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        p[i] = __builtin_amdgcn_exp2f(sc[i / 4][i % 4] * scale - m);
        top = __builtin_elementwise_maximum(top, p[i]);
      }
      return !(top < 2.f);
    };
    if (__builtin_amdgcn_ballot_w64(exponentials())) {
      float a = -__builtin_inff();
#pragma unroll
      for (int i = 0; i < 8; ++i) a = fmaxf(a, sc[i / 4][i % 4]);
      a = fmaxf(a, xor_lane_f<16>(a));
      a = fmaxf(a, xor_lane_f<32>(a)) * scale;
      const float mnew = a - m > 0.99f ? a + 8.f : m, alpha = __builtin_amdgcn_exp2f(m - mnew);
      m = mnew;
      l *= alpha;
      if constexpr (Q4) {
        low *= alpha;
        pacc *= alpha;
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) oacc[mt] *= alpha;
      exponentials();
    }
    uint32_t pk[4];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      l += p[i];
      if constexpr (Q4) {
        const uint32_t u = vs[i / 4][i % 4];
        const float step = __uint_as_float(u << 16);
        low += p[i] * (7.5f * step + __uint_as_float(u & 0xFFFF0000u));
        p[i] *= step;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) pk[i] = pack_bf16x2(p[2 * i], p[2 * i + 1]);
    const bf16x8 bp = __builtin_bit_cast(bf16x8, uint4{pk[0], pk[1], pk[2], pk[3]});
#pragma unroll
    for (int i = 0; i < 4; ++i)
      pk[i] = pack_bf16x2(p[2 * i] - __uint_as_float(pk[i] << 16), p[2 * i + 1] - __uint_as_float(pk[i] & 0xFFFF0000u));
    const bf16x8 rest = __builtin_bit_cast(bf16x8, uint4{pk[0], pk[1], pk[2], pk[3]});
    if constexpr (Q4) {
      pacc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, bp, pacc, 0, 0, 0);
      pacc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, rest, pacc, 0, 0, 0);
#pragma unroll
      for (int j = 0; j < MT / 2; ++j) {     // byte j: dims 2 j and 2 j + 1 of the lane's
        uint32_t a[4], c[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t w = __builtin_amdgcn_perm(x.v[2 * e + 1][0], x.v[2 * e][0], 0x0C000C00u | (uint32_t)j | (4u + j) << 16);
          a[e] = (w & low4) | 0x43004300u;
          c[e] = (w >> 4 & low4) | 0x43004300u;
        }
        const bf16x8 even = __builtin_bit_cast(bf16x8, uint4{a[0], a[1], a[2], a[3]});
        const bf16x8 odd = __builtin_bit_cast(bf16x8, uint4{c[0], c[1], c[2], c[3]});
        oacc[2 * j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(even, bp, oacc[2 * j], 0, 0, 0);
        oacc[2 * j + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(odd, bp, oacc[2 * j + 1], 0, 0, 0);
        oacc[2 * j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(even, rest, oacc[2 * j], 0, 0, 0);
        oacc[2 * j + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(odd, rest, oacc[2 * j + 1], 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        uint32_t a[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          a[e] = __builtin_amdgcn_perm(x.v[2 * e + 1][mt / 2], x.v[2 * e][mt / 2], mt % 2 ? 0x07060302u : 0x05040100u);
          if (!full) {       // what lies behind the last token may be anything, and 0 times a NaN is one
            const int i = 2 * (e & 1), kt = e / 2;
            a[e] = (4 * g + i < valid[kt] ? a[e] & 0xFFFFu : 0u) | (4 * g + i + 1 < valid[kt] ? a[e] & 0xFFFF0000u : 0u);
          }
        }
        const bf16x8 v = __builtin_bit_cast(bf16x8, uint4{a[0], a[1], a[2], a[3]});
        oacc[mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, bp, oacc[mt], 0, 0, 0);
        oacc[mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, rest, oacc[mt], 0, 0, 0);
      }
    }
    if (t + 1 < t1) load_values();
  };

  if (t0 < t1) {
    load_keys(t0);
    load_values();
    for (int t = t0; t < t1; ++t) compute(t);
  }

  l += xor_lane_f<16>(l);
  l += xor_lane_f<32>(l);
  if constexpr (Q4) {
    low += xor_lane_f<16>(low);
    low += xor_lane_f<32>(low);
  }
  // the wavefronts' sums: lane (r, g) holds dims (4 g + i) HD / 16 + mt of query r
  float *stats = smem + NW * 16 * HD;
  if (r < nq) {
    float *o = smem + (wave * 16 + r) * HD;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) o[(4 * g + i) * MT + mt] = Q4 ? oacc[mt][i] - 135.5f * pacc[i] + low : oacc[mt][i];
    if (g == 0) stats[(wave * 16 + r) * 2] = m, stats[(wave * 16 + r) * 2 + 1] = l;
  }
  __syncthreads();
  for (int i = tid; i < nq * HD; i += NW * 64) {
    const int qi = i / HD, d = i % HD;
    float top = -3.0e38f, sum = 0.f, total = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) top = fmaxf(top, stats[(w * 16 + qi) * 2]);
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = __builtin_amdgcn_exp2f(stats[(w * 16 + qi) * 2] - top);
      sum += f * smem[(w * 16 + qi) * HD + d];
      total += f * stats[(w * 16 + qi) * 2 + 1];
    }
    const int64_t at = (int64_t)b * A.H + h0 + qi;
    if (A.splits == 1) {
      A.y[at * HD + d] = (uint16_t)(pack_bf16x2(total != 0.f ? sum / total : 0.f, 0.f) & 0xFFFFu);
    } else {
      A.parts[(at * A.splits + split) * HD + d] = sum;
      if (d == 0) A.stats[(at * A.splits + split) * 2] = top, A.stats[(at * A.splits + split) * 2 + 1] = total;
    }
  }
}

// the splits of one (sequence, query head) joined: 256 threads = 1024 / HD runs of splits x HD / 4 groups of dims
template <int HD>
__global__ void __launch_bounds__(256) paged_join_kernel(const float *parts, const float *stats, int splits, uint16_t *y) {
  constexpr int RUNS = 1024 / HD;
  __shared__ float s_w[kMaxSplits], s_m[4], s_l[4];
  __shared__ float4 s_o[RUNS][HD / 4];
  const int64_t at = blockIdx.x;
  const int tid = threadIdx.x, d = tid % (HD / 4), run = tid / (HD / 4);
  const float4 *in = (const float4 *)(parts + at * splits * HD) + d;
  // (splits <= 256: one a thread)
  const float mine = tid < splits ? stats[(at * splits + tid) * 2] : -3.0e38f;
  const float mass = tid < splits ? stats[(at * splits + tid) * 2 + 1] : 0.f;
  float top = mine;
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, kWave));
  if (tid % kWave == 0) s_m[tid / kWave] = top;
  __syncthreads();
  top = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
  const float f = __builtin_amdgcn_exp2f(mine - top);
  s_w[tid] = f;
  const float part = wave_sum(f * mass);
  if (tid % kWave == 0) s_l[tid / kWave] = part;
  __syncthreads();
  float4 sum{0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int s = run; s < splits; s += RUNS) {
    const float4 v = in[(int64_t)s * (HD / 4)];
    const float w = s_w[s];
    sum.x += w * v.x, sum.y += w * v.y, sum.z += w * v.z, sum.w += w * v.w;
  }
  s_o[run][d] = sum;
  __syncthreads();
  if (tid < HD) {
    const float *o = (const float *)s_o + tid;
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < RUNS; ++i) v += o[i * HD];
    const float total = (s_l[0] + s_l[1]) + (s_l[2] + s_l[3]);
    y[at * HD + tid] = (uint16_t)(pack_bf16x2(total != 0.f ? v / total : 0.f, 0.f) & 0xFFFFu);
  }
}

// How the walks are split.  One workgroup per sequence and group of heads, of 4 wavefronts, or of 8 where there are few of them and
// the table holds at most 1,024 tokens (32 sequences of up to 700, 6 heads of 64, 4 bits: 10.0 us as splits and a join, 7.5 so;
// 16 of 2,000, one kv head: 8.6 and 14.5).  Longer ones are split, into ranges of some 256 tokens of a full table (fewer by what
// rounds the number of splits up) or more: into 768 workgroups, three for each of the 256 compute units, all of them running at
// once (2 x 131,072 tokens in 4 bits: 68 us; 1,024 workgroups 80, 2,304 79), or, from 8 sequences on, into three times as many,
// which even out where lengths differ (48 of up to 8,191: 768 workgroups 78 us, 2,304 71).  The lengths are on the device alone, so
// their number stands in for whether they differ: 48 of 4,500 each take 58 us in 768 and 66 in 2,304; 9 of 30,000, whose 792
// workgroups do not all run at once, 98 and 79; 7 of up to 40,000 53 either way.  The plan follows the table, not the
// lengths: short sequences in a long table pay for its splits and their join.
// (Shares of equally many tiles, cut from the lengths on the device, before the second term above: 72 -> 70 us for these 48, 65 ->
// 61 for equal ones, but 10.5 -> 14.2 for 16 of 2,000 tokens, whose prefix sums and divisions take as long as their walk.)
struct Plan {
  int waves, splits;
};
Plan plan_of(int64_t B, int kv_heads, int groups, int64_t cap) {
  const int64_t units = std::max<int64_t>(1, B * kv_heads * groups);
  const int64_t target = B < 8 ? 768 : 2304;
  const int splits = (int)std::max<int64_t>(1, std::min<int64_t>({(target + units - 1) / units, (cap + 255) / 256, kMaxSplits}));
  return splits > 1 && cap <= 1024 ? Plan{8, 1} : Plan{4, splits};
}

template <int HD, bool Q4, int NW>
void launch_walk(const DecodeArgs &A, const KVPages &P, int64_t B, hipStream_t s) {
  const size_t lds = (size_t)NW * 16 * (HD + 2) * sizeof(float);
  hipLaunchKernelGGL((paged_attention_kernel<HD, Q4, NW>), dim3((unsigned)(B * P.kv_heads * A.groups * A.splits)), dim3(NW * 64), lds,
                     s, A, P);
}

template <int HD, bool Q4>
int launch(const DecodeArgs &A, const KVPages &P, int waves, int64_t B, hipStream_t s) {
  if (waves == 8) {
    if constexpr (HD == 128) {                  // over 64 KB
      const hipError_t e = hipFuncSetAttribute((const void *)paged_attention_kernel<HD, Q4, 8>,
                                               hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
      if (e != hipSuccess) return fail(SMLM_EHIP, "smlm_paged_attention: hipFuncSetAttribute: %s", hipGetErrorString(e));
    }
    launch_walk<HD, Q4, 8>(A, P, B, s);
  } else {
    launch_walk<HD, Q4, 4>(A, P, B, s);
  }
  if (A.splits > 1)
    hipLaunchKernelGGL((paged_join_kernel<HD>), dim3((unsigned)(B * A.H)), dim3(256), 0, s, A.parts, A.stats, A.splits, A.y);
  return launch_status("smlm_paged_attention");
}

}  // namespace
}  // namespace smlm

extern "C" int64_t smlm_paged_attention_workspace(int64_t B, int H, int kv_heads, int head_dim, int page_size,
                                                  int64_t max_pages) {
  using namespace smlm;
  if (B <= 0 || B > 0x7FFFFFFF || H < 1 || H > 65536 || kv_heads < 1 || head_dim < 1 || page_size < 1 || max_pages < 1 || max_pages > 0x7FFFFFFF ||
      H % kv_heads)
    return 0;
  const int splits = plan_of(B, kv_heads, (H / kv_heads + 15) / 16, max_pages * page_size).splits;
  return splits == 1 ? 0 : B * H * splits * (head_dim + 2) * (int64_t)sizeof(float);
}

extern "C" int smlm_paged_attention(const void *q, int64_t q_row_stride, const smlm_kv_pages *pages, const int *block_table,
                                    int64_t table_row_stride, int64_t max_pages, const int *lengths, int64_t B, int H,
                                    float scale, void *y, void *workspace, int64_t workspace_bytes, void *stream) {
  using namespace smlm;
  const char *name = "smlm_paged_attention";
  KVPages P;
  if (const int rc = kv_pages(name, pages, &P)) return rc;
  if (!q || !block_table || !lengths || !y) return fail(SMLM_EINVAL, "%s: null pointer argument", name);
  const int hd = pages->head_dim;
  if (B < 0 || B > 0x7FFFFFFF || H < 1 || H > 65536 || H % pages->kv_heads || max_pages < 0 ||
      max_pages > 0x7FFFFFFF || table_row_stride < max_pages)
    return fail(SMLM_EINVAL, "%s: bad shape B=%lld H=%d kv_heads=%d max_pages=%lld", name, (long long)B, H, pages->kv_heads,
                (long long)max_pages);
  if (q_row_stride < (int64_t)H * hd || q_row_stride % 8 || ((uintptr_t)q | (uintptr_t)y) % 16 ||
      ((uintptr_t)block_table | (uintptr_t)lengths) % 4)
    return fail(SMLM_EINVAL, "%s: q and y must be 16-byte aligned, q's row stride >= H * head_dim and a multiple of 8", name);
  if (!(scale > 0.f) || scale > 1e38f) return fail(SMLM_EINVAL, "%s: the scale must be positive, at most 1e38", name);
  if (max_pages * pages->page_size > 0x7FFFFF00LL)
    return fail(SMLM_EUNSUPPORTED, "%s: a block table of %lld pages is more than 2^31 tokens", name, (long long)max_pages);
  const int G = H / pages->kv_heads, groups = (G + 15) / 16;
  const auto [waves, splits] = plan_of(B, pages->kv_heads, groups, max_pages * pages->page_size);
  if (B * pages->kv_heads * groups * splits > 0x7FFFFFFFLL || B * H > 0x7FFFFFFFLL)
    return fail(SMLM_EUNSUPPORTED, "%s: B=%lld sequences are too many workgroups", name, (long long)B);
  const int64_t need = smlm_paged_attention_workspace(B, H, pages->kv_heads, hd, pages->page_size, max_pages);
  if (need && (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < need))
    return fail(SMLM_EINVAL, "%s: the workspace must be %lld bytes, 16-byte aligned", name, (long long)need);
  if (B == 0) return SMLM_OK;
  float *parts = (float *)workspace;
  const DecodeArgs A{(const uint16_t *)q, q_row_stride, block_table, table_row_stride, (int)max_pages, lengths, (uint16_t *)y,
                     parts, parts + B * H * splits * hd, H, G, groups, splits, scale * 1.4426950408889634f};
  const bool q4 = pages->kind == SMLM_Q4;
  hipStream_t s = (hipStream_t)stream;
  if (hd == 32) return q4 ? launch<32, true>(A, P, waves, B, s) : launch<32, false>(A, P, waves, B, s);
  if (hd == 64) return q4 ? launch<64, true>(A, P, waves, B, s) : launch<64, false>(A, P, waves, B, s);
  return q4 ? launch<128, true>(A, P, waves, B, s) : launch<128, false>(A, P, waves, B, s);
}
