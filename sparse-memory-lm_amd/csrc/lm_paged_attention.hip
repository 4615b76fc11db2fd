// Single-token attention over a paged cache in bf16 or 4 bits, with grouped heads: per sequence b and query head h,
//   y = softmax(scale q k_t) v_t  over the cached tokens t < lengths[b],  kv head h / G,  G = H / kv_heads;
// zeros where a sequence has no token.
//
// Bound by the cache's bytes, so each row is read once for all G query heads of its kv head (groups of 16), straight into
// registers, while the tile before is computed.  A wavefront walks its own range of tokens in tiles of 32 (two runs of 16, each
// within one page) with an online softmax of its own; nothing is shared until the ranges are joined, first the workgroup's
// wavefronts through LDS, then, where few sequences leave compute units idle, the splits of a sequence by a second launch.
//
// Products on v_mfma_f32_16x16x32_bf16 with the tokens (then the dims) as M and up to 16 query heads as N.  S = K Q^T: a lane
// (r, g) loads token r's dims and receives tokens 4 g .. 4 g + 3 of query r.  O^T = V^T P^T: a lane loads the 8 tokens that its
// own probabilities belong to, HD / 16 dims r HD / 16 .. of each, so 16 lanes read a row, and one v_perm per pair of tokens
// turns them into operands: dim r HD / 16 + i of the 8 tokens for product i.
//
// 4 bits: a row is lo + step * code, code 0 .. 15.  Codes become bf16 by their bits alone (0x4300 | code is 128 + code, exactly)
// and step and lo act on sums:  q k = step (q (128 + c) - 128 sum q) + lo sum q,  the accumulator starting from -128 sum q,
// and  sum_t p_t v_t = sum_t p'_t (128 + c_t) - 135.5 sum_t p'_t + sum_t p_t (lo_t + 7.5 step_t)  with p' = p step rounded to
// bf16 (as a probability is), whose sum is taken of the same rounded values on the matrix cores: the rounding acts on step (c -
// 7.5), a value's distance from its row's middle (on step c, from the row's lowest, it took the result's error from 0.0021 to
// 0.0046).  fp32 sums; the 128s cost 2^-20 of a sum.
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

template <int HD, bool Q4>
struct Tile {
  static constexpr int KS = HD / 32;
  static constexpr int VB = HD / 16 * (Q4 ? 1 : 4) / 2;    // bytes of a value row that a lane reads
  uint32_t k[2][KS * (Q4 ? 1 : 4)];
  uint32_t v[8][VB >= 4 ? VB / 4 : 1];
  uint4 ks[2], vs[2];              // steps and lowest values of tokens 4 g .. 4 g + 3 of each run
  int valid[2];                    // tokens of each run (uniform)
};

template <int BYTES>
__device__ __forceinline__ void load_bytes(const char *p, uint32_t *o) {
  if constexpr (BYTES == 64) {
#pragma unroll
    for (int i = 0; i < 4; ++i) load_bytes<16>(p + 16 * i, o + 4 * i);
  } else if constexpr (BYTES == 16) {
    const uint4 w = *(const uint4 *)p;
    o[0] = w.x, o[1] = w.y, o[2] = w.z, o[3] = w.w;
  } else if constexpr (BYTES == 8) {
    const uint2 w = *(const uint2 *)p;
    o[0] = w.x, o[1] = w.y;
  } else if constexpr (BYTES == 4) {
    o[0] = *(const uint32_t *)p;
  } else if constexpr (BYTES == 2) {
    o[0] = *(const uint16_t *)p;
  } else {
    o[0] = *(const uint8_t *)p;
  }
}

template <int HD, bool Q4, int NW>
__global__ void __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(2)))
    paged_attention_kernel(DecodeArgs A, KVPages P) {
  constexpr int KS = HD / 32, MT = HD / 16, ROWB = Q4 ? HD / 2 : HD * 2;
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

  // the queries as B fragments; dims as the keys' lanes hold them (4 bits: a word's nibbles 0 4, 1 5, 2 6, 3 7)
  bf16x8 bq[KS];
  float sum_q = 0.f;
  {
    const uint16_t *row = A.q + b * A.q_stride + (h0 + min(r, nq - 1)) * HD;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const uint4 w = *(const uint4 *)(row + (Q4 ? 8 * (g * KS + s) : 32 * s + 8 * g));
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
      if constexpr (Q4) {
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {      // dims i and i + 4
          o[i] = __builtin_amdgcn_perm(u[2 + i / 2], u[i / 2], i % 2 ? 0x07060302u : 0x05040100u);
          sum_q += __uint_as_float(u[i] << 16) + __uint_as_float(u[i] & 0xFFFF0000u);
        }
        bq[s] = __builtin_bit_cast(bf16x8, uint4{o[0], o[1], o[2], o[3]});
      } else {
        bq[s] = __builtin_bit_cast(bf16x8, w);
      }
    }
    if constexpr (Q4) {
      sum_q += xor_lane_f<16>(sum_q);
      sum_q += xor_lane_f<32>(sum_q);
    }
  }

  // page ids, 64 at a time, one a lane
  const int *table = A.table + b * A.table_stride;
  int window = -1, ids = 0;
  const int64_t head_row = (int64_t)kh << P.page_shift;
  auto load = [&](int t, T &o) {
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
      o.valid[kt] = good ? min(max(len - tok, 0), 16) : 0;
      const int64_t row = (((int64_t)(good ? id : 0) * P.kv_heads) << P.page_shift) + head_row + (tok & ((1 << P.page_shift) - 1));
      const char *kp = (const char *)P.k + row * ROWB, *vp = (const char *)P.v + row * ROWB;
      if constexpr (Q4) {
        load_bytes<KS * 4>(kp + r * ROWB + g * (KS * 4), o.k[kt]);
        o.ks[kt] = *(const uint4 *)((const char *)P.k_scale + (row + 4 * g) * 4);
        o.vs[kt] = *(const uint4 *)((const char *)P.v_scale + (row + 4 * g) * 4);
      } else {
#pragma unroll
        for (int s = 0; s < KS; ++s) load_bytes<16>(kp + r * ROWB + 64 * s + 16 * g, o.k[kt] + 4 * s);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) load_bytes<T::VB>(vp + (4 * g + e) * ROWB + r * T::VB, o.v[4 * kt + e]);
    }
  };

  const floatx4 zero4 = {0.f, 0.f, 0.f, 0.f};
  float m = -3.0e38f, l = 0.f, low = 0.f;
  floatx4 oacc[MT], pacc = zero4;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) oacc[mt] = zero4;
  const bf16x8 ones = __builtin_bit_cast(bf16x8, uint4{0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u});

  auto compute = [&](const T &x) {
    floatx4 sc[2];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      sc[kt] = zero4;
      if constexpr (Q4) sc[kt] = floatx4{-128.f, -128.f, -128.f, -128.f} * sum_q;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        uint4 a;
        if constexpr (Q4) {
          const uint32_t w = x.k[kt][s];
          a = uint4{(w & 0x000F000Fu) | 0x43004300u, (w >> 4 & 0x000F000Fu) | 0x43004300u, (w >> 8 & 0x000F000Fu) | 0x43004300u,
                    (w >> 12 & 0x000F000Fu) | 0x43004300u};
        } else {
          a = uint4{x.k[kt][4 * s], x.k[kt][4 * s + 1], x.k[kt][4 * s + 2], x.k[kt][4 * s + 3]};
        }
        sc[kt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), bq[s], sc[kt], 0, 0, 0);
      }
      if constexpr (Q4) {
        const uint32_t w[4] = {x.ks[kt].x, x.ks[kt].y, x.ks[kt].z, x.ks[kt].w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          sc[kt][i] = __uint_as_float(w[i] << 16) * sc[kt][i] + __uint_as_float(w[i] & 0xFFFF0000u) * sum_q;
      }
    }
    const bool full = x.valid[0] == 16 && x.valid[1] == 16;
    if (!full) {
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (4 * g + i >= x.valid[kt]) sc[kt][i] = -__builtin_inff();
    }
    float mx = fmaxf(fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3])),
                     fmaxf(fmaxf(sc[1][0], sc[1][1]), fmaxf(sc[1][2], sc[1][3])));
    mx = fmaxf(mx, xor_lane_f<16>(mx));
    mx = fmaxf(mx, xor_lane_f<32>(mx)) * A.scale_log2;
    if (__builtin_amdgcn_ballot_w64(mx > m + 8.f)) {       // as long as no maximum grows by 2^8, none is rescaled
      const float mnew = mx > m + 8.f ? mx : m, alpha = __builtin_amdgcn_exp2f(m - mnew);
      m = mnew;
      l *= alpha;
      if constexpr (Q4) {
        low *= alpha;
        pacc *= alpha;
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) oacc[mt] *= alpha;
    }
    uint32_t pk[4];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      float p[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[i] = __builtin_amdgcn_exp2f(sc[kt][i] * A.scale_log2 - m);
        l += p[i];
      }
      if constexpr (Q4) {
        const uint32_t w[4] = {x.vs[kt].x, x.vs[kt].y, x.vs[kt].z, x.vs[kt].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t u = full || 4 * g + i < x.valid[kt] ? w[i] : 0u;
          const float step = __uint_as_float(u << 16);
          low += p[i] * (7.5f * step + __uint_as_float(u & 0xFFFF0000u));
          p[i] *= step;
        }
      }
      pk[2 * kt] = pack_bf16x2(p[0], p[1]);
      pk[2 * kt + 1] = pack_bf16x2(p[2], p[3]);
    }
    const bf16x8 bp = __builtin_bit_cast(bf16x8, uint4{pk[0], pk[1], pk[2], pk[3]});
    if constexpr (Q4) {
      pacc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, bp, pacc, 0, 0, 0);
#pragma unroll
      for (int j = 0; j < MT / 2; ++j) {     // byte j: dims 2 j and 2 j + 1 of the lane's
        uint32_t a[4], c[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t w = __builtin_amdgcn_perm(x.v[2 * e + 1][0], x.v[2 * e][0], 0x0C000C00u | (uint32_t)j | (4u + j) << 16);
          a[e] = (w & 0x000F000Fu) | 0x43004300u;
          c[e] = (w >> 4 & 0x000F000Fu) | 0x43004300u;
        }
        oacc[2 * j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, uint4{a[0], a[1], a[2], a[3]}), bp,
                                                              oacc[2 * j], 0, 0, 0);
        oacc[2 * j + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, uint4{c[0], c[1], c[2], c[3]}), bp,
                                                                  oacc[2 * j + 1], 0, 0, 0);
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
            a[e] = (4 * g + i < x.valid[kt] ? a[e] & 0xFFFFu : 0u) | (4 * g + i + 1 < x.valid[kt] ? a[e] & 0xFFFF0000u : 0u);
          }
        }
        oacc[mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, uint4{a[0], a[1], a[2], a[3]}), bp,
                                                           oacc[mt], 0, 0, 0);
      }
    }
  };

  if (t0 < t1) {
    T even, odd;
    load(t0, even);
    for (int t = t0; t < t1; t += 2) {
      if (t + 1 < t1) load(t + 1, odd);
      compute(even);
      if (t + 2 < t1) load(t + 2, even);
      if (t + 1 < t1) compute(odd);
    }
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

// the splits of one (sequence, query head) joined: 256 threads = 256 / HD runs of splits x HD dims
template <int HD>
__global__ void __launch_bounds__(256) paged_join_kernel(const float *parts, const float *stats, int splits, uint16_t *y) {
  constexpr int RUNS = 256 / HD;
  __shared__ float s_w[kMaxSplits], s_o[RUNS][HD], s_m[4], s_l[4];
  const int64_t at = blockIdx.x;
  const int tid = threadIdx.x, d = tid % HD, run = tid / HD;
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
  float sum = 0.f;
  for (int s = run; s < splits; s += RUNS) sum += s_w[s] * parts[(at * splits + s) * HD + d];
  s_o[run][d] = sum;
  __syncthreads();
  if (run == 0) {
#pragma unroll
    for (int i = 1; i < RUNS; ++i) sum += s_o[i][d];
    const float total = (s_l[0] + s_l[1]) + (s_l[2] + s_l[3]);
    y[at * HD + d] = (uint16_t)(pack_bf16x2(total != 0.f ? sum / total : 0.f, 0.f) & 0xFFFFu);
  }
}

constexpr int kWaves = 4;

// How many splits: enough workgroups to fill the 256 compute units several times over, so that sequences of different lengths
// even out, with at least 256 tokens of the longest possible sequence in each.
int splits_of(int64_t B, int kv_heads, int groups, int64_t cap) {
  const int64_t units = std::max<int64_t>(1, B * kv_heads * groups);
  return (int)std::max<int64_t>(1, std::min<int64_t>({(1024 + units - 1) / units, (cap + 255) / 256, kMaxSplits}));
}

template <int HD, bool Q4>
void launch(const DecodeArgs &A, const KVPages &P, int64_t B, hipStream_t s) {
  const size_t lds = (size_t)kWaves * 16 * (HD + 2) * sizeof(float);
  hipLaunchKernelGGL((paged_attention_kernel<HD, Q4, kWaves>), dim3((unsigned)(B * P.kv_heads * A.groups * A.splits)),
                     dim3(kWaves * 64), lds, s, A, P);
  if (A.splits > 1)
    hipLaunchKernelGGL((paged_join_kernel<HD>), dim3((unsigned)(B * A.H)), dim3(256), 0, s, A.parts, A.stats, A.splits, A.y);
}

}  // namespace
}  // namespace smlm

extern "C" int64_t smlm_paged_attention_workspace(int64_t B, int H, int kv_heads, int head_dim, int page_size,
                                                  int64_t max_pages) {
  using namespace smlm;
  if (B <= 0 || B > 0x7FFFFFFF || H < 1 || H > 65536 || kv_heads < 1 || head_dim < 1 || page_size < 1 || max_pages < 1 || max_pages > 0x7FFFFFFF ||
      H % kv_heads)
    return 0;
  const int splits = splits_of(B, kv_heads, (H / kv_heads + 15) / 16, max_pages * page_size);
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
  if (!(scale > 0.f) || scale > 3e38f) return fail(SMLM_EINVAL, "%s: the scale must be positive and finite", name);
  if (max_pages * pages->page_size > 0x7FFFFF00LL)
    return fail(SMLM_EUNSUPPORTED, "%s: a block table of %lld pages is more than 2^31 tokens", name, (long long)max_pages);
  const int G = H / pages->kv_heads, groups = (G + 15) / 16;
  const int splits = splits_of(B, pages->kv_heads, groups, max_pages * pages->page_size);
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
  if (hd == 32) q4 ? launch<32, true>(A, P, B, s) : launch<32, false>(A, P, B, s);
  else if (hd == 64) q4 ? launch<64, true>(A, P, B, s) : launch<64, false>(A, P, B, s);
  else q4 ? launch<128, true>(A, P, B, s) : launch<128, false>(A, P, B, s);
  return launch_status(name);
}
