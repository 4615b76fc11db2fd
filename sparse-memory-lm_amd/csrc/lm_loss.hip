// The language model's loss over its vocabulary, from the hidden states and the output embedding, with its gradient
// (F.cross_entropy(lm_head(x).float(), targets) of smlm/model.py:286-293), without ever holding the logits:
//   s_n = x_n W^T, loss_n = logsumexp(s_n) - s_n[t_n], dx = G W, dW = G^T x, G = c_n (softmax(s_n) - 1[t_n]).
//
// Forward: a workgroup takes up to 256 tokens and a range of the vocabulary, forms 256 columns of logits at a time in its
// accumulators and keeps a running maximum and sum of exponentials per lane, each lane over its own columns (no exchange
// between lanes until the range ends).  The (maximum, sum) of every range go to a small array, which a second kernel joins,
// one wavefront per token; the target's logit is picked from the accumulators, so that it is the very value in the sum.
// A third launch adds the tokens' losses up (in fp64, in a fixed order).  Only lse (fp32 per token) is kept.
//
// Gradient, in pieces of the vocabulary: the logits of a piece again, G of the piece as bf16 (of up to 128 tokens as two
// bf16 terms; c_n is 0 or 1 where the loss is a mean or sum, so that G needs no scale: 1 / count goes on at the end), then
// its two products (lm_mm.hip): dW's rows of the piece are final, dx gathers over the pieces in fp32.
//
// Bound by the products: 2 M V d operations forward, three times that in the gradient (one third for the logits again, which
// is what not keeping them costs).  With d = 384 a tile's sum is short, six units of 64 k, and 128 exponentials a lane follow
// it: the stages of successive tiles run through one pipeline, so that a tile's first loads are on their way during its
// predecessor's exponentials.  Measured (d = 384, V = 50,304): 16,384 tokens 600 to 640 us forward (1,030 TFLOP/s; d = 1,024
// reaches 1,240), in the gradient 900 to 980 for G (its 1.65 GB are written in whole 64-byte lines, which do not overlap its
// products: 65 us of each 412 MB), 640 to 720 for dx, 590 to 630 for dW.  64 tokens of 32,000 are bound by W's bytes and the
// launches: 60 us for all.
#include "lm_mm.h"

#include <algorithm>

namespace smlm {
namespace {

constexpr int kLsCols = 256;                              // vocabulary columns per tile
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kLsFinishRows = 4;                          // tokens per workgroup of the joining kernel, one a wavefront
constexpr int64_t kLsPieceBytes = 1LL << 30;            // most bytes of one piece's G
constexpr int kNoTarget = -0x40000000;

typedef uint16_t __attribute__((may_alias)) Overlaid;     // a value stored over a part of a wider store, behind it

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

struct LossArgs {
  const uint16_t *x, *w;
  int64_t ldx, ldw, M, d, v0, v1, V;                      // vocabulary columns [v0, v1) of V
  const int64_t *targets;
  int64_t ignore;
  int nsplit, tiles;                                      // ranges of the vocabulary, and its tiles of columns
  float2 *parts;                                          // forward: (maximum, sum) to base 2, [M][nsplit][wavefronts over a tile]
  float *picked;                                          // forward: the target's logit [M]
  const float *lse, *coef, *grad, *count;                 // gradient: coef per token, or null; grad and count: see below
  float *scale;                                           // gradient: *grad / *count (count null: *grad), written here
  uint16_t *g;                                            // gradient: G of the piece [M][ldg]
  int64_t ldg, rest;                                      // where G's second term is, elements on, or 0 (mm_terms)
};

// Eight wavefronts, 256 columns: of 256 tokens, each wavefront 128 x 64 (fewer tokens a lane: fewer running maxima), of 128 or
// 64, each 64 x 64 or 64 x 32.
typedef MmShape<2, 4, 8, 4> Tokens256;
typedef MmShape<4, 2, 4, 4> Tokens128;
typedef MmShape<4, 2, 4, 2> Tokens64;

template <class S>
struct LossKernel {
  typedef MmTile<S::kF, true, true, S::kThreads, 64> F;
  typedef MmTile<S::kT, true, false, S::kThreads, 64> T;
  typedef MmLoop<F, T, S::NI, S::NJ> Loop;
};

template <class S, bool GRAD>
__global__ void __launch_bounds__(S::kThreads, 2) loss_kernel(LossArgs a) {
  static_assert(S::kF == kLsCols, "columns");
  constexpr int NI = S::NI, NJ = S::NJ, C = 4 * NI;       // C columns of a token per lane
  typedef typename LossKernel<S>::F FT;
  typedef typename LossKernel<S>::T TT;
  typedef typename LossKernel<S>::Loop Loop;
  extern __shared__ __align__(16) unsigned char smem[];
  const unsigned nt = (unsigned)((a.M + S::kT - 1) / S::kT);
  if (GRAD && blockIdx.x == 0 && threadIdx.x == 0 && a.grad)   // for the products that follow
    *a.scale = a.count ? (*a.count > 0.f ? *a.grad / *a.count : 0.f) : *a.grad;
  const int unit = mm_tile_of(blockIdx.x, nt * a.nsplit);
  if (unit < 0) return;  // workgroup-uniform
  // the token tiles of one range are neighbours: an XCD reads its ranges of W from memory once
  const int split = unit / nt;
  const int64_t t0 = (int64_t)(unit - split * nt) * S::kT;
  const int first = (int)((int64_t)a.tiles * split / a.nsplit), last = (int)((int64_t)a.tiles * (split + 1) / a.nsplit);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), wf = S::feature(wave), wt = S::token(wave);
  const int lane = threadIdx.x % kWave, r = lane & 15, g = lane >> 4;

  // the targets' columns in [v0, ..) wait in LDS (registers are short); kNoTarget: not in this piece or none
  int *targets = (int *)(smem + Loop::kLds);
  if (threadIdx.x < S::kT) {
    const int64_t t = t0 + threadIdx.x, y = t < a.M ? a.targets[t] : a.ignore;
    targets[threadIdx.x] = y != a.ignore && y >= a.v0 && y < a.v1 ? (int)(y - a.v0) : kNoTarget;
  }
  float m[NJ], l[NJ];                 // forward: running maximum and sum; gradient: m = lse
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int64_t t = t0 + wt + 16 * j + r;
    m[j] = GRAD ? __builtin_inff() : -__builtin_inff();   // gradient, an ignored token: every probability is 0
    l[j] = 0.f;
    if (GRAD && t < a.M) {
      // an index outside the vocabulary makes its token's gradient NaN, as its loss
      const int64_t y = a.targets[t];
      if (y != a.ignore) m[j] = y < 0 || y >= a.V ? __builtin_nanf("") : a.lse[t];
    }
  }

  Loop L;
  L.init(smem, a.ldw, a.ldx, wf, wt);
  // the loads run two stages ahead of the products, over the ends of tiles (past the last tile they load what is not used)
  const int units = mm_units(a.d);
  int ahead_tile = first, ahead = 0;
  MmSource<FT> fs;
  MmSource<TT> ts;
  auto begin_tile = [&]() {
    fs.init(a.w, a.ldw, a.V, a.d, a.v0 + (int64_t)ahead_tile * kLsCols, 0);
    ts.init(a.x, a.ldx, a.M, a.d, t0, 0);
    if (a.d % kMmUnit) L.offsets(a.ldw, a.ldx);          // the last stage's clipped them
    ahead = 0;
  };
  auto loaded = [&]() {
    if (++ahead == units) {
      ++ahead_tile;
      begin_tile();
    }
  };
  floatx4 acc[NI][NJ];
  typename Loop::Frags x, y;
  uint32_t stage = 0;
  begin_tile();
  if (first < last) {
    L.issue(fs, ts, 0);
    loaded();
    L.issue(fs, ts, Loop::kStage);
    loaded();
    mm_wait_barrier<Loop::kLoads>();
    L.read(x, 0, 0);
  }
  for (int tile = first; tile < last; ++tile) {
    mm_zero(acc);
    for (int u = 0; u < units; ++u) {
      L.multiply(fs, ts, x, y, stage, acc);
      loaded();
    }

    // lane (r, g): columns c0 + 32 (q / 8) + q % 8, q < C, of token r of each 16
    const int c0 = tile * kLsCols + wf + 8 * g;
    const int64_t end = (GRAD ? a.v1 : a.V) - a.v0;
    if ((int64_t)(tile + 1) * kLsCols > end) {          // columns past the end count for nothing
      const int valid = (int)(end - c0);
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][e] = 32 * (i / 2) + 4 * (i % 2) + e < valid ? acc[i][j][e] : -__builtin_inff();
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      // the target's q in this lane, if it is here
      const int off = targets[wt + 16 * j + r] - c0;
      const unsigned rel = (unsigned)off < 8u * NI * 2 && (off & 24) == 0 ? (unsigned)(off / 32 * 8 + off % 8) : ~0u;
      if constexpr (!GRAD) {
        if (__any(rel < (unsigned)C)) {                   // rare: 16 NI of the vocabulary's columns for 16 tokens
          float v = 0.f;
#pragma unroll
          for (int q = 0; q < C; ++q) v = rel == (unsigned)q ? acc[q / 4][j][q % 4] : v;
          if (rel < (unsigned)C) a.picked[t0 + wt + (unsigned)(16 * j + r)] = v;
        }
        float top = -__builtin_inff();
#pragma unroll
        for (int q = 0; q < C; ++q) top = fmaxf(top, acc[q / 4][j][q % 4]);
        // to base 2: the sum is of 2^(s log2(e) - m), m the maximum times log2(e) as rounded, which makes its rounding no error
        // (one fma per exponent)
        top = fmaxf(m[j], top * kLog2e);
        const float ref = top == -__builtin_inff() ? 0.f : top;   // nothing yet: every exponential is 0
        float sum = l[j] * exp2_hw(m[j] - ref), more = 0.f;
#pragma unroll
        for (int q = 0; q < C; q += 2) {
          sum += exp2_hw(fmaf(acc[q / 4][j][q % 4], kLog2e, -ref));
          more += exp2_hw(fmaf(acc[q / 4][j][q % 4 + 1], kLog2e, -ref));
        }
        m[j] = top;
        l[j] = sum + more;
      } else {
        const int64_t t = t0 + wt + 16 * j + r;
        float p[C];
#pragma unroll
        for (int q = 0; q < C; ++q) p[q] = exp2_hw((acc[q / 4][j][q % 4] - m[j]) * kLog2e);
        float c = 1.f;
        if (a.coef) {                                     // uniform
          c = t < a.M ? a.coef[t] : 0.f;
#pragma unroll
          for (int q = 0; q < C; ++q) p[q] = p[q] == 0.f ? 0.f : p[q] * c;   // (an ignored token's coefficient may be NaN)
        }
        if (t < a.M) {
          // a wave-uniform base and 32 bits a lane
          char *out = (char *)(a.g + (t0 + wt + 16 * j) * a.ldg + tile * kLsCols + wf);
          const uint32_t at = (uint32_t)(r * a.ldg + 8 * g) * 2;
#pragma unroll
          for (int q = 0; q < C / 8; ++q) *(uint4 *)(out + (at + 64 * q)) = mm_pack(p + 8 * q);
          if (a.rest) {                                   // uniform
#pragma unroll
            for (int q = 0; q < C; ++q) p[q] = mm_rest(p[q]);
#pragma unroll
            for (int q = 0; q < C / 8; ++q) *(uint4 *)(out + 2 * a.rest + (at + 64 * q)) = mm_pack(p + 8 * q);
          }
        }
        if (__any(rel < (unsigned)C)) {                   // rare: the target's, over what its lane has just stored
          float v = 0.f;
#pragma unroll
          for (int q = 0; q < C; ++q) v = rel == (unsigned)q ? acc[q / 4][j][q % 4] : v;
          v = (exp2_hw((v - m[j]) * kLog2e) - 1.f) * c;
          if (rel < (unsigned)C) {
            const float rest = mm_rest(v);
            Overlaid *to = (Overlaid *)(a.g + t * a.ldg + c0 + off);
            *to = (uint16_t)(pack_bf16x2(v, v) & 0xFFFFu);
            if (a.rest) to[a.rest] = (uint16_t)(pack_bf16x2(rest, rest) & 0xFFFFu);
          }
        }
      }
    }
  }

  mm_finish();
  if constexpr (!GRAD) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
#pragma unroll
      for (int o = 16; o <= 32; o *= 2) {
        const float m2 = __shfl_xor(m[j], o, kWave), l2 = __shfl_xor(l[j], o, kWave);
        const float top = fmaxf(m[j], m2), ref = top == -__builtin_inff() ? 0.f : top;
        l[j] = l[j] * exp2_hw(m[j] - ref) + l2 * exp2_hw(m2 - ref);
        m[j] = top;
      }
      const int64_t t = t0 + wt + 16 * j + r;
      if (g == 0 && t < a.M) a.parts[(t * a.nsplit + split) * S::WF + wave % S::WF] = make_float2(m[j], l[j]);
    }
  }
}

// Joins the ranges of kLsFinishRows tokens: lse, and the losses (each) or their sum and number (sums, counts).  64 tokens
// have 500 parts each: eight loads a lane in flight, 6 us (one after the other, four tokens a wavefront: 14 us).
__global__ void __launch_bounds__(256)
    loss_join_kernel(const float2 *__restrict__ parts, int nparts, const float *__restrict__ picked,
                     const int64_t *__restrict__ targets, int64_t ignore, int64_t M, int64_t V, float *__restrict__ lse,
                     float *__restrict__ each, double *__restrict__ sums) {
  __shared__ double sum[kLsFinishRows];
  __shared__ int num[kLsFinishRows];
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const int64_t t = (int64_t)blockIdx.x * kLsFinishRows + wave;
  double total = 0.0;
  int count = 0;
  if (t < M) {  // wave-uniform
    const int64_t y = targets[t];
    const bool valid = y != ignore && y >= 0 && y < V;
    const float s = valid ? picked[t] : 0.f;
    float m = -__builtin_inff(), l = 0.f;
    for (int p0 = 0; p0 < nparts; p0 += 8 * kWave) {
      float2 v[8];
      float top = m;
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const int p = p0 + q * kWave + lane;
        v[q] = p < nparts ? parts[t * nparts + p] : make_float2(-__builtin_inff(), 0.f);
      }
#pragma unroll
      for (int q = 0; q < 8; ++q) top = fmaxf(top, v[q].x);
      const float ref = top == -__builtin_inff() ? 0.f : top;
      l *= exp2_hw(m - ref);
#pragma unroll
      for (int q = 0; q < 8; ++q) l += v[q].y * exp2_hw(v[q].x - ref);
      m = top;
    }
    for (int o = 32; o > 0; o >>= 1) {
      const float m2 = __shfl_xor(m, o, kWave), l2 = __shfl_xor(l, o, kWave);
      const float top = fmaxf(m, m2), ref = top == -__builtin_inff() ? 0.f : top;
      l = l * exp2_hw(m - ref) + l2 * exp2_hw(m2 - ref);
      m = top;
    }
    // loss = (m + log2(l) - s log2(e)) / log2(e), the large terms first: m and s log2(e) cancel without a rounding of
    // their size, so that it does not fall below 0 by more than the logarithm's own rounding; lse = s + loss, so that a
    // certain token's probability is exactly 1 in the gradient (s may be -inf, lse is finite then)
    const float log2l = log2f(l);
    float loss = 0.f, z = (m + log2l) * kLn2;
    if (valid) {
      loss = (fmaf(-s, kLog2e, m) + log2l) * kLn2;
      loss = loss < 0.f ? 0.f : loss;
      z = s == -__builtin_inff() ? z : s + loss;
    } else if (y != ignore) {
      loss = __builtin_nanf("");
    }
    if (lane == 0) {
      lse[t] = z;
      if (each) each[t] = loss;
    }
    total = loss;
    count = y != ignore;
  }
  if (!sums) return;  // workgroup-uniform
  if (lane == 0) {
    sum[wave] = total;
    num[wave] = count;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    sums[2 * (int64_t)blockIdx.x] = sum[0] + sum[1] + sum[2] + sum[3];
    sums[2 * (int64_t)blockIdx.x + 1] = num[0] + num[1] + num[2] + num[3];
  }
}

// The loss, and the number of tokens that count.
__global__ void __launch_bounds__(1024)
    loss_sum_kernel(const double *__restrict__ sums, int64_t n, int mean, float *loss, float *count) {
  __shared__ double s[2][16];
  double v[2] = {0.0, 0.0};
  for (int64_t i = threadIdx.x; i < n; i += 4 * 1024) {
    double2 u[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) u[q] = i + q * 1024 < n ? ((const double2 *)sums)[i + q * 1024] : make_double2(0.0, 0.0);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      v[0] += u[q].x;
      v[1] += u[q].y;
    }
  }
  for (int o = 32; o > 0; o >>= 1)
    for (int q = 0; q < 2; ++q) v[q] += __shfl_xor(v[q], o, kWave);
  if (threadIdx.x % kWave == 0)
    for (int q = 0; q < 2; ++q) s[q][threadIdx.x / kWave] = v[q];
  __syncthreads();
  if (threadIdx.x == 0) {
    double a = 0.0, b = 0.0;
    for (int i = 0; i < 16; ++i) {
      a += s[0][i];
      b += s[1][i];
    }
    *loss = (float)(mean ? a / b : a);  // no token counts: NaN, as F.cross_entropy
    *count = (float)b;
  }
}

template <class S, bool GRAD>
int launch_loss(LossArgs a, hipStream_t stream, const char *what) {
  constexpr int kLds = LossKernel<S>::Loop::kLds + S::kT * 4;
  static std::atomic<uint64_t> done;
  if (const int rc = mm_allow_lds((const void *)loss_kernel<S, GRAD>, kLds, done, what)) return rc;
  const int64_t n = ceil_div(a.M, S::kT) * a.nsplit;
  if (mm_grid(n) > 0x7FFFFFFFLL) return fail(SMLM_EUNSUPPORTED, "%s: too many workgroups", what);
  hipLaunchKernelGGL((loss_kernel<S, GRAD>), dim3((unsigned)mm_grid(n)), dim3(S::kThreads), kLds, stream, a);
  return launch_status(what);
}

// Tokens of a tile, and its wavefronts over the columns (each leaves its own maximum and sum).  Two smaller tiles beat one
// half empty, as the ranges are short then (32,000 x 384, forward and gradient of x): 128 tokens 40 us in tiles of 64, 45
// of 128, 52 of 256; 200 tokens 52, 50 and 59; 300 tokens 66, 65 and 64; 1,000 tokens 137, 118 and 111.
int tile_tokens(int64_t M) { return M > 256 ? 256 : M > 128 ? 128 : 64; }
int tile_parts(int64_t M) { return M > 256 ? Tokens256::WF : Tokens128::WF; }

template <bool GRAD>
int dispatch_loss(const LossArgs &a, hipStream_t stream, const char *what) {
  switch (tile_tokens(a.M)) {
    case 256: return launch_loss<Tokens256, GRAD>(a, stream, what);
    case 128: return launch_loss<Tokens128, GRAD>(a, stream, what);
    default: return launch_loss<Tokens64, GRAD>(a, stream, what);
  }
}

// Ranges of `tiles` vocabulary tiles: one workgroup for each CU, all of them at once on the card.
int range_count(int64_t M, int64_t tiles) {
  const int64_t nt = ceil_div(M, tile_tokens(M));
  return (int)std::min<int64_t>(tiles, std::max<int64_t>(1, 256 / nt));
}
int64_t part_count(int64_t M, int64_t V) { return (int64_t)tile_parts(M) * range_count(M, ceil_div(V, kLsCols)); }

struct GradPlan {
  int64_t cols, pieces, g_bytes, part_bytes;
  MmPlan dx, dw;
};
GradPlan grad_plan(int64_t M, int64_t V, int64_t d) {
  GradPlan p;
  // at most the products' widest rows: few tokens would have wider ones
  const int64_t row = 2 * M * mm_terms(M);                // bytes of a column of G
  const int64_t most = std::min<int64_t>(kMmMaxStride, std::max<int64_t>(kLsPieceBytes / row / kLsCols, 1) * kLsCols);
  p.pieces = ceil_div(V, most);
  p.cols = ceil_div(ceil_div(V, p.pieces), kLsCols) * kLsCols;
  p.pieces = ceil_div(V, p.cols);
  p.dx = mm_plan(M, d, p.cols, true);
  // Never split over the tokens, so that its rows of bf16 are final: from some 20,000 columns on its tiles fill the card.  Below
  // they do not, and it takes longer than dx, which is split (16,384 tokens, d = 384): 98 us for 22 of 1,000 columns, 185 for
  // 122 of 8,192, 290 for 279 of 20,000.
  p.dw = mm_plan(p.cols, d, M, false);
  p.g_bytes = row * p.cols;
  p.part_bytes = p.pieces * p.dx.splits > 1 ? p.dx.splits * M * d * 4 : 0;
  return p;
}

int check_loss(const char *what, const void *x, int64_t x_stride, const void *w, int64_t w_stride, const void *targets,
               int64_t M, int64_t V, int64_t d) {
  if (!x || !w || !targets) return fail(SMLM_EINVAL, "%s: null x, weight or targets pointer", what);
  if (M < 0 || V < 1 || d < 1)
    return fail(SMLM_EINVAL, "%s: bad shape M=%lld V=%lld d=%lld", what, (long long)M, (long long)V, (long long)d);
  if (d % 8) return fail(SMLM_EUNSUPPORTED, "%s: d=%lld must be a multiple of 8", what, (long long)d);
  if (V > (1 << 30) || d > (1 << 20) || M > (1 << 30) || M > (1LL << 36) / d)
    return fail(SMLM_EUNSUPPORTED, "%s: M=%lld V=%lld d=%lld too large", what, (long long)M, (long long)V, (long long)d);
  // the lanes' 32-bit byte offsets span 256 rows
  if (x_stride < d || w_stride < d || x_stride % 8 || w_stride % 8 || x_stride > kMmMaxStride || w_stride > kMmMaxStride ||
      ((uintptr_t)x | (uintptr_t)w) % 16 || (uintptr_t)targets % 8)
    return fail(SMLM_EINVAL, "%s: rows must be 16-byte aligned with strides from their widths to 2^21 elements (x %lld, "
                "weight %lld)", what, (long long)x_stride, (long long)w_stride);
  return SMLM_OK;
}

}  // namespace
}  // namespace smlm

extern "C" int64_t smlm_linear_ce_workspace(int64_t M, int64_t V, int64_t d, int grad) {
  using namespace smlm;
  if (M < 1 || V < 1 || d < 1) return 0;
  if (grad) {
    const GradPlan p = grad_plan(M, V, d);
    return 256 + p.g_bytes + p.part_bytes;
  }
  // (maximum, sum) of every range, the picked logits, and the partial sums of the losses
  return M * part_count(M, V) * 8 + 8 + ceil_div(M, 4) * 16 + ceil_div(M, kLsFinishRows) * 16;
}

extern "C" int smlm_linear_ce(const void *x, int64_t x_row_stride, const void *w, int64_t w_row_stride,
                              const int64_t *targets, int64_t ignore_index, int reduction, int64_t M, int64_t V, int64_t d,
                              float *loss, float *count, float *lse, void *workspace, int64_t workspace_bytes, void *stream) {
  using namespace smlm;
  const char *what = "smlm_linear_ce";
  if (const int rc = check_loss(what, x, x_row_stride, w, w_row_stride, targets, M, V, d)) return rc;
  if (!loss || !lse || (!count && reduction != SMLM_REDUCE_NONE))
    return fail(SMLM_EINVAL, "%s: null loss, count or lse pointer", what);
  if (reduction < SMLM_REDUCE_NONE || reduction > SMLM_REDUCE_SUM)
    return fail(SMLM_EINVAL, "%s: unknown reduction %d", what, reduction);
  if (M == 0) return reduction == SMLM_REDUCE_NONE ? SMLM_OK : fail(SMLM_EINVAL, "%s: nothing to reduce", what);
  if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < smlm_linear_ce_workspace(M, V, d, 0))
    return fail(SMLM_EINVAL, "%s: the workspace needs %lld bytes, 16-byte aligned", what,
                (long long)smlm_linear_ce_workspace(M, V, d, 0));
  hipStream_t s = (hipStream_t)stream;
  LossArgs a{};
  a.x = (const uint16_t *)x;
  a.w = (const uint16_t *)w;
  a.ldx = x_row_stride;
  a.ldw = w_row_stride;
  a.M = M;
  a.d = d;
  a.v0 = 0;
  a.v1 = a.V = V;
  a.targets = targets;
  a.ignore = ignore_index;
  a.tiles = (int)ceil_div(V, kLsCols);
  a.nsplit = range_count(M, a.tiles);
  char *ws = (char *)workspace;
  a.parts = (float2 *)ws;
  ws += (M * part_count(M, V) * 8 + 15) / 16 * 16;
  a.picked = (float *)ws;
  double *sums = reduction == SMLM_REDUCE_NONE ? nullptr : (double *)(ws + ceil_div(M, 4) * 16);
  if (const int rc = dispatch_loss<false>(a, s, what)) return rc;
  const int64_t blocks = ceil_div(M, kLsFinishRows);
  if (blocks > 0x7FFFFFFFLL) return fail(SMLM_EUNSUPPORTED, "%s: M=%lld too large", what, (long long)M);
  hipLaunchKernelGGL(loss_join_kernel, dim3((unsigned)blocks), dim3(256), 0, s, a.parts, (int)part_count(M, V), a.picked, targets,
                     ignore_index, M, V, lse, reduction == SMLM_REDUCE_NONE ? loss : nullptr, sums);
  if (const int rc = launch_status(what)) return rc;
  if (!sums) return SMLM_OK;
  hipLaunchKernelGGL(loss_sum_kernel, dim3(1), dim3(1024), 0, s, sums, blocks, reduction == SMLM_REDUCE_MEAN ? 1 : 0, loss,
                     count);
  return launch_status(what);
}

extern "C" int smlm_linear_ce_backward(const float *grad, const float *count, int per_token, const void *x,
                                       int64_t x_row_stride, const void *w, int64_t w_row_stride, const int64_t *targets,
                                       int64_t ignore_index, const float *lse, int64_t M, int64_t V, int64_t d, void *dx,
                                       void *dw, void *workspace, int64_t workspace_bytes, void *stream) {
  using namespace smlm;
  const char *what = "smlm_linear_ce_backward";
  if (const int rc = check_loss(what, x, x_row_stride, w, w_row_stride, targets, M, V, d)) return rc;
  if (!grad || !lse || (!dx && !dw)) return fail(SMLM_EINVAL, "%s: null grad, lse or gradient pointers", what);
  if (((uintptr_t)dx | (uintptr_t)dw) % 16) return fail(SMLM_EINVAL, "%s: dx and dw must be 16-byte aligned", what);
  if (M < 1) return fail(SMLM_EINVAL, "%s: no tokens", what);
  if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < smlm_linear_ce_workspace(M, V, d, 1))
    return fail(SMLM_EINVAL, "%s: the workspace needs %lld bytes, 16-byte aligned", what,
                (long long)smlm_linear_ce_workspace(M, V, d, 1));
  hipStream_t s = (hipStream_t)stream;
  const GradPlan p = grad_plan(M, V, d);
  LossArgs a{};
  a.x = (const uint16_t *)x;
  a.w = (const uint16_t *)w;
  a.ldx = x_row_stride;
  a.ldw = w_row_stride;
  a.M = M;
  a.d = d;
  a.V = V;
  a.targets = targets;
  a.ignore = ignore_index;
  a.lse = lse;
  a.coef = per_token ? grad : nullptr;
  a.grad = per_token ? nullptr : grad;
  a.count = count;
  a.scale = (float *)workspace;
  a.g = (uint16_t *)((char *)workspace + 256);
  a.ldg = p.cols;
  a.rest = mm_terms(M) > 1 ? M * p.cols : 0;
  float *parts = (float *)((char *)workspace + 256 + p.g_bytes);
  const float *scale = per_token ? nullptr : a.scale;
  for (int64_t piece = 0; piece < p.pieces; ++piece) {
    a.v0 = piece * p.cols;
    a.v1 = std::min(V, a.v0 + p.cols);
    const int64_t n = a.v1 - a.v0;
    a.tiles = (int)ceil_div(n, kLsCols);
    a.nsplit = range_count(M, a.tiles);
    if (const int rc = dispatch_loss<true>(a, s, what)) return rc;
    if (dx) {   // the sum over the piece's columns
      MmArgs m{};
      m.feat = a.w + a.v0 * a.ldw;
      m.ldf = a.ldw;
      m.Kf = n;
      m.tok = a.g;
      m.ldt = a.ldg;
      m.tok_rest = a.rest;
      m.F = d;
      m.T = M;
      m.K = (n + 7) / 8 * 8;
      m.f32 = p.part_bytes > 0;
      m.out = m.f32 ? (void *)parts : dx;
      m.ldo = d;
      m.scale = scale;
      m.accumulate = piece > 0;
      if (const int rc = mm_launch(m, false, true, p.dx, s, what)) return rc;
    }
    if (dw) {   // the sum over the tokens
      MmArgs m{};
      m.feat = a.x;
      m.ldf = a.ldx;
      m.Kf = m.K = M;
      m.tok = a.g;
      m.ldt = a.ldg;
      m.tok_rest = a.rest;
      m.F = d;
      m.T = n;
      m.out = (uint16_t *)dw + a.v0 * d;
      m.ldo = d;
      m.scale = scale;
      if (const int rc = mm_launch(m, false, false, p.dw, s, what)) return rc;
    }
  }
  if (dx && p.part_bytes > 0) return mm_reduce_launch(parts, p.dx.splits, M, d, scale, dx, d, s, what);
  return SMLM_OK;
}
