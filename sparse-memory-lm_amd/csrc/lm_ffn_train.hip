// The gated feed-forward block of a recorded pass and its gradients (SwiGLU.forward, smlm/model.py:110-118, and what
// autograd derives from it):
//   a | b = x w13^T, s = sigmoid(a), act = a s b, y = act w2^T
//   dact = dy w2, da = dact b (s + a s (1 - s)), db = dact a s, dx = [da | db] w13, dw13 = [da | db]^T x, dw2 = dy^T act
//
// Only the inputs are kept for the gradient: a and b are formed again there, in the launch that forms dact, so that the
// gate's derivative is taken on fp32 accumulators and neither the projection nor dact touches memory.  (Keeping a | b
// would save a quarter of the gradient's first launch, and cost 4 hidden bytes a token written and read, and a rounding.)
//   gate_kernel   x w13^T and the activation; each lane holds matching a and b.  For the gradient (GRAD) dy w2 on the
//                 same tokens and features through the same stages: writes act and [da | db] in bf16
//   mm_kernel     y, dx, dw13, dw2 (lm_mm.hip); the weights' sums over the tokens are split over workgroups
// Bound by the products: 6 M d hidden operations forward, 18 with the recomputed a | b in the gradient; their rate is that of
// the way from cache into LDS (lm_mm.h), and d = 384 of them are only six units of 64 k a tile.  Measured for 32,768 tokens
// of d = 384, hidden 1,024: the gate 63 us (820 TFLOP/s), y 35, the gradient's gate 129 (its three results are 201 MB, and
// take 60 us of it: they do not overlap its products), dx 61, dw13 51, dw2 48 and the joining of their parts 14.
#include "lm_mm.h"

#include <algorithm>

namespace smlm {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

struct GateArgs {
  const uint16_t *x, *w13, *dy, *w2;
  int64_t ldx, ldw13, lddy, ldw2, M, d, hidden, n_out;
  uint16_t *act, *dab;                                    // [M][hidden], [M][2 hidden]
  int64_t rest;                                           // M hidden: act's second term is so many on, dab's twice; or 0
};

__device__ __forceinline__ float sigmoid(float a) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-a * kLog2e));
}

// A tile takes S::kF rows of w13: half of them a's, and b's for the same features; each wavefront 8 NI features of either.
template <class S>
struct GateKernel {
  static constexpr int kFeat = S::kF / 2, kHalf = S::NI / 2;   // features of a tile, row groups of either half
  typedef MmTile<S::kF, true, true, S::kThreads, 64> F;        // rows of w13
  typedef MmTile<kFeat, false, true, S::kThreads, 64> W2;      // columns of w2
  typedef MmTile<S::kT, true, false, S::kThreads, 64> T;
  typedef MmLoop<F, T, S::NI, S::NJ> Gate;
  typedef MmLoop<W2, T, kHalf, S::NJ> Out;
};

template <class S, bool GRAD>
__global__ void __launch_bounds__(S::kThreads, 2) gate_kernel(GateArgs p) {
  typedef GateKernel<S> K;
  typedef typename K::Gate Gate;
  typedef typename K::Out Out;
  constexpr int NI = S::NI, NJ = S::NJ, kHalf = K::kHalf;
  constexpr uint32_t kStage = Gate::kStage;               // the larger of the two
  extern __shared__ __align__(16) unsigned char smem[];
  const unsigned nf = (unsigned)((p.hidden + K::kFeat - 1) / K::kFeat), nt = (unsigned)((p.M + S::kT - 1) / S::kT);
  const int tile = mm_tile_of(blockIdx.x, nf * nt);
  if (tile < 0) return;  // workgroup-uniform
  // the feature tiles of a token tile are neighbours: on one XCD its rows are read from memory once
  const unsigned row = tile / nf;
  const int64_t f0 = (int64_t)(tile - row * nf) * K::kFeat, t0 = (int64_t)row * S::kT;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), wf = S::feature(wave) / 2, wt = S::token(wave);
  const int lane = threadIdx.x % kWave, r = lane & 15, g = lane >> 4;

  Gate A;
  A.init(smem, p.ldw13, p.ldx, wf, wt);
  Out B;
  if constexpr (GRAD) B.init(smem, p.ldw2, p.lddy, wf, wt);
  // rows of a beyond hidden are b's, whose results are not stored; rows of b beyond the weight read as zeros
  MmSource<typename K::F> as, bs;
  MmSource<typename K::T> xs, ys;
  MmSource<typename K::W2> ss;
  as.init(p.w13, p.ldw13, 2 * p.hidden, p.d, f0, 0);
  bs.init(p.w13, p.ldw13, 2 * p.hidden, p.d, p.hidden + f0 - K::kFeat, 0);   // its loads are those of rows kFeat on
  xs.init(p.x, p.ldx, p.M, p.d, t0, 0);
  if constexpr (GRAD) {
    ss.init(p.w2, p.ldw2, p.hidden, p.n_out, f0, 0);
    ys.init(p.dy, p.lddy, p.M, p.n_out, t0, 0);
  }
  // The loads of the next stage of x w13^T or dy w2 to `at`, part i of `parts`; then the sources step on.
  auto load_gate = [&](uint32_t at, int i, int parts) {
    constexpr int kF = K::F::kLoads;
#pragma unroll
    for (int l = 0; l < Gate::kLoads; ++l)
      if (l >= i * Gate::kLoads / parts && l < (i + 1) * Gate::kLoads / parts) {
        if (l < kF / 2) Gate::load_one(as, A.fo, l, A.lds + at);
        else if (l < kF) Gate::load_one(bs, A.fo, l, A.lds + at);
        else Gate::load_one(xs, A.to, l - kF, A.lds + at + K::F::kBytes);
      }
  };
  auto clip_gate = [&]() {
    Gate::clip(as, A.fo);
    Gate::clip(xs, A.to);
  };
  auto next_gate = [&]() {
    as.next();
    bs.next();
    xs.next();
  };
  auto load_out = [&](uint32_t at, int i, int parts) {
#pragma unroll
    for (int l = 0; l < Out::kLoads; ++l)
      if (l >= i * Out::kLoads / parts && l < (i + 1) * Out::kLoads / parts) B.load(l, ss, ys, at);
  };
  // fragments of a in the first half of the row groups, of b (kFeat rows on, the same swizzle) in the second
  auto read_gate = [&](typename Gate::Frags &x, uint32_t stage, int h, int i) {
    x.a[i] = K::F::frag(A.fa, i % kHalf, h, stage + (i < kHalf ? 0 : K::kFeat * K::F::kRowBytes));
#pragma unroll
    for (int j = 0; j < NJ; ++j)
      if (j >= i * NJ / NI && j < (i + 1) * NJ / NI) x.b[j] = K::T::frag(A.ta, j, h, stage);
  };

  floatx4 ab[NI][NJ], dact[kHalf][NJ];
  mm_zero(ab);
  mm_zero(dact);
  typename Gate::Frags x, y;
  const int n1 = mm_units(p.d), n2 = GRAD ? mm_units(p.n_out) : 0;
  clip_gate();
  load_gate(0, 0, 1);
  next_gate();
  if (!GRAD || n1 > 1) {                                  // uniform
    clip_gate();
    load_gate(kStage, 0, 1);
    next_gate();
    mm_wait_barrier<Gate::kLoads>();
  } else {
    B.issue(ss, ys, kStage);
    mm_wait_barrier<Out::kLoads>();
  }
#pragma unroll
  for (int i = 0; i < NI; ++i) read_gate(x, 0, 0, i);
  uint32_t stage = 0;
  for (int left = n1; left > 0; --left) {
    const uint32_t here = stage;
    stage = kStage - stage;
    Gate::products(x, ab, [&](int i) { read_gate(y, here, 1, i); });
    mm_wait_barrier<0>();                                 // the next stage has landed, all have read this one
    if (!GRAD || left > 2) {
      clip_gate();
      Gate::products(y, ab, [&](int i) {
        load_gate(here, i, NI);
        read_gate(x, stage, 0, i);
      });
      next_gate();
    } else {                                              // the last two stages' places take dy w2's first two
      Out::clip(ys, B.to);
      Gate::products(y, ab, [&](int i) {
        load_out(here, i, NI);
        if (left > 1) read_gate(x, stage, 0, i);
      });
      ss.next();
      ys.next();
    }
  }
  if constexpr (GRAD) {
    typename Out::Frags u, v;
    B.read(u, stage, 0);                                  // landed by the last barrier
    for (int left = n2; left > 0; --left) {
      const uint32_t here = stage;
      stage = kStage - stage;
      Out::products(u, dact, [&](int i) { B.read_part(v, here, 1, i); });
      mm_wait_barrier<0>();
      Out::clip(ys, B.to);
      Out::products(v, dact, [&](int i) {
        load_out(here, i, kHalf);
        B.read_part(u, stage, 0, i);
      });
      ss.next();
      ys.next();
    }
  }
  mm_finish();

  // lane (r, g): 8 features from f + 32 p on, p < kHalf / 2, of token r of each 16
  const int64_t f = f0 + wf + 8 * g;
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int64_t t = t0 + wt + 16 * j + r;
    if (t >= p.M) continue;
#pragma unroll
    for (int o = 0; o < 16 * kHalf; o += 32) {
      if (f + o >= p.hidden) continue;                    // hidden is a multiple of 8
      float h[8], da[8], db[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const int i = o / 16 + q / 4, e = q % 4;
        const float a = ab[i][j][e], b = ab[kHalf + i][j][e], s = sigmoid(a), as = a * s;
        h[q] = as * b;
        if constexpr (GRAD) {
          const float dh = dact[i][j][e];
          da[q] = dh * b * (s + as * (1.f - s));
          db[q] = dh * as;
        }
      }
      auto store = [&](uint16_t *to, float *v, int64_t rest) {
        *(uint4 *)to = mm_pack(v);
        if (p.rest) {                                     // uniform
#pragma unroll
          for (int q = 0; q < 8; ++q) v[q] = mm_rest(v[q]);
          *(uint4 *)(to + rest) = mm_pack(v);
        }
      };
      store(p.act + t * p.hidden + f + o, h, p.rest);
      if constexpr (GRAD) {
        store(p.dab + t * 2 * p.hidden + f + o, da, 2 * p.rest);
        store(p.dab + t * 2 * p.hidden + p.hidden + f + o, db, 2 * p.rest);
      }
    }
  }
}

typedef MmShape<2, 4, 8, 4> Gate256;                     // 128 features x 256 tokens
typedef MmShape<4, 2, 4, 4> Gate128;                     // 128 x 128
typedef MmShape<2, 2, 4, 2> Gate64;                      // 64 x 64, four wavefronts

template <class S, bool GRAD>
int launch_gate(const GateArgs &p, hipStream_t stream, const char *what) {
  constexpr int kLds = GateKernel<S>::Gate::kLds;
  static std::atomic<uint64_t> done;
  if (const int rc = mm_allow_lds((const void *)gate_kernel<S, GRAD>, kLds, done, what)) return rc;
  const int64_t n = ceil_div(p.hidden, GateKernel<S>::kFeat) * ceil_div(p.M, S::kT);
  if (mm_grid(n) > 0x7FFFFFFFLL) return fail(SMLM_EUNSUPPORTED, "%s: too many workgroups", what);
  hipLaunchKernelGGL((gate_kernel<S, GRAD>), dim3((unsigned)mm_grid(n)), dim3(S::kThreads), kLds, stream, p);
  return launch_status(what);
}

// The largest tile of which there is one for each CU at least (d = 384, hidden = 1,024; forward with its y product, the
// gradient with dw2's): 32,768 tokens take 90 us in Gate256, 100 in Gate128, 107 in Gate64; the gradient 174 in Gate128,
// 194 in Gate64 (in Gate256 its registers do not suffice); 1,024 tokens 22, 17 and 14, the gradient 25 and 21.
template <bool GRAD>
int dispatch_gate(const GateArgs &p, hipStream_t stream, const char *what) {
  const int64_t n128 = ceil_div(p.hidden, 128);
  if constexpr (!GRAD)
    if (n128 * ceil_div(p.M, 256) >= 256) return launch_gate<Gate256, GRAD>(p, stream, what);
  if (n128 * ceil_div(p.M, 128) >= 256) return launch_gate<Gate128, GRAD>(p, stream, what);
  return launch_gate<Gate64, GRAD>(p, stream, what);
}

int check_ffn(const char *what, const void *x, int64_t ldx, const void *w13, int64_t ldw13, const void *w2, int64_t ldw2,
              int64_t M, int64_t d, int64_t hidden, int64_t n_out) {
  if (!x || !w13 || !w2) return fail(SMLM_EINVAL, "%s: null x, w13 or w2 pointer", what);
  if (M < 0 || d < 1 || hidden < 1 || n_out < 1)
    return fail(SMLM_EINVAL, "%s: bad shape M=%lld d=%lld hidden=%lld n_out=%lld", what, (long long)M, (long long)d,
                (long long)hidden, (long long)n_out);
  if (d % 8 || hidden % 8 || n_out % 8)
    return fail(SMLM_EUNSUPPORTED, "%s: d=%lld, hidden=%lld and n_out=%lld must be multiples of 8", what, (long long)d,
                (long long)hidden, (long long)n_out);
  const int64_t widest = std::max(std::max(d, 2 * hidden), n_out);
  if (widest > (1 << 20) || M > (1LL << 36) / widest)
    return fail(SMLM_EUNSUPPORTED, "%s: M=%lld d=%lld hidden=%lld n_out=%lld too large", what, (long long)M, (long long)d,
                (long long)hidden, (long long)n_out);
  if (ldx < d || ldw13 < d || ldw2 < hidden || ldx % 8 || ldw13 % 8 || ldw2 % 8 || std::max(std::max(ldx, ldw13), ldw2) >
      kMmMaxStride || ((uintptr_t)x | (uintptr_t)w13 | (uintptr_t)w2) % 16)
    return fail(SMLM_EINVAL, "%s: rows must be 16-byte aligned with strides from their widths to 2^21 elements (x %lld, "
                "w13 %lld, w2 %lld)", what, (long long)ldx, (long long)ldw13, (long long)ldw2);
  return SMLM_OK;
}

// The products besides the gate's: y over hidden, dx over a and b, the weights' gradients over the tokens.
struct FfnPlan {
  MmPlan y, dx, dw13, dw2;
  int64_t act, parts_forward, parts_backward;             // bytes; da and db take twice act's
};
FfnPlan ffn_plan(int64_t M, int64_t d, int64_t hidden, int64_t n_out) {
  FfnPlan p;
  const int terms = mm_terms(M);
  p.y = mm_plan(M, n_out, hidden * terms, true);
  p.dx = mm_plan(M, d, 2 * hidden * terms, true);
  p.dw13 = mm_plan(2 * hidden, d, M * terms, true);
  p.dw2 = mm_plan(n_out, hidden, M * terms, true);
  p.act = M * hidden * 2 * mm_terms(M);
  p.parts_forward = p.y.part_bytes(M, n_out);
  p.parts_backward = std::max(p.dx.part_bytes(M, d), std::max(p.dw13.part_bytes(2 * hidden, d), p.dw2.part_bytes(n_out, hidden)));
  return p;
}

// out [T][F] = sum over k of tok feat, contiguous
MmArgs product(const void *feat, int64_t ldf, int64_t feat_rest, const void *tok, int64_t ldt, int64_t tok_rest, int64_t F,
               int64_t T, int64_t K, void *out) {
  MmArgs m{};
  m.feat_rest = feat_rest;
  m.tok_rest = tok_rest;
  m.feat = (const uint16_t *)feat;
  m.tok = (const uint16_t *)tok;
  m.ldf = ldf;
  m.ldt = ldt;
  m.F = F;
  m.T = T;
  m.K = m.Kf = K;
  m.out = out;
  m.ldo = F;
  return m;
}

}  // namespace
}  // namespace smlm

extern "C" int64_t smlm_gated_ffn_workspace(int64_t M, int64_t d, int64_t hidden, int64_t n_out, int grad) {
  using namespace smlm;
  if (M < 1 || d < 1 || hidden < 1 || n_out < 1) return 0;
  const FfnPlan p = ffn_plan(M, d, hidden, n_out);
  return grad ? 3 * p.act + p.parts_backward : p.act + p.parts_forward;
}

extern "C" int smlm_gated_ffn(const void *x, int64_t x_row_stride, const void *w13, int64_t w13_row_stride, const void *w2,
                              int64_t w2_row_stride, int64_t M, int64_t d, int64_t hidden, int64_t n_out, void *y,
                              void *workspace, int64_t workspace_bytes, void *stream) {
  using namespace smlm;
  const char *what = "smlm_gated_ffn";
  if (const int rc = check_ffn(what, x, x_row_stride, w13, w13_row_stride, w2, w2_row_stride, M, d, hidden, n_out)) return rc;
  if (!y || (uintptr_t)y % 16) return fail(SMLM_EINVAL, "%s: y must be a 16-byte aligned tensor", what);
  if (M == 0) return SMLM_OK;
  if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < smlm_gated_ffn_workspace(M, d, hidden, n_out, 0))
    return fail(SMLM_EINVAL, "%s: the workspace needs %lld bytes, 16-byte aligned", what,
                (long long)smlm_gated_ffn_workspace(M, d, hidden, n_out, 0));
  hipStream_t s = (hipStream_t)stream;
  GateArgs p{};
  p.x = (const uint16_t *)x;
  p.w13 = (const uint16_t *)w13;
  p.ldx = x_row_stride;
  p.ldw13 = w13_row_stride;
  p.M = M;
  p.d = d;
  p.hidden = hidden;
  p.act = (uint16_t *)workspace;
  p.rest = mm_terms(M) > 1 ? M * hidden : 0;
  const FfnPlan plan = ffn_plan(M, d, hidden, n_out);
  if (const int rc = dispatch_gate<false>(p, s, what)) return rc;
  return mm_run(product(w2, w2_row_stride, 0, p.act, hidden, p.rest, n_out, M, hidden, y), true, true, plan.y,
                (float *)((char *)workspace + plan.act), s, what);
}

extern "C" int smlm_gated_ffn_backward(const void *dy, int64_t dy_row_stride, const void *x, int64_t x_row_stride,
                                       const void *w13, int64_t w13_row_stride, const void *w2, int64_t w2_row_stride,
                                       int64_t M, int64_t d, int64_t hidden, int64_t n_out, void *dx, void *dw13, void *dw2,
                                       void *workspace, int64_t workspace_bytes, void *stream) {
  using namespace smlm;
  const char *what = "smlm_gated_ffn_backward";
  if (const int rc = check_ffn(what, x, x_row_stride, w13, w13_row_stride, w2, w2_row_stride, M, d, hidden, n_out)) return rc;
  if (!dy || dy_row_stride < n_out || dy_row_stride % 8 || dy_row_stride > kMmMaxStride || (uintptr_t)dy % 16)
    return fail(SMLM_EINVAL, "%s: dy must have 16-byte aligned rows with a stride from %lld to 2^21 elements", what,
                (long long)n_out);
  if ((!dx && !dw13 && !dw2) || ((uintptr_t)dx | (uintptr_t)dw13 | (uintptr_t)dw2) % 16)
    return fail(SMLM_EINVAL, "%s: dx, dw13 and dw2 must be 16-byte aligned, one of them at least given", what);
  if (M < 1) return fail(SMLM_EINVAL, "%s: no tokens", what);
  if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < smlm_gated_ffn_workspace(M, d, hidden, n_out, 1))
    return fail(SMLM_EINVAL, "%s: the workspace needs %lld bytes, 16-byte aligned", what,
                (long long)smlm_gated_ffn_workspace(M, d, hidden, n_out, 1));
  hipStream_t s = (hipStream_t)stream;
  GateArgs p{};
  p.x = (const uint16_t *)x;
  p.w13 = (const uint16_t *)w13;
  p.dy = (const uint16_t *)dy;
  p.w2 = (const uint16_t *)w2;
  p.ldx = x_row_stride;
  p.ldw13 = w13_row_stride;
  p.lddy = dy_row_stride;
  p.ldw2 = w2_row_stride;
  p.M = M;
  p.d = d;
  p.hidden = hidden;
  p.n_out = n_out;
  p.act = (uint16_t *)workspace;
  p.rest = mm_terms(M) > 1 ? M * hidden : 0;
  p.dab = p.act + M * hidden * mm_terms(M);
  float *parts = (float *)(p.dab + 2 * M * hidden * mm_terms(M));
  if (const int rc = dispatch_gate<true>(p, s, what)) return rc;
  const FfnPlan plan = ffn_plan(M, d, hidden, n_out);
  if (dx)
    if (const int rc = mm_run(product(w13, w13_row_stride, 0, p.dab, 2 * hidden, 2 * p.rest, d, M, 2 * hidden, dx), false, true,
                              plan.dx, parts, s, what))
      return rc;
  if (dw13)
    if (const int rc = mm_run(product(x, x_row_stride, 0, p.dab, 2 * hidden, 2 * p.rest, d, 2 * hidden, M, dw13), false, false,
                              plan.dw13, parts, s, what))
      return rc;
  if (dw2)
    return mm_run(product(p.act, hidden, p.rest, dy, dy_row_stride, 0, hidden, n_out, M, dw2), false, false, plan.dw2, parts, s,
                  what);
  return SMLM_OK;
}
