// The gated feed-forward block of a recorded pass and its gradients (SwiGLU.forward, smlm/model.py:110-118, and what
// autograd derives from it):
//   a | b = x w13^T, s = sigmoid(a), act = a s b, y = act w2^T
//   dact = dy w2, da = dact b (s + a s (1 - s)), db = dact a s, dx = [da | db] w13, dw13 = [da | db]^T x, dw2 = dy^T act
//
// Only the inputs are kept for the gradient: a and b are formed again there, in the launch that forms dact, so that the
// gate's derivative is taken on fp32 accumulators and neither the projection nor dact touches memory.  (Keeping a | b
// would save a quarter of the gradient's first launch, and cost 4 hidden bytes a token written and read, and a rounding.)
//   gate_kernel       x w13^T and the activation: tiles of 64 a- and 64 b-rows, so that a lane holds matching a and b
//   gate_grad_kernel  the same, then dy w2 on the same tokens and features: writes act and [da | db] in bf16
//   mm_kernel         y, dx, dw13, dw2 (lm_mm.hip); the weights' sums over the tokens are split over workgroups
// Bound by the products: 6 M d hidden operations forward, 16 in the gradient.  The gradient's first launch has 32
// features x 64 tokens per wavefront and operand and is held by its LDS reads (14 KB per 24 products of 16 x 16 x 32).
#include "lm_mm.h"

#include <algorithm>

namespace smlm {
namespace {

constexpr int kGateFeat = 64;                             // features per tile: 64 rows of a and 64 of b
constexpr float kLog2e = 1.4426950408889634f;

struct GateArgs {
  const uint16_t *x, *w13, *dy, *w2;
  int64_t ldx, ldw13, lddy, ldw2, M, d, hidden, n_out;
  uint16_t *act, *dab;                                    // [M][hidden], [M][2 hidden]
};

__device__ __forceinline__ float sigmoid(float a) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-a * kLog2e));
}

template <int NJ, bool GRAD>
__global__ void __launch_bounds__(kMmThreads, 2) gate_kernel(GateArgs p) {
  typedef MmTile<2 * kGateFeat, true, 8> FT;              // rows of w13: 64 of a, then 64 of b
  typedef MmTile<kGateFeat, false, 8> ST;                 // columns of w2
  typedef MmTile<32 * NJ, true, 0> TT;
  typedef MmLoop<FT, TT, 4, NJ> Gate;
  typedef MmLoop<ST, TT, 2, NJ> Out;
  constexpr uint32_t kStage = Gate::kStage;               // the larger of the two
  extern __shared__ __align__(16) unsigned char smem[];
  const unsigned nf = (unsigned)((p.hidden + kGateFeat - 1) / kGateFeat), nt = (unsigned)((p.M + TT::kRows - 1) / TT::kRows);
  const int tile = mm_tile_of(blockIdx.x, nf * nt);
  if (tile < 0) return;  // workgroup-uniform
  // the feature tiles of a token tile are neighbours: on one XCD its rows are read from memory once
  const unsigned row = tile / nf;
  const int64_t f0 = (int64_t)(tile - row * nf) * kGateFeat, t0 = (int64_t)row * TT::kRows;
  const int wave = threadIdx.x / kWave, wf = (wave & 1) * 32, wt = (wave >> 1) * 16 * NJ;
  const int lane = threadIdx.x % kWave, r = lane & 15, g = lane >> 4;

  Gate A;
  A.init(smem, p.ldw13, p.ldx, wf, wt);
#pragma unroll
  for (int i = 0; i < 2; ++i) A.fa[2 + i] = A.fa[i] + kGateFeat * FT::kRowBytes;   // b's rows: the same swizzle
  Out B;
  if constexpr (GRAD) B.init(smem, p.ldw2, p.lddy, wf, wt);
  const int n1 = mm_chunks(p.d), n2 = GRAD ? mm_chunks(p.n_out) : 0;
  // rows of a beyond hidden are b's, whose results are not stored; rows of b beyond the weight read as zeros
  MmSource<FT> as, bs;
  MmSource<TT> xs, ys;
  MmSource<ST> ss;
  as.init(p.w13, p.ldw13, 2 * p.hidden, p.d, f0, 0);
  bs.init(p.w13, p.ldw13, 2 * p.hidden, p.d, p.hidden + f0 - kGateFeat, 0);   // load 1 adds 64 rows
  xs.init(p.x, p.ldx, p.M, p.d, t0, 0);
  if constexpr (GRAD) {
    ss.init(p.w2, p.ldw2, p.hidden, p.n_out, f0, 0);
    ys.init(p.dy, p.lddy, p.M, p.n_out, t0, 0);
  }
  floatx4 ab[4][NJ], dact[2][NJ];
  mm_zero(ab);
  mm_zero(dact);
  uint32_t stage = 0;
  auto advance = [&]() {
    const uint32_t here = stage;
    stage = stage == 2 * kStage ? 0 : stage + kStage;
    return here;
  };
  // Loads of the next chunk, of x w13^T or (OUT) of dy w2, part i of `parts`.
  struct Chunk {
    intx4 a, b, t;
  };
  auto next_gate = [&]() {
    Gate::template clip<FT>(as, A.fo);
    Gate::template clip<TT>(xs, A.to);
    const Chunk c{as.rsrc(), bs.rsrc(), xs.rsrc()};
    as.next();
    bs.next();
    xs.next();
    return c;
  };
  auto next_out = [&]() {
    Out::template clip<TT>(ys, B.to);
    const Chunk c{ss.rsrc(), ss.rsrc(), ys.rsrc()};
    ss.next();
    ys.next();
    return c;
  };
  auto load_gate = [&](const Chunk &c, uint32_t at, int i, int parts) {
#pragma unroll
    for (int l = 0; l < Gate::kLoads; ++l)
      if (l >= i * Gate::kLoads / parts && l < (i + 1) * Gate::kLoads / parts)
        mm_load_lds(l == 0 ? c.a : l == 1 ? c.b : c.t, l < 2 ? A.fo[l] : A.to[l - 2], A.lds + at + l * 4096);
  };
  auto load_out = [&](const Chunk &c, uint32_t at, int i, int parts) {
#pragma unroll
    for (int l = 0; l < Out::kLoads; ++l)
      if (l >= i * Out::kLoads / parts && l < (i + 1) * Out::kLoads / parts) B.load(l, c.a, c.t, at);
  };

  // Steps of x w13^T: loading a chunk of the same, or (the last three) of dy w2.
  auto step = [&](const typename Gate::Frags &cur, typename Gate::Frags &next) {
    const uint32_t here = advance();
    const Chunk c = next_gate();
    Gate::products(cur, ab, [&](int i) { load_gate(c, here, i, 4); }, [&](int i) { A.read_part(next, stage, i); });
  };
  auto step_to_out = [&](const typename Gate::Frags &cur, typename Gate::Frags &next) {
    const uint32_t here = advance();
    const Chunk c = next_out();
    Gate::products(cur, ab, [&](int i) { load_out(c, here, i, 4); }, [&](int i) { A.read_part(next, stage, i); });
  };
  typename Gate::Frags x, y;
  load_gate(next_gate(), 0, 0, 1);
  load_gate(next_gate(), kStage, 0, 1);
  int left = n1;                          // chunks of x w13^T not yet multiplied, an even number
  if constexpr (GRAD) {
    if (n1 > 2) {
      load_gate(next_gate(), 2 * kStage, 0, 1);
      mm_wait_barrier<2 * Gate::kLoads>();
    } else {
      load_out(next_out(), 2 * kStage, 0, 1);
      mm_wait_barrier<Gate::kLoads + Out::kLoads>();
    }
    A.read(x, 0);
    for (; left > 4; left -= 2) {
      mm_wait_barrier<Gate::kLoads>();
      step(x, y);
      mm_wait_barrier<Gate::kLoads>();
      step(y, x);
    }
    if (left > 2) {
      mm_wait_barrier<Gate::kLoads>();
      step(x, y);
      mm_wait_barrier<Gate::kLoads>();
      step_to_out(y, x);
    }
    mm_wait_barrier<Out::kLoads>();
    step_to_out(x, y);
    mm_wait_barrier<Out::kLoads>();       // what step_to_out reads ahead now is the next sum's, and not used
    step_to_out(y, x);
    typename Out::Frags u, v;
    B.read(u, stage);                     // the first chunk of dy w2, landed by the barrier before
    auto out_step = [&](const typename Out::Frags &cur, typename Out::Frags &next) {
      mm_wait_barrier<Out::kLoads>();
      const uint32_t here = advance();
      const Chunk c = next_out();
      Out::products(cur, dact, [&](int i) { load_out(c, here, i, 2); }, [&](int i) { B.read_part(next, stage, i); });
    };
    for (int more = n2; more > 0; more -= 2) {
      out_step(u, v);
      out_step(v, u);
    }
  } else {
    load_gate(next_gate(), 2 * kStage, 0, 1);
    mm_wait_barrier<2 * Gate::kLoads>();
    A.read(x, 0);
    for (; left > 0; left -= 2) {
      mm_wait_barrier<Gate::kLoads>();
      step(x, y);
      mm_wait_barrier<Gate::kLoads>();
      step(y, x);
    }
  }
  __builtin_amdgcn_s_waitcnt(0x0F70);     // no load is on its way into LDS when the workgroup ends

  // lane (r, g): features f .. f + 7 of token r of each 16
  const int64_t f = f0 + wf + 8 * g;
  if (f >= p.hidden) return;                              // hidden is a multiple of 8
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int64_t t = t0 + wt + 16 * j + r;
    if (t >= p.M) continue;
    float h[8], da[8], db[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const float a = ab[q / 4][j][q % 4], b = ab[2 + q / 4][j][q % 4], s = sigmoid(a), as = a * s;
      h[q] = as * b;
      if constexpr (GRAD) {
        const float dh = dact[q / 4][j][q % 4];
        da[q] = dh * b * (s + as * (1.f - s));
        db[q] = dh * as;
      }
    }
    auto store = [&](uint16_t *o, const float *v) {
      *(uint4 *)o = uint4{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
    };
    store(p.act + t * p.hidden + f, h);
    if constexpr (GRAD) {
      store(p.dab + t * 2 * p.hidden + f, da);
      store(p.dab + t * 2 * p.hidden + p.hidden + f, db);
    }
  }
}

template <int NJ, bool GRAD>
int launch_gate(const GateArgs &p, hipStream_t stream, const char *what) {
  constexpr int kLds = kMmStages * (2 * kGateFeat + 32 * NJ) * kMmK * 2;
  const hipError_t e = hipFuncSetAttribute((const void *)gate_kernel<NJ, GRAD>, hipFuncAttributeMaxDynamicSharedMemorySize,
                                           kLds);
  if (e != hipSuccess) return fail(SMLM_EHIP, "%s: %s", what, hipGetErrorString(e));
  const int64_t n = ceil_div(p.hidden, kGateFeat) * ceil_div(p.M, 32 * NJ);
  if (mm_grid(n) > 0x7FFFFFFFLL) return fail(SMLM_EUNSUPPORTED, "%s: too many workgroups", what);
  hipLaunchKernelGGL((gate_kernel<NJ, GRAD>), dim3((unsigned)mm_grid(n)), dim3(kMmThreads), kLds, stream, p);
  return launch_status(what);
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
      (1 << 22) || ((uintptr_t)x | (uintptr_t)w13 | (uintptr_t)w2) % 16)
    return fail(SMLM_EINVAL, "%s: rows must be 16-byte aligned with strides from their widths to 2^22 elements (x %lld, "
                "w13 %lld, w2 %lld)", what, (long long)ldx, (long long)ldw13, (long long)ldw2);
  return SMLM_OK;
}

// out [T][F] = sum over k of tok[k][T] feat[k][F], k split over workgroups
struct WeightGrad {
  int64_t T, F, K, splits;
  int64_t bytes() const { return splits > 1 ? splits * T * F * 4 : 0; }
};
WeightGrad weight_grad(int64_t T, int64_t F, int64_t K) { return {T, F, K, mm_splits(T, F, K, 256)}; }

int run_weight_grad(const WeightGrad &g, const void *tok, int64_t ldt, const void *feat, int64_t ldf, float *parts, void *out,
                    hipStream_t s, const char *what) {
  MmArgs m{};
  m.feat = (const uint16_t *)feat;
  m.tok = (const uint16_t *)tok;
  m.ldf = ldf;
  m.ldt = ldt;
  m.F = g.F;
  m.T = g.T;
  m.K = m.Kf = g.K;
  m.f32 = g.splits > 1;
  m.out = m.f32 ? (void *)parts : out;
  m.ldo = g.F;
  m.nsplit = g.splits;
  m.k_per = mm_k_per(g.K, g.splits);
  if (const int rc = mm_launch(m, false, false, s, what)) return rc;
  return m.f32 ? mm_reduce_launch(parts, g.splits, g.T, g.F, nullptr, out, g.F, s, what) : SMLM_OK;
}

}  // namespace
}  // namespace smlm

extern "C" int smlm_gated_ffn(const void *x, int64_t x_row_stride, const void *w13, int64_t w13_row_stride, const void *w2,
                              int64_t w2_row_stride, int64_t M, int64_t d, int64_t hidden, int64_t n_out, void *act, void *y,
                              void *stream) {
  using namespace smlm;
  const char *what = "smlm_gated_ffn";
  if (const int rc = check_ffn(what, x, x_row_stride, w13, w13_row_stride, w2, w2_row_stride, M, d, hidden, n_out)) return rc;
  if (!act || !y || ((uintptr_t)act | (uintptr_t)y) % 16)
    return fail(SMLM_EINVAL, "%s: act and y must be 16-byte aligned tensors", what);
  if (M == 0) return SMLM_OK;
  hipStream_t s = (hipStream_t)stream;
  GateArgs p{};
  p.x = (const uint16_t *)x;
  p.w13 = (const uint16_t *)w13;
  p.ldx = x_row_stride;
  p.ldw13 = w13_row_stride;
  p.M = M;
  p.d = d;
  p.hidden = hidden;
  p.act = (uint16_t *)act;
  const int64_t nf = ceil_div(hidden, kGateFeat);
  const int rc = nf * ceil_div(M, 256) >= 384 ? launch_gate<8, false>(p, s, what)
                 : nf * ceil_div(M, 128) >= 256 ? launch_gate<4, false>(p, s, what)
                                                : launch_gate<2, false>(p, s, what);
  if (rc) return rc;
  MmArgs m{};
  m.feat = (const uint16_t *)w2;
  m.ldf = w2_row_stride;
  m.tok = p.act;
  m.ldt = hidden;
  m.F = n_out;
  m.T = M;
  m.K = m.Kf = hidden;
  m.out = y;
  m.ldo = n_out;
  m.nsplit = 1;
  m.k_per = mm_k_per(hidden, 1);
  return mm_launch(m, true, true, s, what);
}

extern "C" int64_t smlm_gated_ffn_workspace(int64_t M, int64_t d, int64_t hidden, int64_t n_out) {
  using namespace smlm;
  if (M < 1 || d < 1 || hidden < 1 || n_out < 1) return 0;
  return M * hidden * 6 + std::max(weight_grad(2 * hidden, d, M).bytes(), weight_grad(n_out, hidden, M).bytes());
}

extern "C" int smlm_gated_ffn_backward(const void *dy, int64_t dy_row_stride, const void *x, int64_t x_row_stride,
                                       const void *w13, int64_t w13_row_stride, const void *w2, int64_t w2_row_stride,
                                       int64_t M, int64_t d, int64_t hidden, int64_t n_out, void *dx, void *dw13, void *dw2,
                                       void *workspace, int64_t workspace_bytes, void *stream) {
  using namespace smlm;
  const char *what = "smlm_gated_ffn_backward";
  if (const int rc = check_ffn(what, x, x_row_stride, w13, w13_row_stride, w2, w2_row_stride, M, d, hidden, n_out)) return rc;
  if (!dy || dy_row_stride < n_out || dy_row_stride % 8 || dy_row_stride > (1 << 22) || (uintptr_t)dy % 16)
    return fail(SMLM_EINVAL, "%s: dy must have 16-byte aligned rows with a stride from %lld to 2^22 elements", what,
                (long long)n_out);
  if ((!dx && !dw13 && !dw2) || ((uintptr_t)dx | (uintptr_t)dw13 | (uintptr_t)dw2) % 16)
    return fail(SMLM_EINVAL, "%s: dx, dw13 and dw2 must be 16-byte aligned, one of them at least given", what);
  if (M < 1) return fail(SMLM_EINVAL, "%s: no tokens", what);
  if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < smlm_gated_ffn_workspace(M, d, hidden, n_out))
    return fail(SMLM_EINVAL, "%s: the workspace needs %lld bytes, 16-byte aligned", what,
                (long long)smlm_gated_ffn_workspace(M, d, hidden, n_out));
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
  p.dab = p.act + M * hidden;
  float *parts = (float *)(p.dab + 2 * M * hidden);
  const int64_t nf = ceil_div(hidden, kGateFeat);
  if (const int rc = nf * ceil_div(M, 128) >= 256 ? launch_gate<4, true>(p, s, what) : launch_gate<2, true>(p, s, what))
    return rc;
  if (dx) {
    MmArgs m{};
    m.feat = p.w13;
    m.ldf = p.ldw13;
    m.tok = p.dab;
    m.ldt = 2 * hidden;
    m.F = d;
    m.T = M;
    m.K = m.Kf = 2 * hidden;
    m.out = dx;
    m.ldo = d;
    m.nsplit = 1;
    m.k_per = mm_k_per(m.K, 1);
    if (const int rc = mm_launch(m, false, true, s, what)) return rc;
  }
  if (dw13)
    if (const int rc = run_weight_grad(weight_grad(2 * hidden, d, M), p.dab, 2 * hidden, x, x_row_stride, parts, dw13, s, what))
      return rc;
  if (dw2) return run_weight_grad(weight_grad(n_out, hidden, M), dy, dy_row_stride, p.act, hidden, parts, dw2, s, what);
  return SMLM_OK;
}
