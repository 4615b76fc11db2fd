// Plain products of a training step's gradients (lm_mm.h): one tile per workgroup, k split over workgroups where the
// tiles alone are too few (a weight's gradient: few outputs, many tokens), the parts added in order by a second kernel (the
// same bits on every call).
#include "lm_mm.h"

#include <algorithm>

namespace smlm {
namespace {

constexpr int64_t kCus = 256;

typedef MmShape<2, 4, 8, 4> Square;                       // 256 features x 256 tokens, 8 wavefronts
typedef MmShape<4, 2, 6, 4> Wide;                         // 384 x 128, 8 wavefronts
typedef MmShape<2, 2, 4, 4> Small;                        // 128 x 128, 4 wavefronts, two workgroups a CU
typedef MmShape<2, 2, 2, 2> Tiny;                         // 64 x 64, 4 wavefronts, six a CU

template <class S, bool FKC, bool TKC>
struct MmKernel {
  static constexpr bool kPerm = FKC;                      // (k strided features: the transposing reads would conflict)
  // k strided: stages of 32 k, three of them; with 64 the same products took 2 to 10% longer (two stages fit, not three)
  static constexpr int kK = FKC && TKC ? 64 : 32;
  typedef MmTile<S::kF, FKC, kPerm, S::kThreads, kK> F;
  typedef MmTile<S::kT, TKC, false, S::kThreads, kK> T;
  typedef MmLoop<F, T, S::NI, S::NJ> Loop;
  static constexpr int kLds = Loop::kLds;
};

template <class S, bool FKC, bool TKC, bool F32>
__global__ void __launch_bounds__(S::kThreads, 2) mm_kernel(MmArgs a) {
  typedef MmKernel<S, FKC, TKC> K;
  typedef typename K::Loop Loop;
  constexpr int NI = S::NI, NJ = S::NJ;
  extern __shared__ __align__(16) unsigned char smem[];
  const unsigned nf = (unsigned)((a.F + S::kF - 1) / S::kF), nt = (unsigned)((a.T + S::kT - 1) / S::kT);
  const int tile = mm_tile_of(blockIdx.x, nf * nt * (unsigned)a.nsplit);   // the host has checked that they are this few
  if (tile < 0) return;  // workgroup-uniform
  // the feature tiles of one token tile are neighbours: on one XCD its rows come from memory once
  const unsigned row = tile / nf, split = row / nt;
  const int64_t f0 = (int64_t)(tile - row * nf) * S::kF, t0 = (int64_t)(row - split * nt) * S::kT, s = split;
  const int64_t k_begin = s * a.k_per, k_end = min(a.K, k_begin + a.k_per);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), wf = S::feature(wave), wt = S::token(wave);
  Loop L;
  L.init(smem, a.ldf, a.ldt, wf, wt);
  floatx4 acc[NI][NJ];
  mm_zero(acc);
  MmSource<typename K::F> fs;
  MmSource<typename K::T> ts;
  const bool two = a.feat_rest | a.tok_rest;
  for (int term = 0; term <= two; ++term) {               // uniform
    fs.init(a.feat + term * a.feat_rest, a.ldf, a.F, FKC ? a.K : a.Kf, f0, k_begin);
    ts.init(a.tok + term * a.tok_rest, a.ldt, TKC ? a.T : (a.T + 7) & ~7LL, a.K, t0, k_begin);
    if (term) {
      __syncthreads();                                    // all have read the stages
      L.offsets(a.ldf, a.ldt);                            // the last stage's clipped them
    }
    if (k_end > k_begin) {  // workgroup-uniform; k_end is K or a whole number of units on
      typename Loop::Frags x, y;
      L.start(fs, ts, x);
      uint32_t stage = 0;
      for (int left = mm_units(k_end - k_begin); left > 0; --left) L.multiply(fs, ts, x, y, stage, acc);
      mm_finish();
    }
  }

  const int lane = threadIdx.x % kWave, r = lane & 15, g = lane >> 4;
  const float scale = !F32 && a.scale ? *a.scale : 1.0f;
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int64_t t = t0 + wt + 16 * j + r;
    if (t >= a.T) continue;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int64_t f = f0 + wf + mm_feature<K::kPerm>(i, g);
      if (f >= a.F) continue;                 // F is a multiple of 8
      floatx4 v = acc[i][j];
      if constexpr (F32) {
        float4 *o = (float4 *)((float *)a.out + (s * a.T + t) * a.F + f);
        if (a.accumulate) {
          const float4 w = *o;
          v += floatx4{w.x, w.y, w.z, w.w};
        }
        *o = make_float4(v[0], v[1], v[2], v[3]);
      } else {
        auto packed = [&](const floatx4 &u) {
          return uint2{pack_bf16x2(u[0] * scale, u[1] * scale), pack_bf16x2(u[2] * scale, u[3] * scale)};
        };
        uint16_t *o = (uint16_t *)a.out + t * a.ldo + f;
        if constexpr (K::kPerm) {             // with the next row group: 8 features
          const uint2 lo = packed(v), hi = packed(acc[i + 1 < NI ? i + 1 : i][j]);
          if (i % 2 == 0) *(uint4 *)o = uint4{lo.x, lo.y, hi.x, hi.y};
        } else {
          *(uint2 *)o = packed(v);
        }
      }
    }
  }
}

// One thread per 4 outputs.
__global__ void __launch_bounds__(256)
    mm_reduce_kernel(const float *__restrict__ parts, int64_t nsplit, int64_t T, int64_t F, const float *__restrict__ scale,
                     uint16_t *__restrict__ out, int64_t ldo) {
  const int64_t n4 = T * F / 4, i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n4) return;
  const float4 *p = (const float4 *)parts + i;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int64_t s = 0; s < nsplit; s += 8) {
    float4 w[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) w[q] = s + q < nsplit ? p[(s + q) * n4] : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      v.x += w[q].x;
      v.y += w[q].y;
      v.z += w[q].z;
      v.w += w[q].w;
    }
  }
  const float c = scale ? *scale : 1.0f;
  const int64_t t = 4 * i / F, f = 4 * i % F;
  *(uint2 *)(out + t * ldo + f) = uint2{pack_bf16x2(v.x * c, v.y * c), pack_bf16x2(v.z * c, v.w * c)};
}

struct __attribute__((packed, aligned(2))) Piece {
  uint32_t v[4];
};

// One thread per 8 elements of the copy; bound by memory and, for what is padded most often, by its launch.
__global__ void __launch_bounds__(256)
    pad_rows_kernel(const uint16_t *__restrict__ src, int64_t ld, int64_t rows, int64_t cols, uint16_t *__restrict__ dst,
                    int64_t rows_out, int64_t cols_out, int64_t total) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= total) return;
  const int64_t at = i / (cols_out / 8), c = 8 * (i - at * (cols_out / 8)), block = at / rows_out, r = at - block * rows_out;
  const int64_t n = r < rows ? cols - c : 0;
  const uint16_t *p = src + (block * rows + r) * ld + c;
  uint4 v = make_uint4(0, 0, 0, 0);
  if (n >= 8) {
    const Piece w = *(const Piece *)p;
    v = make_uint4(w.v[0], w.v[1], w.v[2], w.v[3]);
  } else if (n > 0) {
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) w[e / 2] |= (uint32_t)p[e] << 16 * (e % 2);
    v = make_uint4(w[0], w[1], w[2], w[3]);
  }
  *(uint4 *)(dst + at * cols_out + c) = v;
}

template <class S, bool FKC, bool TKC>
int launch(const MmArgs &a, hipStream_t stream, const char *what) {
  constexpr int kLds = MmKernel<S, FKC, TKC>::kLds;
  const int64_t n = ceil_div(a.F, S::kF) * ceil_div(a.T, S::kT) * a.nsplit;
  if (mm_grid(n) > 0x7FFFFFFFLL) return fail(SMLM_EUNSUPPORTED, "%s: too many workgroups", what);
  const void *k = a.f32 ? (const void *)mm_kernel<S, FKC, TKC, true> : (const void *)mm_kernel<S, FKC, TKC, false>;
  static std::atomic<uint64_t> done[2];
  if (const int rc = mm_allow_lds(k, kLds, done[a.f32 ? 1 : 0], what)) return rc;
  const dim3 grid((unsigned)mm_grid(n)), block(S::kThreads);
  if (a.f32) hipLaunchKernelGGL((mm_kernel<S, FKC, TKC, true>), grid, block, kLds, stream, a);
  else hipLaunchKernelGGL((mm_kernel<S, FKC, TKC, false>), grid, block, kLds, stream, a);
  return launch_status(what);
}

template <bool FKC, bool TKC>
int choose(const MmArgs &a, int shape, hipStream_t stream, const char *what) {
  switch (shape) {
    case 0: return launch<Square, FKC, TKC>(a, stream, what);
    case 1: return launch<Wide, FKC, TKC>(a, stream, what);
    case 2: return launch<Small, FKC, TKC>(a, stream, what);
    default: return launch<Tiny, FKC, TKC>(a, stream, what);
  }
}

}  // namespace

// The shape and the splits with the least estimated time. The workgroups of a CU share its matrix cores and its way into
// LDS, so a unit of 64 k takes a CU `busy` us for each of its workgroups, and at least `wait` us however few they are (the
// way from memory and the barriers); `fixed` us are the beginning, the end and the launch; the outputs' way to memory, or
// the parts' to memory and back and a second launch, comes on top. The figures are a fit to 54 products of 1 to 50,304
// outputs a side, each timed in every shape with up to 104 splits: the choice is the fastest one or within 5% of it, but
// for one token's row of 384 outputs of k = 32,000 (14.7 us for 12.0); 0.5% slower in the mean. One shape for all:
// 4,096 x 384 outputs of k = 1,024 take 10 us in Tiny, 15 in Small and 23 in Wide; 32,768 x 384 of the same k 46, 37
// and 30; 8,192 x 2,048 of k = 5,632 take 143 in Square, 199 in Small.
MmPlan mm_plan(int64_t T, int64_t F, int64_t K, bool may_split) {
  struct Tile {
    int f, t;
    double wait, busy, fixed;                             // us
  };
  static const Tile tiles[4] = {
      {256, 256, 1.32, 1.50, 5.0}, {384, 128, 1.10, 1.17, 5.7}, {128, 128, 0.64, 0.48, 4.5}, {64, 64, 0.29, 0.23, 3.4}};
  const int64_t units = ceil_div(K, kMmUnit);
  MmPlan best{0, 1};
  double least = 1e30;
  for (int64_t s = 1; s <= (may_split ? 128 : 1) && (s == 1 || units / s >= 4); s += s < 16 ? 1 : 8)
    for (int i = 0; i < 4; ++i) {
      const Tile &c = tiles[i];
      const int64_t per_cu = ceil_div(ceil_div(F, c.f) * ceil_div(T, c.t) * s, kCus);
      double time = ceil_div(units, s) * std::max(c.wait, per_cu * c.busy) + c.fixed;
      time += s > 1 ? 2.4 + s * T * F * 8 / 5.9e6 : T * F * 2 / 3.8e6;
      if (time < least) {
        least = time;
        best = {i, s};
      }
    }
  return best;
}

int mm_launch(MmArgs a, bool feat_kc, bool tok_kc, const MmPlan &plan, hipStream_t stream, const char *what) {
  a.nsplit = plan.splits;
  a.k_per = ceil_div(ceil_div(a.K, plan.splits), kMmUnit) * kMmUnit;
  if (feat_kc && tok_kc) return choose<true, true>(a, plan.shape, stream, what);
  if (tok_kc) return choose<false, true>(a, plan.shape, stream, what);
  if (!feat_kc) return choose<false, false>(a, plan.shape, stream, what);
  return fail(SMLM_EUNSUPPORTED, "%s: no product of contiguous features with strided tokens", what);
}

int mm_run(MmArgs a, bool feat_kc, bool tok_kc, const MmPlan &plan, float *parts, hipStream_t stream, const char *what) {
  void *out = a.out;
  a.f32 = plan.splits > 1;
  if (a.f32) a.out = parts;
  if (const int rc = mm_launch(a, feat_kc, tok_kc, plan, stream, what)) return rc;
  return a.f32 ? mm_reduce_launch(parts, plan.splits, a.T, a.F, a.scale, out, a.ldo, stream, what) : SMLM_OK;
}

int mm_reduce_launch(const float *parts, int64_t nsplit, int64_t T, int64_t F, const float *scale, void *out, int64_t ldo,
                     hipStream_t stream, const char *what) {
  const int64_t blocks = ceil_div(T * F / 4, 256);
  if (blocks > 0x7FFFFFFFLL) return fail(SMLM_EUNSUPPORTED, "%s: too many workgroups", what);
  hipLaunchKernelGGL(mm_reduce_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, parts, nsplit, T, F, scale,
                     (uint16_t *)out, ldo);
  return launch_status(what);
}

}  // namespace smlm

extern "C" int smlm_pad_rows(const void *src, int64_t row_stride, int64_t blocks, int64_t rows, int64_t cols, void *dst,
                             int64_t rows_out, int64_t cols_out, void *stream) {
  using namespace smlm;
  const char *what = "smlm_pad_rows";
  if (!src || !dst) return fail(SMLM_EINVAL, "%s: null pointer argument", what);
  if (blocks < 1 || rows < 0 || cols < 0 || rows_out < rows || cols_out < cols || rows_out < 1 || cols_out < 8 || cols_out % 8 ||
      row_stride < cols || (uintptr_t)dst % 16 || (uintptr_t)src % 2)
    return fail(SMLM_EINVAL, "%s: bad shape, or dst not in 16-byte aligned rows", what);
  if (blocks > (1 << 20) || rows_out > (1LL << 40) || cols_out > (1LL << 30) || rows_out > (1LL << 38) / cols_out / blocks)
    return fail(SMLM_EUNSUPPORTED, "%s: too large", what);
  const int64_t total = blocks * rows_out * (cols_out / 8);
  hipLaunchKernelGGL(pad_rows_kernel, dim3((unsigned)ceil_div(total, 256)), dim3(256), 0, (hipStream_t)stream,
                     (const uint16_t *)src, row_stride, rows, cols, (uint16_t *)dst, rows_out, cols_out, total);
  return launch_status(what);
}
