// Plain products of a training step's gradients (lm_mm.h): one tile per workgroup, k split over workgroups where the
// tiles alone are too few (a weight's gradient: few outputs, many tokens), the parts added in order by a second kernel (the
// same bits on every call).
#include "lm_mm.h"

#include <algorithm>

namespace smlm {
namespace {

template <int NI, int NJ, bool FKC, bool TKC, bool F32>
__global__ void __launch_bounds__(kMmThreads, 2) mm_kernel(MmArgs a) {
  typedef MmTile<32 * NI, FKC, FKC ? 4 * NI : 0> FT;
  typedef MmTile<32 * NJ, TKC, 0> TT;
  typedef MmLoop<FT, TT, NI, NJ> Loop;
  extern __shared__ __align__(16) unsigned char smem[];
  const unsigned nf = (unsigned)((a.F + FT::kRows - 1) / FT::kRows), nt = (unsigned)((a.T + TT::kRows - 1) / TT::kRows);
  const int tile = mm_tile_of(blockIdx.x, nf * nt * (unsigned)a.nsplit);   // the host has checked that they are this few
  if (tile < 0) return;  // workgroup-uniform
  // the feature tiles of one token tile are neighbours: on one XCD its rows come from memory once
  const unsigned row = tile / nf, split = row / nt;
  const int64_t f0 = (int64_t)(tile - row * nf) * FT::kRows, t0 = (int64_t)(row - split * nt) * TT::kRows, s = split;
  const int64_t k_begin = s * a.k_per, k_end = min(a.K, k_begin + a.k_per);
  const int wave = threadIdx.x / kWave, wf = (wave & 1) * 16 * NI, wt = (wave >> 1) * 16 * NJ;
  Loop L;
  L.init(smem, a.ldf, a.ldt, wf, wt);
  floatx4 acc[NI][NJ];
  mm_zero(acc);
  MmSource<FT> fs;
  MmSource<TT> ts;
  fs.init(a.feat, a.ldf, a.F, FKC ? a.K : a.Kf, f0, k_begin);
  ts.init(a.tok, a.ldt, TKC ? a.T : (a.T + 7) & ~7LL, a.K, t0, k_begin);
  if (k_end > k_begin) {  // workgroup-uniform; k_end is K or a whole number of double chunks on
    typename Loop::Frags x, y;
    L.start(fs, ts, x);
    uint32_t stage = 0;
    for (int left = mm_chunks(k_end - k_begin); left > 0; left -= 2) {
      L.step(fs, ts, x, y, stage, acc);
      L.step(fs, ts, y, x, stage, acc);
    }
    __builtin_amdgcn_s_waitcnt(0x0F70);  // no load is on its way into LDS when the workgroup ends
  }

  // lane (r, g): features 4 NI g .. (permuted) or 4 g .. of each 16, of token r of each 16
  const int lane = threadIdx.x % kWave, r = lane & 15, g = lane >> 4;
  const float scale = !F32 && a.scale ? *a.scale : 1.0f;
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int64_t t = t0 + wt + 16 * j + r;
    if (t >= a.T) continue;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int64_t f = f0 + wf + (FKC ? 4 * NI * g + 4 * i : 16 * i + 4 * g);
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
        *(uint2 *)((uint16_t *)a.out + t * a.ldo + f) =
            uint2{pack_bf16x2(v[0] * scale, v[1] * scale), pack_bf16x2(v[2] * scale, v[3] * scale)};
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

template <int NI, int NJ, bool FKC, bool TKC>
int launch(const MmArgs &a, hipStream_t stream, const char *what) {
  typedef MmLoop<MmTile<32 * NI, FKC, FKC ? 4 * NI : 0>, MmTile<32 * NJ, TKC, 0>, NI, NJ> Loop;
  constexpr int kLds = kMmStages * Loop::kStage;
  const int64_t n = ceil_div(a.F, 32 * NI) * ceil_div(a.T, 32 * NJ) * a.nsplit;
  if (mm_grid(n) > 0x7FFFFFFFLL) return fail(SMLM_EUNSUPPORTED, "%s: too many workgroups", what);
  const void *k = a.f32 ? (const void *)mm_kernel<NI, NJ, FKC, TKC, true> : (const void *)mm_kernel<NI, NJ, FKC, TKC, false>;
  const hipError_t e = hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
  if (e != hipSuccess) return fail(SMLM_EHIP, "%s: %s", what, hipGetErrorString(e));
  const dim3 grid((unsigned)mm_grid(n)), block(kMmThreads);
  if (a.f32) hipLaunchKernelGGL((mm_kernel<NI, NJ, FKC, TKC, true>), grid, block, kLds, stream, a);
  else hipLaunchKernelGGL((mm_kernel<NI, NJ, FKC, TKC, false>), grid, block, kLds, stream, a);
  return launch_status(what);
}

// Largest tile of which there are enough for the 256 CUs.
template <bool FKC, bool TKC>
int choose(const MmArgs &a, hipStream_t stream, const char *what) {
  const int64_t big = ceil_div(a.F, 128) * a.nsplit;
  if (big * ceil_div(a.T, 256) >= 384) return launch<4, 8, FKC, TKC>(a, stream, what);
  if (big * ceil_div(a.T, 128) >= 256) return launch<4, 4, FKC, TKC>(a, stream, what);
  return launch<2, 2, FKC, TKC>(a, stream, what);
}

}  // namespace

int mm_launch(const MmArgs &a, bool feat_kc, bool tok_kc, hipStream_t stream, const char *what) {
  if (feat_kc && tok_kc) return choose<true, true>(a, stream, what);
  if (tok_kc) return choose<false, true>(a, stream, what);
  return choose<false, false>(a, stream, what);   // feat_kc without tok_kc: no caller
}

int64_t mm_splits(int64_t T, int64_t F, int64_t K, int64_t min_k) {
  const int64_t tiles = ceil_div(F, 128) * ceil_div(T, 128), most = std::max<int64_t>(1, K / min_k);
  return std::min(most, std::max<int64_t>(1, 512 / tiles));
}

int64_t mm_k_per(int64_t K, int64_t nsplit) { return ceil_div(ceil_div(K, nsplit), 2 * kMmK) * 2 * kMmK; }

int mm_reduce_launch(const float *parts, int64_t nsplit, int64_t T, int64_t F, const float *scale, void *out, int64_t ldo,
                     hipStream_t stream, const char *what) {
  const int64_t blocks = ceil_div(T * F / 4, 256);
  if (blocks > 0x7FFFFFFFLL) return fail(SMLM_EUNSUPPORTED, "%s: too many workgroups", what);
  hipLaunchKernelGGL(mm_reduce_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, parts, nsplit, T, F, scale,
                     (uint16_t *)out, ldo);
  return launch_status(what);
}

}  // namespace smlm
