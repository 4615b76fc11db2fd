// Residual add and RMSNorm of a recorded pass, with their gradient (the norms of smlm/model.py:124-126, 156-163):
//   xs = x + delta (rounded to x's type), h = xs rstd w, rstd = 1 / sqrt(mean(xs^2) + eps)
//   dx = rstd (gw - hat mean(gw hat)) + dxs, gw = dh w, hat = xs rstd;  dw = sum over the rows of dh hat
//
// Bound by memory: forward reads x and delta once and writes xs and h, the gradient reads dxs, dh and xs once and writes dx
// (and ddelta, the same values in delta's type); a row stays in registers between its sum and its result.  A row takes 16,
// 32 or 64 lanes or a workgroup of 128 to 1,024 threads, 8 columns per lane, 16 or 32 bytes a load; rows that are not
// 16-byte aligned (odd widths) use the same loads unaligned, and the last lane of a width that is no multiple of 8 takes
// its last 8 columns, some of them its neighbour's too: both write the same values, and one counts them.  Measured from 200
// to 16,384 columns (21M elements, bf16 delta and h): forward 5.8 to 6.4 TB/s of an fp32 stream, 4.9 to 6.3 of a bf16 one;
// the gradient 3.8 to 5.5 and 3.7 to 5.7 (beyond 8,192 columns 2.6 and 2.2: two steps by 1,024 threads).
// dw: every workgroup walks a contiguous range of rows with its lanes' columns summed in registers, and writes one row of
// parts; a second launch adds the parts in order (the same bits on every call, no atomics).
#include "pkm_common.h"

#include <algorithm>

namespace smlm {
namespace {

constexpr int kRnMaxCols = 16384;

struct __attribute__((packed, aligned(2))) Raw16 {
  uint32_t v[4];
};
struct __attribute__((packed, aligned(4))) Raw32 {
  float v[8];
};

// A lane's columns of a step: 8 from `at` on, of which the first `skip` are a neighbour's too; n: how many it writes (8, less
// in rows of less than 8, 0 past the row, where it reads the last 8: loads without a branch stay in flight together).
struct Columns {
  int at, n, skip;
  __device__ __forceinline__ void init(int c, int C) {
    n = c < C ? min(8, C) : 0;
    at = max(0, min(c, C - 8));
    skip = c - at;
  }
};

// 8 values from element i on; if SHORT the first n of them (the others 0).
template <bool SHORT>
__device__ __forceinline__ void load8(const void *p, bool f32, int64_t i, int n, float *v) {
  if (!SHORT || n == 8) {
    if (f32) {
      const Raw32 a = *(const Raw32 *)((const float *)p + i);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = a.v[e];
    } else {
      const Raw16 a = *(const Raw16 *)((const uint16_t *)p + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[2 * e] = __uint_as_float(a.v[e] << 16);
        v[2 * e + 1] = __uint_as_float(a.v[e] & 0xFFFF0000u);
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      v[e] = e >= n ? 0.f : f32 ? ((const float *)p)[i + e] : bf16_bits_to_f32(((const uint16_t *)p)[i + e]);
  }
}

template <bool SHORT>
__device__ __forceinline__ void store8(void *p, bool f32, int64_t i, int n, const float *v) {
  if (n == 8) {
    if (f32) {
      Raw32 a;
#pragma unroll
      for (int e = 0; e < 8; ++e) a.v[e] = v[e];
      *(Raw32 *)((float *)p + i) = a;
    } else {
      Raw16 a;
#pragma unroll
      for (int e = 0; e < 4; ++e) a.v[e] = pack_bf16x2(v[2 * e], v[2 * e + 1]);
      *(Raw16 *)((uint16_t *)p + i) = a;
    }
  } else if constexpr (SHORT) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) {
        if (f32) ((float *)p)[i + e] = v[e];
        else ((uint16_t *)p)[i + e] = (uint16_t)(pack_bf16x2(v[e], v[e]) & 0xFFFFu);
      }
  }
}

// Lanes of a row, and what follows from them.
template <int LANES>
struct RowLanes {
  static constexpr int kThreads = LANES > kWave ? LANES : 256, kRows = kThreads / LANES, kWaves = LANES / kWave;
  static constexpr bool kShort = LANES == 16;             // rows of less than 8 columns
  // The lanes' sum; `sums`: one of each wavefront, reused (hence two barriers).
  static __device__ __forceinline__ float sum(float v, float *sums) {
    if constexpr (LANES < kWave) {
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
      return v;
    } else {
      v = wave_sum(v);
      if constexpr (LANES == kWave) return v;
      __syncthreads();
      if (threadIdx.x % kWave == 0) sums[threadIdx.x / kWave] = v;
      __syncthreads();
      v = 0.f;
#pragma unroll
      for (int q = 0; q < kWaves; ++q) v += sums[q];
      return v;
    }
  }
};

struct NormArgs {
  const void *x, *delta, *w, *dxs, *dh;   // the gradient: x = xs
  void *xs, *h, *dx, *ddelta;
  float *rstd, *parts;
  float eps;
  int64_t M, C, rows;                     // gradient: rows per workgroup
  bool x32, d32, w32, h32;
};

template <int NCH, int LANES>
__global__ void __launch_bounds__(RowLanes<LANES>::kThreads) norm_kernel(NormArgs a) {
  typedef RowLanes<LANES> R;
  constexpr bool kShort = R::kShort;
  __shared__ float sums[R::kWaves + 1];
  const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
  float w[NCH][8];
  Columns c[NCH];
#pragma unroll
  for (int q = 0; q < NCH; ++q) {
    c[q].init((q * LANES + lane) * 8, (int)a.C);
    load8<kShort>(a.w, a.w32, c[q].at, c[q].n, w[q]);
  }
  for (int64_t row = (int64_t)blockIdx.x * R::kRows + sub; row < a.M; row += (int64_t)gridDim.x * R::kRows) {
    float v[NCH][8], sq = 0.f;
#pragma unroll
    for (int q = 0; q < NCH; ++q) {
      const int64_t i = row * a.C + c[q].at;
      load8<kShort>(a.x, a.x32, i, c[q].n, v[q]);
      if (a.delta) {
        float d[8];
        load8<kShort>(a.delta, a.d32, i, c[q].n, d);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[q][e] = a.x32 ? v[q][e] + d[e] : round_bf16_hw(v[q][e] + d[e]);
        store8<kShort>(a.xs, a.x32, i, c[q].n, v[q]);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) sq += e >= c[q].skip ? v[q][e] * v[q][e] : 0.f;
    }
    const float rstd = 1.0f / sqrtf(R::sum(sq, sums) / (float)a.C + a.eps);
    if (lane == 0) a.rstd[row] = rstd;
#pragma unroll
    for (int q = 0; q < NCH; ++q) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[q][e] = v[q][e] * rstd * w[q][e];
      store8<kShort>(a.h, a.h32, row * a.C + c[q].at, c[q].n, v[q]);
    }
  }
}

template <int NCH, int LANES>
__global__ void __launch_bounds__(RowLanes<LANES>::kThreads) norm_grad_kernel(NormArgs a) {
  typedef RowLanes<LANES> R;
  constexpr bool kShort = R::kShort;
  __shared__ float sums[R::kWaves + 1];
  __shared__ float cols[R::kRows > 1 ? (R::kRows - 1) * NCH * 8 * LANES : 1];
  const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
  float w[NCH][8], dw[NCH][8];
  Columns c[NCH];
#pragma unroll
  for (int q = 0; q < NCH; ++q) {
    c[q].init((q * LANES + lane) * 8, (int)a.C);
    load8<kShort>(a.w, a.w32, c[q].at, c[q].n, w[q]);
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[q][e] = 0.f;
  }
  const int64_t end = min(a.M, (int64_t)(blockIdx.x + 1) * a.rows);
  for (int64_t row = (int64_t)blockIdx.x * a.rows + sub; row < end; row += R::kRows) {
    float hat[NCH][8], gw[NCH][8], res[NCH][8], dot = 0.f;
    const float rstd = a.rstd[row];
#pragma unroll
    for (int q = 0; q < NCH; ++q) {
      const int64_t i = row * a.C + c[q].at;
      load8<kShort>(a.x, a.x32, i, c[q].n, hat[q]);
      if (a.dh) load8<kShort>(a.dh, a.h32, i, c[q].n, gw[q]);
      if (a.dxs) load8<kShort>(a.dxs, a.x32, i, c[q].n, res[q]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        hat[q][e] *= rstd;
        const float dh = a.dh ? gw[q][e] : 0.f;
        if (!a.dxs) res[q][e] = 0.f;
        dw[q][e] += dh * hat[q][e];
        gw[q][e] = dh * w[q][e];
        dot += e >= c[q].skip ? gw[q][e] * hat[q][e] : 0.f;
      }
    }
    const float mean = R::sum(dot, sums) / (float)a.C;
#pragma unroll
    for (int q = 0; q < NCH; ++q) {
      const int64_t i = row * a.C + c[q].at;
#pragma unroll
      for (int e = 0; e < 8; ++e) res[q][e] += rstd * (gw[q][e] - hat[q][e] * mean);
      store8<kShort>(a.dx, a.x32, i, c[q].n, res[q]);
      if (a.ddelta) store8<kShort>(a.ddelta, a.d32, i, c[q].n, res[q]);
    }
  }
  if (!a.parts) return;  // uniform
  float *out = a.parts + (int64_t)blockIdx.x * a.C;
  if constexpr (R::kRows > 1) {   // the columns of the workgroup's other rows, in order
    if (sub > 0)
#pragma unroll
      for (int q = 0; q < NCH; ++q)
#pragma unroll
        for (int e = 0; e < 8; ++e) cols[(((sub - 1) * NCH + q) * 8 + e) * LANES + lane] = dw[q][e];
    __syncthreads();
    if (sub > 0) return;
    for (int s = 0; s < R::kRows - 1; ++s)
#pragma unroll
      for (int q = 0; q < NCH; ++q)
#pragma unroll
        for (int e = 0; e < 8; ++e) dw[q][e] += cols[((s * NCH + q) * 8 + e) * LANES + lane];
  }
#pragma unroll
  for (int q = 0; q < NCH; ++q) store8<kShort>(out, true, c[q].at, c[q].n, dw[q]);
}

// dw[c] = the parts' sum, 32 columns per workgroup, 32 threads a column.
__global__ void __launch_bounds__(1024)
    norm_weight_kernel(const float *__restrict__ parts, int nparts, int64_t C, bool w32, void *__restrict__ dw) {
  __shared__ float s[32][33];
  const int c = threadIdx.x % 32, p0 = threadIdx.x / 32;
  const int64_t col = (int64_t)blockIdx.x * 32 + c;
  float v = 0.f;
  if (col < C)
    for (int p = p0; p < nparts; p += 256) {   // 8 loads in flight, added in order (one by one: 10.6 us for 1,024 parts)
      float u[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) u[q] = p + 32 * q < nparts ? parts[(p + 32 * q) * C + col] : 0.f;
#pragma unroll
      for (int q = 0; q < 8; ++q) v += u[q];
    }
  s[p0][c] = v;
  __syncthreads();
  if (p0 > 0 || col >= C) return;
  for (int p = 1; p < 32; ++p) v += s[p][c];
  if (w32) ((float *)dw)[col] = v;
  else ((uint16_t *)dw)[col] = (uint16_t)(pack_bf16x2(v, v) & 0xFFFFu);
}

bool known(int dtype) { return dtype == SMLM_F32 || dtype == SMLM_BF16; }
uintptr_t odd(const void *p, int dtype) { return (uintptr_t)p % (dtype == SMLM_F32 ? 4 : 2); }

int check_norm(const char *what, int64_t M, int64_t C, int x, int w, int h, int delta) {
  if (!known(x) || !known(w) || !known(h) || !known(delta) || (x == SMLM_BF16 && delta == SMLM_F32))
    return fail(SMLM_EINVAL, "%s: types must be SMLM_F32 or SMLM_BF16, delta's no wider than x's", what);
  if (M < 0 || C < 1) return fail(SMLM_EINVAL, "%s: bad shape M=%lld C=%lld", what, (long long)M, (long long)C);
  if (C > kRnMaxCols || M > (1LL << 40))
    return fail(SMLM_EUNSUPPORTED, "%s: M=%lld C=%lld (at most %d columns)", what, (long long)M, (long long)C, kRnMaxCols);
  return SMLM_OK;
}

// Lanes of a row of C columns, 8 columns each (beyond 8,192 twice 8).  Few columns a lane and few lanes a row keep rows in
// flight: 27,306 x 768 in bf16, the gradient 53 us by 64 lanes and two steps, 44 by 128; 65,536 x 64 by 64 lanes 44 us, by
// 16 19.
int row_lanes(int64_t C) {
  int lanes = 16;
  while (lanes < 1024 && 8 * lanes < C) lanes *= 2;
  return lanes;
}
// Workgroups of the gradient: each leaves a row of parts; at most 4,096 wavefronts up to 2,048 columns, then 1,024 workgroups
// (8,192 wavefronts up to 4,096 columns, 16,384 beyond), of at least 4 rows each (8 by one wavefront).
int64_t grad_blocks(int64_t M, int64_t C) {
  const int lanes = row_lanes(C);
  const int64_t per = lanes <= 64 ? 512 / lanes : 4, most = lanes == 128 ? 2048 : 1024;
  return std::max<int64_t>(1, std::min<int64_t>(most, (M + per - 1) / per));
}

template <int NCH, int LANES>
void launch_norm(const NormArgs &a, bool grad, int64_t blocks, hipStream_t s) {
  const dim3 grid((unsigned)blocks), block(RowLanes<LANES>::kThreads);
  if (grad) hipLaunchKernelGGL((norm_grad_kernel<NCH, LANES>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((norm_kernel<NCH, LANES>), grid, block, 0, s, a);
}

void dispatch_norm(const NormArgs &a, bool grad, int64_t blocks, hipStream_t s) {
  switch (row_lanes(a.C)) {
    case 16: return launch_norm<1, 16>(a, grad, blocks, s);
    case 32: return launch_norm<1, 32>(a, grad, blocks, s);
    case 64: return launch_norm<1, 64>(a, grad, blocks, s);
    case 128: return launch_norm<1, 128>(a, grad, blocks, s);
    case 256: return launch_norm<1, 256>(a, grad, blocks, s);
    case 512: return launch_norm<1, 512>(a, grad, blocks, s);
    default: return a.C <= 8192 ? launch_norm<1, 1024>(a, grad, blocks, s) : launch_norm<2, 1024>(a, grad, blocks, s);
  }
}

}  // namespace
}  // namespace smlm

extern "C" int smlm_rmsnorm_train(const void *x, int x_dtype, const void *delta, int delta_dtype, const void *w, int w_dtype,
                                  float eps, int64_t M, int64_t C, void *xs, void *h, int h_dtype, float *rstd,
                                  void *stream) {
  using namespace smlm;
  const char *what = "smlm_rmsnorm_train";
  if (!x || !w || !h || !rstd || (delta && !xs)) return fail(SMLM_EINVAL, "%s: null pointer argument", what);
  if (!(eps >= 0.f)) return fail(SMLM_EINVAL, "%s: eps must not be negative", what);
  if (const int rc = check_norm(what, M, C, x_dtype, w_dtype, h_dtype, delta ? delta_dtype : x_dtype)) return rc;
  if (odd(x, x_dtype) | odd(w, w_dtype) | odd(h, h_dtype) | odd(rstd, SMLM_F32) | odd(delta, delta_dtype) | odd(xs, x_dtype))
    return fail(SMLM_EINVAL, "%s: tensors must be aligned to their elements", what);
  if (M == 0) return SMLM_OK;
  NormArgs a{};
  a.x = x;
  a.delta = delta;
  a.w = w;
  a.xs = xs;
  a.h = h;
  a.rstd = rstd;
  a.eps = eps;
  a.M = M;
  a.C = C;
  a.x32 = x_dtype == SMLM_F32;
  a.d32 = delta_dtype == SMLM_F32;
  a.w32 = w_dtype == SMLM_F32;
  a.h32 = h_dtype == SMLM_F32;
  const int64_t rows = C <= 512 ? 256 / row_lanes(C) : 1;
  dispatch_norm(a, false, std::min<int64_t>((M + rows - 1) / rows, 4096), (hipStream_t)stream);
  return launch_status(what);
}

extern "C" int64_t smlm_rmsnorm_parts(int64_t M, int64_t C) { return M < 1 || C < 1 ? 0 : smlm::grad_blocks(M, C) * C; }

extern "C" int smlm_rmsnorm_train_backward(const void *dxs, const void *dh, int h_dtype, const void *xs, int x_dtype,
                                           const void *w, int w_dtype, const float *rstd, int64_t M, int64_t C, void *dx,
                                           void *ddelta, int delta_dtype, void *dw, float *parts, void *stream) {
  using namespace smlm;
  const char *what = "smlm_rmsnorm_train_backward";
  if (!xs || !w || !rstd || !dx || (!dxs && !dh) || (dw && !parts)) return fail(SMLM_EINVAL, "%s: null pointer argument", what);
  if (const int rc = check_norm(what, M, C, x_dtype, w_dtype, h_dtype, ddelta ? delta_dtype : x_dtype)) return rc;
  if (odd(dxs, x_dtype) | odd(dh, h_dtype) | odd(xs, x_dtype) | odd(w, w_dtype) | odd(rstd, SMLM_F32) | odd(dx, x_dtype) |
      odd(ddelta, delta_dtype) | odd(dw, w_dtype) | odd(parts, SMLM_F32))
    return fail(SMLM_EINVAL, "%s: tensors must be aligned to their elements", what);
  if (M < 1) return fail(SMLM_EINVAL, "%s: no rows", what);
  NormArgs a{};
  a.dxs = dxs;
  a.dh = dh;
  a.x = xs;
  a.w = w;
  a.rstd = (float *)rstd;
  a.dx = dx;
  a.ddelta = ddelta;
  a.parts = dw ? parts : nullptr;
  a.M = M;
  a.C = C;
  a.x32 = x_dtype == SMLM_F32;
  a.d32 = delta_dtype == SMLM_F32;
  a.w32 = w_dtype == SMLM_F32;
  a.h32 = h_dtype == SMLM_F32;
  const int64_t blocks = grad_blocks(M, C);
  a.rows = (M + blocks - 1) / blocks;
  hipStream_t s = (hipStream_t)stream;
  dispatch_norm(a, true, blocks, s);
  if (const int rc = launch_status(what)) return rc;
  if (!dw) return SMLM_OK;
  hipLaunchKernelGGL(norm_weight_kernel, dim3((unsigned)((C + 31) / 32)), dim3(1024), 0, s, parts, (int)blocks, C, a.w32, dw);
  return launch_status(what);
}
