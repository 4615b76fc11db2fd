// Sampling: per row of logits x (V), the token at the given random number u of
//   w = exp((x - max) / temperature), kept where the token is among the top_k largest, in the smallest run of largest of these
//   whose mass reaches top_p of theirs, and no less than min_p of the largest;
// the token is the first one, in the vocabulary's order, whose running kept mass exceeds u times the kept mass.  Equal logits
// rank by index.  Temperature 0 takes the largest.
//
// Masses are whole numbers of 2^-45 of the largest weight, from weights in fp64: a sum is exact whatever its order, so every
// call gives the same token, and one that lies within rounding of its neighbour's border is as rare as in fp64 (fp32 sums over
// 50,000 tokens would give another token once in some hundred calls).  exp2 by a table of 2^(i / 256) and a polynomial of degree
// 4: with |r| <= ln 2 / 512 the next term is r^5 / 120 < 4e-17.
//
// One workgroup of 1,024 a row, the row in LDS where it fits (a wavefront has a run of the vocabulary of its own, so that the running
// mass is a sum over wavefronts, then over the found wavefront's vectors).  A cut -- the top_k-th token, or the one at which
// the mass reaches top_p -- is found by histograms: 1,024 bins of count (and mass) between the largest and smallest logit,
// a scan over the bins, then the bin that holds the cut as the next range, until it has at most 512 tokens, which are ranked
// against each other in LDS.
#include "pkm_common.h"

namespace smlm {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / kWave, kBins = 1024, kList = 512;
constexpr float kLowest = -3.3895313892515355e38f;   // the lowest bf16: masked logits and NaN
constexpr double kUnit = 0x1p45;

struct SampleArgs {
  const void *logits;
  int64_t row_stride;
  int V, vecs;                        // 16-byte vectors of a row a lane reads
  const float *u, *temperature, *top_p, *min_p;
  const int *top_k;
  float temperature1, top_p1, min_p1;
  int top_k1;
  int64_t *token;
};

struct Shared {
  double exp2[256];
  uint64_t mass[kBins];
  uint32_t count[kBins];
  float list_x[kList];
  int list_i[kList];
  uint64_t list_w[kList];
  uint64_t wave_mass[kWaves];
  uint32_t wave_count[kWaves];
  float wave_f[2][kWaves];
  // what one thread found for all
  uint64_t mass_above, total;
  uint32_t count_above, n, lo, hi;
  int bin, index, cut_rank;
  uint32_t fill;
};
constexpr int kSharedVecs = (sizeof(Shared) + 15) / 16;
constexpr int kLdsVecs = 160 * 1024 / 16 - kSharedVecs;      // vectors of a row that LDS holds

__device__ __forceinline__ uint32_t code_of(float x) { return order32(__float_as_uint(x)); }
__device__ __forceinline__ float value_of(uint32_t c) { return __uint_as_float(unorder32(c)); }

__device__ __forceinline__ uint64_t shfl_up64(uint64_t v, int o) {
  return (uint64_t)__shfl_up((uint32_t)v, o, kWave) | (uint64_t)__shfl_up((uint32_t)(v >> 32), o, kWave) << 32;
}
__device__ __forceinline__ uint64_t wave_sum64(uint64_t v) {
  v += xor_lane64<1>(v);
  v += xor_lane64<2>(v);
  v += xor_lane64<4>(v);
  v += xor_lane64<8>(v);
  v += xor_lane64<16>(v);
  v += xor_lane64<32>(v);
  return v;
}

// A row as its workgroup reads it, pass after pass: from LDS where it fits, else from memory.  Every lane reads only what it
// wrote, so the passes need no barrier between them.
template <bool BF16, bool LDS>
struct Row {
  static constexpr int W = BF16 ? 8 : 4;
  const char *base;
  uint4 *kept;
  int V, first, vecs;                 // first vector of this lane, vectors of its run
  bool aligned;

  __device__ __forceinline__ static float fix(float x) { return x > kLowest ? fminf(x, -kLowest) + 0.f : kLowest; }

  // vector j of the lane: masked logits and NaN as the lowest value, -0 as 0, -infinity behind the row's end
  __device__ __forceinline__ uint4 fetch(int j) const {
    const int at = (first + 64 * j) * W;
    float x[W];
    if (aligned && at + W <= V) {
      const uint4 raw = *(const uint4 *)(base + (int64_t)at * (BF16 ? 2 : 4));
      const uint32_t r[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
      for (int e = 0; e < W; ++e)
        x[e] = fix(BF16 ? __uint_as_float(e % 2 ? r[e / 2] & 0xFFFF0000u : r[e / 2] << 16) : __uint_as_float(r[e % 4]));
    } else {
#pragma unroll
      for (int e = 0; e < W; ++e) {
        x[e] = -__builtin_inff();
        if (at + e < V)
          x[e] = fix(BF16 ? bf16_bits_to_f32(((const uint16_t *)base)[at + e]) : ((const float *)base)[at + e]);
      }
    }
    uint32_t u[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      u[e] = BF16 ? __float_as_uint(x[(2 * e) % W]) >> 16 | (__float_as_uint(x[(2 * e + 1) % W]) & 0xFFFF0000u)
                  : __float_as_uint(x[e % W]);
    return uint4{u[0], u[1], u[2], u[3]};
  }

  __device__ __forceinline__ Row(const void *p, int64_t row, int64_t stride, int n, int wave, int lane, int vecs_, uint4 *lds)
      : base((const char *)p + row * stride * (BF16 ? 2 : 4)), kept(lds), V(n), first(wave * vecs_ * 64 + lane), vecs(vecs_),
        aligned((uintptr_t)base % 16 == 0) {
    if constexpr (LDS) {
#pragma unroll 4
      for (int j = 0; j < vecs; ++j) kept[first + 64 * j] = fetch(j);
    }
  }

  __device__ __forceinline__ uint4 vector(int j) const {
    if constexpr (LDS) return kept[first + 64 * j];
    else return fetch(j);
  }
  // f(x, index) for every element of vector j
  template <class F>
  __device__ __forceinline__ void vec(int j, const uint4 &raw, F &&f) const {
    const uint32_t r[4] = {raw.x, raw.y, raw.z, raw.w};
    const int at = (first + 64 * j) * W;
#pragma unroll
    for (int e = 0; e < W; ++e)
      f(BF16 ? __uint_as_float(e % 2 ? r[e / 2] & 0xFFFF0000u : r[e / 2] << 16) : __uint_as_float(r[e % 4]), at + e);
  }
  template <class F>
  __device__ __forceinline__ void each(F &&f) const {
#pragma unroll 2
    for (int j = 0; j < vecs; ++j) vec(j, vector(j), f);
  }
};

struct Weight {
  const double *table;
  double scale;                       // log2(e) / temperature
  float top, min_p;

  // 2^((x - top) scale)
  __device__ __forceinline__ double weight(float x) const {
    const double t = ((double)x - (double)top) * scale;
    if (!(t > -46.0)) return 0.0;
    const double k = __builtin_rint(t * 256.0);
    const double r = __builtin_fma(k, -1.0 / 256.0, t) * 0.693147180559945309417;
    const int ki = (int)k;
    double p = __builtin_fma(r, 1.0 / 24.0, 1.0 / 6.0);
    p = __builtin_fma(p, r, 0.5);
    p = __builtin_fma(p, r, 1.0);
    p = __builtin_fma(p, r, 1.0);
    return ldexp(p * table[ki & 255], ki >> 8);
  }
  __device__ __forceinline__ uint64_t mass_of(double w) const {
    return (uint64_t)__double_as_longlong(__builtin_fma(w, kUnit, 0x1p52)) & 0xFFFFFFFFFFFFFull;
  }
  __device__ __forceinline__ uint64_t mass(float x) const { return mass_of(weight(x)); }
  __device__ __forceinline__ uint64_t kept_mass(float x) const {
    const double w = weight(x);
    return w >= (double)min_p ? mass_of(w) : 0;
  }
};

// The kept tokens: those above `value`, and of those equal to it the ones up to `index`; how many.
struct Cut {
  float value;
  int index;
  uint32_t n;
  __device__ __forceinline__ bool keeps(float x, int i) const { return x > value || (x == value && i <= index); }
};

// The cut after the k-th kept token (MASS false), or after the one at which the mass reaches `share` of the kept mass.
template <bool MASS, class R>
__device__ Cut select(const R &row, const Weight &weight, Shared &S, const Cut cut, float top, float bottom, uint32_t k, double share) {
  const int tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave;
  uint32_t lo = code_of(fmaxf(bottom, cut.value)), hi = code_of(top), n = cut.n, above = 0;
  uint64_t mass_above = 0;
  double target = 0.0;                 // of the mass, once the total is known
  bool first = true;
  // every pass leaves the cut's bin as the range lo .. hi of codes, both of tokens in it: fewer tokens, or one value alone
  while (n > kList && lo < hi) {
    S.mass[tid] = 0;
    S.count[tid] = 0;
    __syncthreads();
    const float fhi = value_of(hi), flo = value_of(lo), span = fhi * 0.5f - flo * 0.5f;
    const bool linear = first && span > 1e-30f && span < 1e30f;   // bins of equal width in value, later in code
    const float inv = linear ? 511.5f / span : 0.f;
    const int shift = max(0, 32 - __builtin_clz(hi - lo) - 10);
    auto bin_of = [&](float x) {
      return linear ? min((int)((fhi - x) * inv), kBins - 1) : (int)((hi - code_of(x)) >> shift);
    };
    row.each([&](float x, int i) {
      if (x >= flo && x <= fhi && cut.keeps(x, i)) {
        const int b = bin_of(x);
        atomicAdd(&S.count[b], 1u);
        if constexpr (MASS) atomicAdd((unsigned long long *)&S.mass[b], (unsigned long long)weight.mass(x));
      }
    });
    __syncthreads();
    // running count and mass up to this thread's bin
    const uint32_t c = S.count[tid];
    const uint64_t w = MASS ? S.mass[tid] : 0;
    uint32_t cs = c;
    uint64_t ws = w;
#pragma unroll
    for (int o = 1; o < kWave; o *= 2) {
      const uint32_t a = __shfl_up(cs, o, kWave);
      const uint64_t b = MASS ? shfl_up64(ws, o) : 0;
      if (lane >= o) cs += a, ws += b;
    }
    if (lane == kWave - 1) S.wave_count[wave] = cs, S.wave_mass[wave] = ws;
    __syncthreads();
    uint64_t total = mass_above;
    cs += above, ws += mass_above;
    for (int i = 0; i < kWaves; ++i) {
      if (i < wave) cs += S.wave_count[i], ws += S.wave_mass[i];
      total += S.wave_mass[i];
    }
    if (MASS && first) target = fmax(share * (double)total, 1.0);
    const bool here = MASS ? (double)(ws - w) < target && target <= (double)ws : cs - c < k && k <= cs;
    if (here) S.bin = tid, S.n = c, S.count_above = cs - c, S.mass_above = ws - w;
    if (tid == 0) S.lo = 0xFFFFFFFFu, S.hi = 0;
    __syncthreads();
    const int bin = S.bin;
    n = S.n, above = S.count_above, mass_above = S.mass_above;
    uint32_t bl = 0xFFFFFFFFu, bh = 0;
    row.each([&](float x, int i) {
      if (x >= flo && x <= fhi && cut.keeps(x, i) && bin_of(x) == bin) bl = min(bl, code_of(x)), bh = max(bh, code_of(x));
    });
    if (bh) atomicMin(&S.lo, bl), atomicMax(&S.hi, bh);
    __syncthreads();
    lo = S.lo, hi = S.hi;
    first = false;
  }

  const float flo = value_of(lo), fhi = value_of(hi);
  if (n <= kList) {
    // the range's tokens ranked against each other
    if (tid == 0) S.fill = 0, S.cut_rank = -1;
    __syncthreads();
    row.each([&](float x, int i) {
      if (x >= flo && x <= fhi && cut.keeps(x, i)) {
        const uint32_t at = atomicAdd(&S.fill, 1u);
        if (at < kList) S.list_x[at] = x, S.list_i[at] = i;
      }
    });
    __syncthreads();
    n = min(n, S.fill);
    if (MASS && tid < (int)n) S.list_w[tid] = weight.mass(S.list_x[tid]);
    __syncthreads();
    float x = 0.f;
    int index = 0, before = 0;
    bool keep = false;
    if (tid < (int)n) {
      x = S.list_x[tid], index = S.list_i[tid];
      uint64_t mass = mass_above, total = mass_above;
      for (int i = 0; i < (int)n; ++i) {
        const float y = S.list_x[i];
        const bool ahead = y > x || (y == x && S.list_i[i] < index);
        before += ahead;
        if constexpr (MASS) {
          mass += ahead ? S.list_w[i] : 0;
          total += S.list_w[i];
        }
      }
      if (MASS && first) target = fmax(share * (double)total, 1.0);
      keep = MASS ? (double)mass < target : above + before < k;
      if (keep) atomicMax(&S.cut_rank, before);
    }
    __syncthreads();
    if (keep && before == S.cut_rank) S.list_x[0] = x, S.index = index;   // (read by nobody else any more)
    __syncthreads();
    const Cut got{S.list_x[0], S.index, above + (uint32_t)S.cut_rank + 1};
    __syncthreads();
    return got;
  }
  // more equal tokens than the list holds: the first c of them, the last of which is found by bisection of the index
  uint64_t c = k - above;
  if constexpr (MASS) {
    const uint64_t one = weight.mass(fhi);
    if (first) target = fmax(share * ((double)n * (double)one), 1.0);
    const double more = ceil(target) - (double)mass_above;      // the least whole mass beyond what lies above
    c = one ? ((uint64_t)fmax(more, 1.0) - 1) / one + 1 : n;
  }
  c = c < 1 ? 1 : c > n ? n : c;
  int a = 0, b = row.V - 1;
  while (a < b) {
    const int mid = a + (b - a) / 2;
    uint32_t here = 0;
    row.each([&](float x, int i) { here += x == fhi && i <= mid && cut.keeps(x, i); });
    for (int o = 32; o > 0; o >>= 1) here += __shfl_xor(here, o, kWave);
    __syncthreads();
    if (lane == 0) S.wave_count[wave] = here;
    __syncthreads();
    uint32_t all = 0;
    for (int i = 0; i < kWaves; ++i) all += S.wave_count[i];
    if (all >= c) b = mid;
    else a = mid + 1;
  }
  __syncthreads();
  return Cut{fhi, a, above + (uint32_t)c};
}

template <bool BF16, bool LDS>
__global__ void __launch_bounds__(kThreads) sample_kernel(SampleArgs A) {
  extern __shared__ __align__(16) uint4 smem[];
  Shared &S = *(Shared *)smem;
  const int64_t at = blockIdx.x;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave;
  const Row<BF16, LDS> row(A.logits, at, A.row_stride, A.V, wave, lane, A.vecs, smem + kSharedVecs);
  const float temperature = A.temperature ? A.temperature[at] : A.temperature1;
  const float top_p = A.top_p ? A.top_p[at] : A.top_p1, min_p = A.min_p ? A.min_p[at] : A.min_p1;
  const int top_k = A.top_k ? A.top_k[at] : A.top_k1;
  const double u = A.u[at];
  if (tid < 256) S.exp2[tid] = exp2(tid * (1.0 / 256.0));

  float top = kLowest, bottom = -kLowest;
  row.each([&](float x, int) {
    top = fmaxf(top, x);
    bottom = x >= kLowest ? fminf(bottom, x) : bottom;
  });
  for (int o = 32; o > 0; o >>= 1) {
    top = fmaxf(top, __shfl_xor(top, o, kWave));
    bottom = fminf(bottom, __shfl_xor(bottom, o, kWave));
  }
  if (lane == 0) S.wave_f[0][wave] = top, S.wave_f[1][wave] = bottom;
  if (tid == 0) S.index = A.V - 1;
  __syncthreads();
  for (int i = 0; i < kWaves; ++i) top = fmaxf(top, S.wave_f[0][i]), bottom = fminf(bottom, S.wave_f[1][i]);

  if (!(temperature > 0.f)) {
    int best = A.V - 1;
    row.each([&](float x, int i) { best = x == top ? min(best, i) : best; });
    for (int o = 32; o > 0; o >>= 1) best = min(best, __shfl_xor(best, o, kWave));
    if (lane == 0) atomicMin(&S.index, best);
    __syncthreads();
    if (tid == 0) A.token[at] = S.index;
    return;
  }

  const Weight weight{S.exp2, 1.4426950408889634074 / (double)temperature, top, fminf(min_p, 1.f)};
  Cut cut{kLowest, 0x7FFFFFFF, (uint32_t)A.V};
  if (top_k > 0 && top_k < A.V) cut = select<false>(row, weight, S, cut, top, bottom, (uint32_t)top_k, 0.0);
  if (top_p < 1.f) cut = select<true>(row, weight, S, cut, top, bottom, 0u, (double)top_p);

  uint64_t sum = 0;
  row.each([&](float x, int i) {
    if (cut.keeps(x, i)) sum += weight.kept_mass(x);
  });
  sum = wave_sum64(sum);
  if (lane == 0) S.wave_mass[wave] = sum;
  __syncthreads();
  uint64_t total = 0, before = 0;
  for (int i = 0; i < kWaves; ++i) total += S.wave_mass[i];
  const double aim = u * (double)total;
  uint64_t target = aim > 0.0 ? (uint64_t)fmin(aim, 9.2e18) : 0;      // the token's running mass is above it
  if (target >= total) target = total - 1;
  for (int i = 0; i < wave; ++i) before += S.wave_mass[i];
  if (before > target || before + sum <= target) return;               // one wavefront goes on
  for (int j = 0; j < row.vecs; ++j) {
    const uint4 raw = row.vector(j);
    uint64_t mine = 0;
    row.vec(j, raw, [&](float x, int i) {
      if (cut.keeps(x, i)) mine += weight.kept_mass(x);
    });
    uint64_t run = mine;
#pragma unroll
    for (int o = 1; o < kWave; o *= 2) {
      const uint64_t b = shfl_up64(run, o);
      if (lane >= o) run += b;
    }
    const uint64_t all = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)run, 63) |
                         (uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(run >> 32), 63) << 32;
    if (before + all > target) {
      uint64_t mass = before + run - mine;
      if (mass <= target && before + run > target) {
        int64_t found = -1;
        row.vec(j, raw, [&](float x, int i) {
          if (cut.keeps(x, i)) mass += weight.kept_mass(x);
          if (found < 0 && mass > target) found = i;
        });
        A.token[at] = found;
      }
      return;
    }
    before += all;
  }
}

template <bool BF16>
int launch(const SampleArgs &A, int64_t B, hipStream_t s) {
  const int row = A.vecs * kThreads;
  if (row <= kLdsVecs) {
    const hipError_t e = hipFuncSetAttribute((const void *)sample_kernel<BF16, true>,
                                             hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    if (e != hipSuccess) return fail(SMLM_EHIP, "smlm_sample: hipFuncSetAttribute: %s", hipGetErrorString(e));
    hipLaunchKernelGGL((sample_kernel<BF16, true>), dim3((unsigned)B), dim3(kThreads), (kSharedVecs + row) * 16, s, A);
  } else {
    hipLaunchKernelGGL((sample_kernel<BF16, false>), dim3((unsigned)B), dim3(kThreads), kSharedVecs * 16, s, A);
  }
  return launch_status("smlm_sample");
}

}  // namespace
}  // namespace smlm

extern "C" int smlm_sample(const void *logits, int dtype, int64_t row_stride, const float *u, const float *temperature,
                           float temperature_all, const int *top_k, int top_k_all, const float *top_p, float top_p_all,
                           const float *min_p, float min_p_all, int64_t B, int64_t V, int64_t *token, void *stream) {
  using namespace smlm;
  const char *name = "smlm_sample";
  if (!logits || !u || !token) return fail(SMLM_EINVAL, "%s: null pointer argument", name);
  if (dtype != SMLM_BF16 && dtype != SMLM_F32) return fail(SMLM_EINVAL, "%s: logits must be SMLM_BF16 or SMLM_F32", name);
  if (B < 0 || V < 1 || row_stride < V) return fail(SMLM_EINVAL, "%s: bad shape B=%lld V=%lld row_stride=%lld", name,
                                                    (long long)B, (long long)V, (long long)row_stride);
  if (V > 1 << 18 || B > 0x7FFFFFFF)      // masses of 2^45 a token add up in 63 bits
    return fail(SMLM_EUNSUPPORTED, "%s: V=%lld is over 2^18, or B=%lld over 2^31", name, (long long)V, (long long)B);
  if ((uintptr_t)logits % (dtype == SMLM_F32 ? 4 : 2) || (uintptr_t)token % 8 ||
      ((uintptr_t)u | (uintptr_t)temperature | (uintptr_t)top_k | (uintptr_t)top_p | (uintptr_t)min_p) % 4)
    return fail(SMLM_EINVAL, "%s: a pointer is not aligned to its type", name);
  if (B == 0) return SMLM_OK;
  const int W = dtype == SMLM_BF16 ? 8 : 4;
  const SampleArgs A{logits, row_stride, (int)V, (int)((V + kThreads * W - 1) / (kThreads * W)), u, temperature, top_p, min_p,
                     top_k, temperature_all, top_p_all, min_p_all, top_k_all, token};
  return dtype == SMLM_BF16 ? launch<true>(A, B, (hipStream_t)stream) : launch<false>(A, B, (hipStream_t)stream);
}
