// Sampling: per row of logits x (V), the token at the given random number u of
//   w = exp((x - max) / temperature), kept where the token is among the top_k largest, in the smallest run of largest of these
//   whose mass reaches top_p of theirs, and no less than min_p of the largest;
// the token is the first one, in the vocabulary's order, whose running kept mass exceeds u times the kept mass.  Equal logits
// rank by index.  Temperature 0 takes the largest.
//
// Masses are whole numbers of 2^-45 of the largest weight, from weights in fp64: a sum is exact whatever its order, so every
// call gives the same token, and one that lies within rounding of its neighbour's border is as rare as in fp64 (fp32 sums over
// 50,000 tokens would give another token once in some hundred calls).  exp2 by a table of 2^(i / 64) and a
// polynomial of degree 5: with |r| <= ln 2 / 128 the next term is r^6 / 720 < 4e-17.
//
// One workgroup of 1,024 a row, the row in LDS where it fits (a wavefront has a run of the vocabulary of its own, so that the
// running mass is a sum over wavefronts, then over the found wavefront's vectors).  Bound by the passes over the row, vector
// instructions all: of a bf16 row of 50,304, reading it and finding its maximum takes 7 us, a pass that compares 1.5 to 2, one
// with every token's exact weight 12 (20 where it parts them at a cut), one that adds rough ones to a histogram 12.  So the tokens
// that may be kept are listed first, where a bound on them is cheap -- top_k: at least that many tokens lie above the bin that
// holds the k-th largest of the threads' own maxima; min_p: a bound on the logit -- and everything else is done on the list, by ranking
// each of its 512 tokens at most against all (256 of a bf16 row: 256 rows with min_p 0.01 and top_p 46 us with more, 42 so).
// Else a cut, the top_k-th token or the one at which the mass reaches top_p, is found in a bf16 row by counting its distinct
// values, in an fp32 row by a histogram of 1,024 bins, then within its bin.  One row, whole calls, bf16 (fp32): the largest 9.5 us
// (9.5), no cut 24 (23), top_k 50 with top_p 16 (16), min_p 0.1 13 (13), top_p 0.9 alone 37 (53), top_k 2,000 with top_p 36 (63);
// 256 bf16 rows 6 to 17% more, with min_p 0.01 and top_p a third; 256 fp32 rows, which LDS does not hold at this size, 17, 30, 23,
// 22, 65 and 79 us.  Rows of 50,303, of which none but the first is aligned, take as long.  (Forming the weights' rough sum
// while the row is read took top_p alone from 59 to 54 us and top_p with min_p from 25 to 27; masses looked up per distinct value
// instead of formed per token, 23 to 33 us without a cut.)
#include <cstddef>

#include "pkm_common.h"

namespace smlm {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / kWave, kBins = 1024, kList = 512, kPowerBits = 6, kPowers = 1 << kPowerBits;
constexpr float kLowest = -3.3895313892515355e38f;   // the lowest bf16: masked logits (-infinity, NaN, all that is lower)
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
  double power[kPowers];
  uint64_t mass[kBins];
  uint32_t count[kBins];
  float list_x[kList];
  int list_i[kList];
  uint64_t list_w[kList], list_before[kList];
  uint32_t list_rank[kList];
  uint64_t wave_mass[kWaves];
  uint64_t wave_kept[kWaves];
  uint32_t wave_count[kWaves];
  float wave_f[2][kWaves];
  // what one thread found for all
  uint64_t mass_above, total;
  uint32_t count_above, n, lo, hi, fill;
  int bin, index;
};
constexpr int kSharedVecs = (sizeof(Shared) + 15) / 16;
constexpr int kLdsVecs = 160 * 1024 / 16 - kSharedVecs;      // vectors of a row that LDS holds

__device__ __forceinline__ uint32_t code_of(float x) { return order32(__float_as_uint(x + 0.f)); }      // (-0 as 0)
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

// 16 bytes of a row, which begins at a multiple of a logit's size alone: one load all the same
typedef uint32_t Four __attribute__((ext_vector_type(4)));
typedef Four Loose __attribute__((aligned(2)));

// A row as its workgroup reads it, pass after pass: from LDS where it fits, else from memory.  Every lane reads only what it
// wrote, so the passes need no barrier between them.
template <bool BF16, bool LDS>
struct Row {
  static constexpr int W = BF16 ? 8 : 4;
  const char *base;
  uint4 *kept;
  int V, first, vecs;                 // first vector of this lane, vectors of its run
  // (med3 of a NaN is the lowest of the others)
  __device__ __forceinline__ static float fix(float x) { return __builtin_amdgcn_fmed3f(x, kLowest, -kLowest); }

  // vector j of the lane: masked logits and NaN as the lowest value, -infinity behind the row's end
  __device__ __forceinline__ uint4 fetch(int j) const { return fetch_at((first + 64 * j) * W); }
  __device__ __forceinline__ uint4 fetch_at(int at) const {
    float x[W];
    if (at + W <= V) {
      const Loose r = *(const Loose *)(base + (int64_t)at * (BF16 ? 2 : 4));
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
      : base((const char *)p + row * stride * (BF16 ? 2 : 4)), kept(lds), V(n), first(wave * vecs_ * 64 + lane), vecs(vecs_) {}
  // the first pass: f(x, index) for every element, and the row into LDS
  template <class F>
  __device__ __forceinline__ void load(F &&f) const {
#pragma unroll 8
    for (int j = 0; j < vecs; ++j) {
      const uint4 raw = fetch(j);
      if constexpr (LDS) kept[first + 64 * j] = raw;
      vec(j, raw, f);
    }
  }

  __device__ __forceinline__ uint4 vector(int j) const {
    if constexpr (LDS) return kept[first + 64 * j];
    else return fetch(j);
  }
  // f(x, index) for every element of vector j
  template <class F>
  __device__ __forceinline__ void vec(int j, const uint4 &raw, F &&f) const { each_of((first + 64 * j) * W, raw, f); }
  // the same of wavefront w's run
  __device__ __forceinline__ uint4 of_run(int w, int j) const {
    const int v = (w * vecs + j) * 64 + (int)(threadIdx.x % kWave);
    if constexpr (LDS) return kept[v];
    else return fetch_at(v * W);
  }
  template <class F>
  __device__ __forceinline__ void vec_of_run(int w, int j, const uint4 &raw, F &&f) const {
    each_of(((w * vecs + j) * 64 + (int)(threadIdx.x % kWave)) * W, raw, f);
  }
  template <class F>
  __device__ __forceinline__ void each_of(int at, const uint4 &raw, F &&f) const {
    const uint32_t r[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int e = 0; e < W; ++e)
      f(BF16 ? __uint_as_float(e % 2 ? r[e / 2] & 0xFFFF0000u : r[e / 2] << 16) : __uint_as_float(r[e % 4]), at + e);
  }
  template <class F>
  __device__ __forceinline__ void each(F &&f) const {
#pragma unroll 2
    for (int j = 0; j < vecs; ++j) vec(j, vector(j), f);
  }
  // f(x, index, whether the cut keeps it) for every element of vector j, or, where no lane has more than three that it keeps,
  // for those alone
  template <class P, class F>
  __device__ __forceinline__ void vec_where(int j, const uint4 &raw, const P &takes, F &&f) const {
    const int at = (first + 64 * j) * W;
    if (takes.all) {
      vec(j, raw, [&](float x, int i) { f(x, i, true); });
      return;
    }
    uint32_t bits = 0;
    vec(j, raw, [&](float x, int i) { bits |= takes.keeps(x, i) ? 1u << (i - at) : 0u; });
    if (__builtin_amdgcn_ballot_w64(__builtin_popcount(bits) > 3)) {
      vec(j, raw, [&](float x, int i) { f(x, i, (bits >> (i - at) & 1) != 0); });
      return;
    }
    each_bit(j, raw, bits, f);
  }
  // f(x, index, whether it is one) for the elements of vector j that have a bit
  template <class F>
  __device__ __forceinline__ void each_bit(int j, const uint4 &raw, uint32_t bits, F &&f) const {
    const int at = (first + 64 * j) * W;
    while (__builtin_amdgcn_ballot_w64(bits != 0)) {
      const int e = bits ? __builtin_ctz(bits) : 0, word = BF16 ? e >> 1 : e;
      uint32_t w = raw.x;
      w = word == 1 ? raw.y : w;
      w = word == 2 ? raw.z : w;
      w = word == 3 ? raw.w : w;
      f(__uint_as_float(!BF16 ? w : e & 1 ? w & 0xFFFF0000u : w << 16), at + e, bits != 0);
      bits &= bits - 1;
    }
  }
};

struct Weight {
  const double *power;                // 2^(i / 64)
  double scale;                       // 64 log2(e) / temperature
  float top;
  double min_p;
  float masked;                       // logits up to here weigh nothing, whatever the temperature (-infinity where all are masked)

  // 2^((x - top) scale / 64), from 2^-47 on, below which a mass is 0 either way (fmax also takes the -infinity times 0 of an
  // infinite temperature there).  No branches, so that the chains of a vector's
  // elements overlap, and rounding and scaling by additions (conversions and ldexp take four times as long).
  __device__ __forceinline__ double weight(float x) const {
    const double t = __builtin_fmax(((double)(x > masked ? x : -__builtin_inff()) - (double)top) * scale, -47.0 * kPowers);
    const double m = t + 0x1.8p52, r = t - (m - 0x1.8p52);             // t rounded, in m's low bits
    const int k = (int)(uint32_t)__double_as_longlong(m);
    constexpr double c = 0.693147180559945309417 / kPowers;
    double p = __builtin_fma(r, c * c * c * c * c / 120, c * c * c * c / 24);
    p = __builtin_fma(p, r, c * c * c / 6);
    p = __builtin_fma(p, r, c * c / 2);
    p = __builtin_fma(p, r, c);
    p = __builtin_fma(p, r, 1.0);
    const uint64_t w = (uint64_t)__double_as_longlong(p * power[k & (kPowers - 1)]);
    return __longlong_as_double((long long)(w + ((uint64_t)(uint32_t)(k >> kPowerBits) << 52)));
  }
  __device__ __forceinline__ uint64_t mass_of(double w) const {
    return (uint64_t)__double_as_longlong(__builtin_fma(w, kUnit, 0x1p52)) & 0xFFFFFFFFFFFFFull;
  }
  __device__ __forceinline__ uint64_t mass(float x) const { return mass_of(weight(x)); }
  __device__ __forceinline__ uint64_t kept_mass(float x) const {
    const double w = weight(x);
    return w >= min_p ? mass_of(w) : 0;
  }
};

// The kept tokens: those above `value`, and of those equal to it the ones up to `index`.
struct Cut {
  float value;
  int index;
  bool all;                            // it keeps every token (and what stands behind the row's end weighs nothing)
  __device__ __forceinline__ bool keeps(float x, int i) const { return all | (x > value) | ((x == value) & (i <= index)); }
};

// The bins of a range of logits, from its top down: of equal width in value, or (always possible) in code.
struct Bins {
  float hi, inv;
  uint32_t hi_code;
  int shift;
  bool linear;
  __device__ __forceinline__ Bins(uint32_t lo_code, uint32_t hi_code_, bool by_value) : hi_code(hi_code_) {
    hi = value_of(hi_code);
    const float span = hi * 0.5f - value_of(lo_code) * 0.5f;
    linear = by_value && span > 1e-30f && span < 1e30f;
    inv = linear ? 511.5f / span : 0.f;
    shift = max(0, 32 - __builtin_clz((hi_code - lo_code) | 1) - 10);
  }
  __device__ __forceinline__ int of(float x) const {
    // (never past the last bin: what stands behind the row's end is below the range)
    return linear ? min((int)((hi - x) * inv), kBins - 1) : (int)min((hi_code - code_of(x)) >> shift, (uint32_t)(kBins - 1));
  }
};

// The running sum of v over the workgroup's threads up to this one; `total` of all.
template <class T>
__device__ __forceinline__ T running(T v, T *wave_sums, T &total) {
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
#pragma unroll
  for (int o = 1; o < kWave; o *= 2) {
    T b;
    if constexpr (sizeof(T) == 8) b = shfl_up64(v, o);
    else b = __shfl_up(v, o, kWave);
    if (lane >= o) v += b;
  }
  __syncthreads();
  if (lane == kWave - 1) wave_sums[wave] = v;
  __syncthreads();
  total = 0;
  T before = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    before += i < wave ? wave_sums[i] : 0;
    total += wave_sums[i];
  }
  return v + before;
}

// Lists the tokens that f takes, in any order; returns how many there are (those beyond kList are not listed).
template <class R, class F>
__device__ __forceinline__ uint32_t list(const R &row, Shared &S, F &&f) {
  __syncthreads();
  if (threadIdx.x == 0) S.fill = 0;
  __syncthreads();
  row.each([&](float x, int i) {
    if (f(x, i)) {
      const uint32_t at = atomicAdd(&S.fill, 1u);
      if (at < kList) S.list_x[at] = x, S.list_i[at] = i;
    }
  });
  __syncthreads();
  return S.fill;
}

// Per listed token (n of them): list_rank of the tokens ahead and list_before of their mass, ahead(x, i, y, j) whether the token
// j of logit y is ahead of the token i of logit x.  Every token is compared with all by several threads, each with a part of
// them.
template <class F>
__device__ __forceinline__ void rank(Shared &S, int n, F &&ahead) {
  const int tid = threadIdx.x;
  if (tid < n) S.list_rank[tid] = 0, S.list_before[tid] = 0;
  __syncthreads();
  const int parts = kThreads / n, part = tid / n, at = tid - part * n;
  if (part < parts) {
    const float x = S.list_x[at];
    const int i = S.list_i[at];
    uint32_t c = 0;
    uint64_t w = 0;
#pragma unroll 4
    for (int o = part; o < n; o += parts) {
      const float y = S.list_x[o];
      const int j = S.list_i[o];
      const uint64_t m = S.list_w[o];
      const bool is = ahead(x, i, y, j);
      c += is;
      w += is ? m : 0;
    }
    if (c) {
      atomicAdd(&S.list_rank[at], c);
      atomicAdd((unsigned long long *)&S.list_before[at], (unsigned long long)w);
    }
  }
  __syncthreads();
}
// the order of the logits, and of the vocabulary
struct ByLogit {
  __device__ __forceinline__ bool operator()(float x, int i, float y, int j) const { return (y > x) | ((y == x) & (j < i)); }
};
struct ByIndex {
  __device__ __forceinline__ bool operator()(float, int i, float, int j) const { return j < i; }
};

// The cut after the k-th kept token (MASS false), or after the one at which the mass reaches `share` of the kept mass.
template <bool MASS, class R>
__device__ __forceinline__ Cut select(const R &row, const Weight &weight, Shared &S, const Cut cut, float top, float bottom,
                                          uint32_t k, double share) {
  const int tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave;
  uint32_t lo = code_of(fmaxf(bottom, cut.value)), hi = code_of(top), above = 0;
  uint64_t mass_above = 0;
  double target = 0.0;                 // of the mass, once the total is known
  // every pass leaves the cut's bin as the range lo .. hi of codes, both of tokens in it: fewer tokens, or one value alone
  for (bool first = true;; first = false) {
    __syncthreads();
    S.mass[tid] = 0;
    S.count[tid] = 0;
    __syncthreads();
    const Bins bins(lo, hi, first);
    const float flo = value_of(lo), fhi = value_of(hi);
    row.each([&](float x, int i) {
      if (x >= flo && x <= fhi && cut.keeps(x, i)) {
        const int b = bins.of(x);
        if constexpr (MASS) atomicAdd((unsigned long long *)&S.mass[b], (unsigned long long)weight.mass(x));
        else atomicAdd(&S.count[b], 1u);
      }
    });
    __syncthreads();
    // running count or mass up to this thread's bin
    bool here;
    if constexpr (MASS) {
      const uint64_t w = S.mass[tid];
      uint64_t total;
      const uint64_t upto = mass_above + running(w, S.wave_mass, total);
      if (first) target = fmax(share * (double)total, 1.0);
      here = (double)(upto - w) < target && target <= (double)upto;
      if (here) S.bin = tid, S.mass_above = upto - w;
    } else {
      const uint32_t c = S.count[tid];
      uint32_t total;
      const uint32_t upto = above + running(c, S.wave_count, total);
      here = upto - c < k && k <= upto;
      if (here) S.bin = tid, S.count_above = upto - c;
    }
    if (tid == 0) S.lo = 0xFFFFFFFFu, S.hi = 0;
    __syncthreads();
    const int bin = S.bin;
    if constexpr (MASS) mass_above = S.mass_above;
    else above = S.count_above;
    const uint32_t n = list(row, S, [&](float x, int i) { return x >= flo && x <= fhi && cut.keeps(x, i) && bins.of(x) == bin; });
    if (n <= kList) {
      // the bin's tokens ranked against each other
      if (tid < (int)n) S.list_w[tid] = MASS ? weight.mass(S.list_x[tid]) : 0;
      __syncthreads();
      rank(S, (int)n, ByLogit());
      const bool keep = tid < (int)n && (MASS ? (double)(mass_above + S.list_before[tid]) < target : above + S.list_rank[tid] < k);
      if (tid == 0) S.n = 0;
      __syncthreads();
      if (keep) atomicMax(&S.n, S.list_rank[tid]);       // the last kept token's rank
      __syncthreads();
      const uint32_t last = S.n;
      if (keep && S.list_rank[tid] == last) S.index = tid;
      __syncthreads();
      const Cut got{S.list_x[S.index], S.list_i[S.index], false};
      __syncthreads();
      return got;
    }
    uint32_t bl = 0xFFFFFFFFu, bh = 0;
    row.each([&](float x, int i) {
      if (x >= flo && x <= fhi && cut.keeps(x, i) && bins.of(x) == bin) bl = min(bl, code_of(x)), bh = max(bh, code_of(x));
    });
    if (bh) atomicMin(&S.lo, bl), atomicMax(&S.hi, bh);
    __syncthreads();
    lo = S.lo, hi = S.hi;
    if (lo < hi) continue;

    // more equal tokens than the list holds: the first c of them, the last of which is found by bisection of the index
    uint64_t c = k - above;
    const float value = value_of(hi);
    if constexpr (MASS) {
      const uint64_t one = weight.mass(value);
      const double more = ceil(target) - (double)mass_above;      // the least whole mass beyond what lies above
      c = one ? ((uint64_t)fmax(more, 1.0) - 1) / one + 1 : n;
    }
    c = c < 1 ? 1 : c > n ? n : c;
    int a = 0, b = row.V - 1;
    while (a < b) {
      const int mid = a + (b - a) / 2;
      uint32_t upto = 0;
      row.each([&](float x, int i) { upto += x == value && i <= mid && cut.keeps(x, i); });
      for (int o = 32; o > 0; o >>= 1) upto += __shfl_xor(upto, o, kWave);
      __syncthreads();
      if (lane == 0) S.wave_count[wave] = upto;
      __syncthreads();
      uint32_t all = 0;
      for (int i = 0; i < kWaves; ++i) all += S.wave_count[i];
      if (all >= c) b = mid;
      else a = mid + 1;
    }
    __syncthreads();
    return Cut{value, a, false};
  }
}

// The cut at which the mass reaches `share` of the kept mass, and the mass that the cut and min_p keep: `sum`, of this thread's
// tokens above the cut's bin, and S.wave_kept, by wavefront, of those in it.  The bin is found from weights in fp32, and then
// its borders' masses are checked exactly: false where they do not hold the cut, or the bin holds more than the list.
template <class R>
__device__ __forceinline__ bool reach(const R &row, const Weight &weight, Shared &S, const Cut cut, float top, float bottom,
                                      double share, double scale, Cut &got, uint64_t &sum) {
  const int tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave;
  const Bins bins(code_of(fmaxf(bottom, cut.value)), code_of(top), true);
  const float s32 = (float)scale;
  auto rough = [&](float x) { return __builtin_amdgcn_exp2f((x - top) * s32); };
  float part = 0.f;
  row.each([&](float x, int i) { part += cut.keeps(x, i) ? rough(x) : 0.f; });
  part = wave_sum(part);
  __syncthreads();
  S.count[tid] = 0;
  if (lane == 0) S.wave_f[0][wave] = part;
  if (tid == 0) S.bin = -1, S.fill = 0;
  if (tid < kWaves) S.wave_kept[tid] = 0;
  __syncthreads();
  part = 0.f;
  for (int i = 0; i < kWaves; ++i) part += S.wave_f[0][i];
  const float unit = 0x1p30f / part;       // whole numbers, for an atomic addition of which the LDS takes 24 clocks (fp32: 240)
  row.each([&](float x, int i) {
    if (cut.keeps(x, i)) atomicAdd(&S.count[bins.of(x)], (uint32_t)(rough(x) * unit + 0.5f));
  });
  __syncthreads();
  const uint32_t mine = S.count[tid];
  uint32_t sums;
  const uint32_t upto = running(mine, S.wave_count, sums);
  const uint32_t reach = (uint32_t)fmaxf((float)share * (float)sums, 1.f);
  if (upto - mine < reach && reach <= upto) S.bin = tid;
  __syncthreads();
  const int bin = S.bin;
  if (bin < 0) return false;
  const bool some = weight.min_p > 0.0;      // min_p drops some of what top_p keeps
  uint64_t all = 0, above = 0;
  sum = 0;
  for (int j = 0; j < row.vecs; ++j)
    row.vec_where(j, row.vector(j), cut,
                  [&](float x, int i, bool keep) {
                    const double w = weight.weight(x);
                    const uint64_t m = keep ? weight.mass_of(w) : 0;
                    const int b = bins.of(x);
                    all += m;
                    above += b < bin ? m : 0;
                    if (some) sum += b < bin && w >= weight.min_p ? m : 0;
                    if (keep && b == bin && x >= kLowest) {
                      const uint32_t at = atomicAdd(&S.fill, 1u);
                      if (at < kList) S.list_x[at] = x, S.list_i[at] = i;
                    }
                  });
  sum = some ? sum : above;
  all = wave_sum64(all), above = wave_sum64(above);
  if (lane == 0) S.wave_mass[wave] = all;
  __syncthreads();
  uint64_t total = 0, over = 0;
  for (int i = 0; i < kWaves; ++i) total += S.wave_mass[i];
  const uint32_t n = S.fill;
  __syncthreads();
  if (lane == 0) S.wave_mass[wave] = above;
  if (n > kList || n == 0) return false;
  double w = 0.0;
  uint64_t mass = 0;
  if (tid < (int)n) w = weight.weight(S.list_x[tid]), S.list_w[tid] = mass = weight.mass_of(w);
  if (tid == 0) S.n = 0, S.total = 0;
  __syncthreads();
  for (int i = 0; i < kWaves; ++i) over += S.wave_mass[i];
  rank(S, (int)n, ByLogit());
  const double target = fmax(share * (double)total, 1.0);
  if (mass) atomicAdd((unsigned long long *)&S.total, (unsigned long long)mass);
  const bool keep = tid < (int)n && (double)(over + S.list_before[tid]) < target;
  if (keep) {
    atomicMax(&S.n, S.list_rank[tid]);
    if (w >= weight.min_p) atomicAdd((unsigned long long *)&S.wave_kept[S.list_i[tid] / (64 * R::W * row.vecs)], (unsigned long long)mass);
  }
  __syncthreads();
  if (!((double)over < target && target <= (double)(over + S.total))) return false;
  const uint32_t last = S.n;
  if (keep && S.list_rank[tid] == last) S.index = tid;
  __syncthreads();
  got = Cut{S.list_x[S.index], S.list_i[S.index], false};
  return true;
}

// The mass that the token's running mass has to exceed: of a total of up to 2^63, and for any u.
__device__ __forceinline__ uint64_t target_of(double u, uint64_t total) {
  const double aim = u * (double)total;
  if (aim >= (double)total) return total - 1;
  const uint64_t target = aim > 0.0 ? (uint64_t)aim : 0;
  return target < total ? target : total - 1;        // ((double)total may be above it)
}

// The distinct values of a bf16 row, from the largest down: kSide magnitudes below the largest one of either sign, and all that is
// nearer to zero as one in the middle (at 3,200, 25 binades, mostly zeros; at 1,088 a cut fell there in one row of 20).
constexpr int kSide = 3200, kCodes = 2 * kSide + 1;
struct Codes {
  uint32_t most;                       // the largest magnitude's bits, of the tokens from `low` on
  float low;                           // no token below it has a mass
  __device__ __forceinline__ Codes(float top, float low_) : low(low_) {
    most = max(__float_as_uint(fabsf(top)) >> 16, (__float_as_uint(fabsf(low_)) + 0xFFFFu) >> 16);
  }
  // (of a value outside low .. top: some code)
  __device__ __forceinline__ int of(float x) const {
    const uint32_t h = __float_as_uint(x) >> 16, d = most - (h & 0x7FFFu);
    return d < (uint32_t)kSide ? (int)(h > 0x8000u ? kCodes - 1 - d : d) : kSide;
  }
  __device__ __forceinline__ float value(int code) const {
    const uint32_t d = code < kSide ? code : kCodes - 1 - code, mag = most - d;
    return d > most || code == kSide ? -__builtin_inff() : __uint_as_float(mag << 16 | (code > kSide ? 0x80000000u : 0u));
  }
};

// The cut of top_k and top_p in a bf16 row: weights are formed once per distinct value, of which a row of 50,000 tokens has some
// 2,000, and summed by counts.  Tokens in the middle, a hundredth of them, have theirs formed one by one.  False where a cut lies
// among these, or more tokens than a list holds have the cut's value.
template <class R>
__device__ __forceinline__ bool cut_by_codes(const R &row, const Weight &weight, Shared &S, float top, float bottom,
                                             uint32_t top_k, double share, double scale, Cut &got) {
  static_assert(offsetof(Shared, wave_mass) - offsetof(Shared, mass) >= kCodes * sizeof(uint32_t));
  uint32_t *count = (uint32_t *)S.mass;
  const int tid = threadIdx.x, lane = tid % kWave;
  constexpr int W = R::W, EACH = (kCodes + kThreads - 1) / kThreads;
  const Codes codes(top, fmaxf(bottom, (float)fmax((double)kLowest, (double)top - 47.5 / scale)));
  __syncthreads();
  for (int i = tid; i < kCodes; i += kThreads) count[i] = 0;
  if (tid == 0) S.total = 0, S.n = 0;
  __syncthreads();
  uint64_t middle = 0;
  uint32_t number = 0;
  for (int j = 0; j < row.vecs; ++j) {
    const uint4 raw = row.vector(j);
    const int at = (row.first + 64 * j) * W;
    uint32_t bits = 0;
    row.vec(j, raw, [&](float x, int i) {
      const int code = codes.of(x);
      if (x >= codes.low) {
        if (code != kSide) atomicAdd(&count[code], 1u);
        else bits |= 1u << (i - at);
      }
    });
    number += __builtin_popcount(bits);
    row.each_bit(j, raw, bits, [&](float x, int, bool is) {
      const uint64_t m = weight.mass(x);
      middle += is ? m : 0;
    });
  }
  middle = wave_sum64(middle);
  for (int o = 32; o > 0; o >>= 1) number += __shfl_xor(number, o, kWave);
  if (lane == 0 && number) {
    atomicAdd((unsigned long long *)&S.total, (unsigned long long)middle);
    atomicAdd(&S.n, number);
  }
  __syncthreads();
  // The code that the cut falls into, and how many tokens of it are kept: found by the thread whose codes it is among.
  int cut = kCodes;
  uint32_t n = 0;
  const int first = EACH * tid, end = min(first + EACH, kCodes);
  auto tokens = [&](int code) { return code == kSide ? S.n : count[code]; };
  if (top_k > 0) {
    if (tid == 0) S.bin = kCodes;
    uint32_t sum = 0, all;
    for (int code = first; code < end; ++code) sum += tokens(code);
    const uint32_t upto = running(sum, S.wave_count, all);
    if (upto - sum < top_k && top_k <= upto) {
      uint32_t before = upto - sum;
      int code = first;
      while (before + tokens(code) < top_k) before += tokens(code++);
      S.bin = code, S.count_above = top_k - before;
    }
    __syncthreads();
    cut = S.bin, n = cut < kCodes ? S.count_above : 0;
    if (cut == kSide) return false;
    __syncthreads();
  }
  if (share < 1.0) {
    if (tid == 0) S.bin = kCodes;
    const int top_cut = cut;
    auto kept = [&](int code) { return code < top_cut ? tokens(code) : code == top_cut ? n : 0u; };
    auto mass = [&](int code) {
      const uint32_t c = kept(code);
      return c == 0 ? 0 : code == kSide ? S.total : c * weight.mass(codes.value(code));
    };
    uint64_t sum = 0, all;
    for (int code = first; code < end; ++code) sum += mass(code);
    const uint64_t upto = running(sum, S.wave_mass, all);
    const double target = fmax(share * (double)all, 1.0);
    if ((double)(upto - sum) < target && target <= (double)upto) {
      uint64_t before = upto - sum;
      int code = first;
      for (uint64_t m; code + 1 < end && (double)(before + (m = mass(code))) < target; ++code) before += m;
      const uint64_t one = code == kSide ? 0 : weight.mass(codes.value(code)), c = kept(code);
      const double more = ceil(target) - (double)before;        // the least whole mass beyond what lies above
      S.bin = code, S.count_above = (uint32_t)(one ? min(((uint64_t)fmax(more, 1.0) - 1) / one + 1, c) : c);
    }
    __syncthreads();
    if (S.bin < kCodes) cut = S.bin, n = S.count_above;
    if (cut == kSide) return false;
  }
  if (cut == kCodes) {                 // every token that has a mass
    got = Cut{codes.low, 0x7FFFFFFF, false};
    return true;
  }
  const float value = codes.value(cut);
  if (tid == 0) S.fill = count[cut];
  __syncthreads();
  const uint32_t all = S.fill;
  got = Cut{value, 0x7FFFFFFF, false};
  if (n >= all) return true;
  if (all > kList) return false;
  // the n-th of those in the vocabulary's order
  list(row, S, [&](float x, int) { return x == value; });
  if (tid < (int)all) S.list_w[tid] = 0;
  __syncthreads();
  rank(S, (int)all, ByIndex());
  if (tid < (int)all && S.list_rank[tid] == n - 1) S.index = S.list_i[tid];
  __syncthreads();
  got.index = S.index;
  return true;
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
  int top_k = A.top_k ? A.top_k[at] : A.top_k1;
  const double u = A.u[at];
  top_k = top_k > 0 && top_k < A.V ? top_k : 0;
  if (tid < kPowers) S.power[tid] = exp2(tid * (1.0 / kPowers));
  S.count[tid] = 0;

  float mine = -__builtin_inff(), top, bottom = -kLowest;        // this thread's largest
  row.load([&](float x, int) {
    mine = fmaxf(mine, x);
    bottom = x >= kLowest ? fminf(bottom, x) : bottom;
  });
  top = mine;
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

  const double scale = 1.4426950408889634074 / (double)temperature;
  const Weight weight{S.power, kPowers * scale, top, fmin((double)min_p, 1.0), top > kLowest ? kLowest : -__builtin_inff()};

  // 1. What may be kept as a list, where that is cheap and short.
  // (a list of more than 256 tokens takes longer to rank than a cut by the distinct values of a bf16 row does)
  constexpr int short_list = BF16 ? 256 : kList;
  float least = -__builtin_inff();                   // no token below it is kept
  bool shorter = true;
  if (top_k == 0 && min_p > 0.f) {                   // w >= min_p, with a margin for the logarithm's and this sum's rounding
    least = (float)fmax((double)kLowest, (double)top + log2(weight.min_p) / scale * 1.000001) - 1e-6f * fabsf(top);
    const uint32_t some = __builtin_popcountll(__builtin_amdgcn_ballot_w64(mine >= fmaxf(least, kLowest)));
    if (lane == 0) S.wave_count[wave] = some;
    __syncthreads();
    uint32_t threads = 0;                            // each of which has a token for the list
    for (int i = 0; i < kWaves; ++i) threads += S.wave_count[i];
    shorter = threads <= short_list;
  } else if (top_k > 0 && top_k <= short_list) {
    const Bins bins(code_of(bottom), code_of(top), true);
    if (mine >= kLowest) atomicAdd(&S.count[bins.of(mine)], 1u);
    if (tid == 0) S.bin = kBins;
    __syncthreads();
    const uint32_t c = S.count[tid];
    uint32_t total;
    const uint32_t upto = running(c, S.wave_count, total);
    if (upto - c < (uint32_t)top_k && (uint32_t)top_k <= upto) S.bin = tid;
    if (tid == 0) S.lo = 0xFFFFFFFFu;
    __syncthreads();
    // the least of the maxima down to that bin: as many tokens as there are maxima lie at or above it
    if (mine >= kLowest && bins.of(mine) <= S.bin) atomicMin(&S.lo, code_of(mine));
    __syncthreads();
    if (S.bin < kBins) least = fmaxf(least, value_of(S.lo));
  }
  const bool lists = (least > -__builtin_inff() || A.V <= short_list) && top_k <= short_list && shorter;
  const uint32_t n = lists ? list(row, S, [&](float x, int) { return x >= least && x >= kLowest; }) : kList + 1;
  if (n <= (uint32_t)short_list) {
    uint64_t kept = 0;                               // the mass that top_p is a share of
    if (top_k == 0 && top_p < 1.f) {
      uint64_t sum = 0;
      for (int j = 0; j < row.vecs; ++j)             // (nothing behind the row's end)
        row.vec(j, row.vector(j), [&](float x, int) { sum += weight.mass(x); });
      sum = wave_sum64(sum);
      if (lane == 0) S.wave_mass[wave] = sum;
      __syncthreads();
      for (int i = 0; i < kWaves; ++i) kept += S.wave_mass[i];
    }
    double w = 0.0;
    if (tid < (int)n) w = weight.weight(S.list_x[tid]), S.list_w[tid] = weight.mass_of(w);
    __syncthreads();
    rank(S, (int)n, ByLogit());
    const uint32_t place = tid < (int)n ? S.list_rank[tid] : kList;
    const uint64_t mass = tid < (int)n ? S.list_w[tid] : 0, ahead = tid < (int)n ? S.list_before[tid] : 0;
    bool keep = tid < (int)n && (top_k == 0 || place < (uint32_t)top_k);
    if (top_k > 0 && top_p < 1.f) {
      if (tid < (int)n && place == min((uint32_t)top_k, n) - 1) S.total = ahead + mass;
      __syncthreads();
      kept = S.total;
    }
    if (top_p < 1.f) keep = keep && (double)ahead < fmax((double)top_p * (double)kept, 1.0);
    keep = keep && w >= weight.min_p;
    if (tid < (int)n) S.list_w[tid] = keep ? mass : 0;
    __syncthreads();
    rank(S, (int)n, ByIndex());
    if (tid < (int)n && place == 0) S.total = 0;
    __syncthreads();
    if (keep) atomicAdd((unsigned long long *)&S.total, (unsigned long long)mass);
    __syncthreads();
    const uint64_t target = target_of(u, S.total);
    if (keep && S.list_before[tid] <= target && S.list_before[tid] + mass > target) A.token[at] = S.list_i[tid];
    return;
  }

  // 2. Cuts: by the distinct values, or by histograms.
  Cut cut{kLowest, 0x7FFFFFFF, true};
  bool found_cut = top_k == 0 && !(top_p < 1.f);
  if constexpr (BF16)
    if (!found_cut)
      found_cut = cut_by_codes(row, weight, S, top, bottom, (uint32_t)top_k, top_p < 1.f ? (double)top_p : 1.0, scale, cut);
  if (!found_cut) cut = Cut{kLowest, 0x7FFFFFFF, true};
  if (!found_cut && top_k > 0) cut = select<false>(row, weight, S, cut, top, bottom, (uint32_t)top_k, 0.0);
  uint64_t sum = 0;                                  // kept, of this thread
  bool summed = false;
  if (!found_cut && top_p < 1.f) {
    Cut got;
    if constexpr (!BF16) summed = reach(row, weight, S, cut, top, bottom, (double)top_p, scale, got, sum);
    cut = summed ? got : select<true>(row, weight, S, cut, top, bottom, 0u, (double)top_p);
  }
  sum = summed ? sum : 0;
  if (!summed)
    for (int j = 0; j < row.vecs; ++j)
      row.vec_where(j, row.vector(j), cut,
                    [&](float x, int, bool keep) {
                      const uint64_t m = weight.kept_mass(x);
                      sum += keep ? m : 0;
                    });
  sum = wave_sum64(sum);
  __syncthreads();
  if (lane == 0) S.wave_mass[wave] = sum + (summed ? S.wave_kept[wave] : 0);
  __syncthreads();
  uint64_t total = 0, before = 0;
  for (int i = 0; i < kWaves; ++i) total += S.wave_mass[i];
  const uint64_t target = target_of(u, total);
  int found = -1;
  // the found wavefront's vectors, by all of them
  for (int i = 0; i < kWaves && found < 0; ++i) {
    if (before + S.wave_mass[i] > target) found = i;
    else before += S.wave_mass[i];
  }
  for (int j0 = 0; j0 < row.vecs; j0 += kWaves) {
    const int j = j0 + wave;
    const bool in = j < row.vecs;
    uint4 raw{0, 0, 0, 0};
    uint64_t mine = 0;
    if (in) {
      raw = row.of_run(found, j);
      row.vec_of_run(found, j, raw, [&](float x, int i) {
        const uint64_t m = weight.kept_mass(x);
        mine += cut.keeps(x, i) ? m : 0;
      });
    }
    uint64_t run = mine;
#pragma unroll
    for (int o = 1; o < kWave; o *= 2) {
      const uint64_t b = shfl_up64(run, o);
      if (lane >= o) run += b;
    }
    __syncthreads();
    if (lane == kWave - 1) S.wave_kept[wave] = run;
    __syncthreads();
    uint64_t upto = before;
    for (int i = 0; i < wave; ++i) upto += S.wave_kept[i];
    for (int i = 0; i < kWaves; ++i) before += S.wave_kept[i];
    uint64_t mass = upto + run - mine;
    if (in && mass <= target && upto + run > target) {
      int64_t token = -1;
      row.vec_of_run(found, j, raw, [&](float x, int i) {
        const uint64_t m = weight.kept_mass(x);
        mass += cut.keeps(x, i) ? m : 0;
        if (token < 0 && mass > target) token = i;
      });
      A.token[at] = token;
    }
    if (before > target) return;
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
