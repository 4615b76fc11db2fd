// Causal attention over packed prompts of different lengths, with grouped heads, flash-style on the matrix cores:
// sequence b has the query rows cu_q[b] .. cu_q[b + 1] - 1 and the key rows cu_k[b] .. cu_k[b + 1] - 1; its T queries are the
// last of its S positions, so query t sees its keys 0 .. S - T + t:  y = softmax(scale q k^T) v, zeros where it sees none.
// Query head h reads key head h / (H / Hkv).
//
// Bound by the matrix and vector instructions together: per tile of 64 keys and 32 queries a wavefront has 36 matrix instructions
// of 16 clocks (68 with a head dim of 128) and 32 exponentials of 16 clocks beside some 70 other vector instructions of 4, so
// the two or three wavefronts of a SIMD overlap one kind with the other, matrix work first (s_setprio).  Measured on 8,192
// tokens, 32 heads: 1,049 TFLOP/s with a head dim of 128 and 911 with 64; a library product of 8,192 cubed reaches 1,385.
//
// A workgroup owns 128 consecutive query rows of one head, whichever sequences they belong to, and walks the key rows from
// the first one that any of them sees to the last: both ranges grow with the row, so they join up, and the grid follows from
// the number of rows alone, without the lengths on the host; the last rows start first, and heads that share keys on one XCD
// (835 -> 1,020 TFLOP/s on 6,001 and 5,000 tokens).  A lane finds its own query's range of keys by binary search in cu_q; tiles
// that hold keys outside some query's range are masked, per query.  (Tiles of their own for every sequence need the running sum
// of their tiles, and leave a part-filled tile per sequence.  Rows taken by the length of their walks, for compute units that all
// have long and short ones: 32 ragged prompts of 6 heads 62 -> 59 us, others 36 -> 37.)
//
// Products as in a causal prompt pass: S^T = K Q^T on v_mfma_f32_16x16x32_bf16 with the keys as M, so a lane (r, g) holds keys
// 4 g .. 4 g + 3 of each 16-key tile for ONE query (r), and the softmax is per lane; O^T = V^T P^T
// with the lane's own probabilities as operand, V^T through transposing LDS reads.  Statistics, scores and
// output sums in fp32, the probabilities' sum of the same rounded values on the matrix cores.
//
// Probabilities are rounded to bf16 once, as in the other prompt pass: the result's error against 64 bits is 1.2 to 1.4 times that
// of its own rounding.  A second term with what that rounding left, which single-token attention takes, would bring it to
// 1.0 and the products of two operands: 11,063 tokens, 32 heads of 128, 627 -> 872 us, 8,192 with 64 dims 293 -> 424.
//
// A masked key weighs exactly nothing, also where its value is an infinity or a NaN (0 times which is NaN): masked tiles sum
// their values' columns, and where a sum is not finite the values that are not are left out of the products and added key by key,
// for the queries that see the key.  So neither masked keys and values nor the queries beside it change a bit of a query's result.
// (Where its sequence lies may: tiles begin at the first key that any query of the workgroup sees, and the order of the sums with them.)
#include "lm_mm.h"

namespace smlm {
namespace {

typedef short short4_t __attribute__((ext_vector_type(4)));

constexpr int kNW = 4;          // wavefronts per workgroup,
constexpr int kQJ = 2;          // with kQJ * 16 query rows each
constexpr int kBM = 16 * kQJ * kNW;
constexpr int kBN = 64;         // keys per tile
constexpr int kCuLds = 512;     // entries of cu_q and cu_k kept in LDS

__device__ __forceinline__ uint2 read_tr16(const char *p) {
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                       (__attribute__((address_space(3))) short4_t *)(p)));
}

// a mask of those halves that are an infinity or a NaN of bf16
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
  return ((w & 0x7F800000u) == 0x7F800000u ? 0xFFFF0000u : 0u) | ((w & 0x7F80u) == 0x7F80u ? 0xFFFFu : 0u);
}

template <int J>
__device__ __forceinline__ float xor_lane_f(float v) { return __uint_as_float(xor_lane<J>(__float_as_uint(v))); }

struct PackedArgs {
  const uint16_t *q, *k, *v;
  uint16_t *y;
  int64_t qsn, qsh, ksn, ksh, vsn, vsh, ysn, ysh;   // strides over rows and heads, in elements
  const int *cu_q, *cu_k;
  int N, S, B, H, G;                                // G = H / Hkv
  int zero_rest;                                    // whether rows of no sequence are zeroed (else left as they are)
  float scale_log2;
};

template <int HD>
__global__ void __launch_bounds__(64 * kNW) __attribute__((amdgpu_waves_per_eu(HD <= 64 ? 3 : 2)))
    packed_attention_kernel(PackedArgs A) {
  constexpr int KS = HD / 32, MT = HD / 16, CPR = HD / 8, LPT = kBN * CPR / (64 * kNW), RB = CPR * 16, SW = CPR < 8 ? CPR : 8;
  __shared__ __align__(16) uint16_t sK[2][kBN * HD];
  __shared__ __align__(16) uint16_t sV[2][kBN * HD];
  __shared__ int s_cu[2][kCuLds];
  __shared__ int s_range[2][kNW];

  // the last rows first (of a long sequence the longest walks); heads that share keys on one XCD where they divide evenly
  const int slot = blockIdx.x % A.H, h = A.H % kMmXcds ? slot : slot % kMmXcds * (A.H / kMmXcds) + slot / kMmXcds;
  const int qt = (A.N + kBM - 1) / kBM - 1 - blockIdx.x / A.H;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, r = lane & 15, g = lane >> 4;
  const int q0 = qt * kBM, qw = q0 + wave * 16 * kQJ;
  const uint16_t *qb = A.q + h * A.qsh, *kb = A.k + h / A.G * A.ksh, *vb = A.v + h / A.G * A.vsh;

  // this wavefront's queries as B fragments: query row qw + 16 j + r, dims 32 s + 8 g .. +7
  bf16x8 bq[kQJ][KS];
#pragma unroll
  for (int j = 0; j < kQJ; ++j) {
    const int t = min(qw + 16 * j + r, A.N - 1);
#pragma unroll
    for (int s = 0; s < KS; ++s) bq[j][s] = *(const bf16x8 *)(qb + t * A.qsn + 32 * s + 8 * g);
  }

  // the keys [lo, hi) that query j of this lane sees; lo = hi where it sees none; owned: whether a sequence has its row
  const bool in_lds = A.B < kCuLds;
  if (in_lds)
    for (int i = tid; i <= A.B; i += 64 * kNW) s_cu[0][i] = A.cu_q[i], s_cu[1][i] = A.cu_k[i];
  __syncthreads();
  int lo[kQJ], hi[kQJ];
  bool owned[kQJ];
#pragma unroll
  for (int j = 0; j < kQJ; ++j) {
    const int i = qw + 16 * j + r;
    int b = 0, e = A.B + 1;          // entries of cu_q not above i
    while (b < e) {
      const int mid = (b + e) >> 1;
      if ((in_lds ? s_cu[0][mid] : A.cu_q[mid]) <= i) b = mid + 1;
      else e = mid;
    }
    owned[j] = i < A.N && b >= 1 && b <= A.B;
    lo[j] = hi[j] = 0;
    if (owned[j]) {
      const int end_q = in_lds ? s_cu[0][b] : A.cu_q[b];
      const int begin_k = in_lds ? s_cu[1][b - 1] : A.cu_k[b - 1], end_k = in_lds ? s_cu[1][b] : A.cu_k[b];
      lo[j] = min(max(begin_k, 0), A.S);
      hi[j] = (int)min(max((int64_t)end_k - end_q + i + 1, (int64_t)lo[j]), (int64_t)A.S);
      hi[j] = max(min(hi[j], end_k), lo[j]);
    }
  }
  // over the wavefront's queries, and the workgroup's: the first key that one sees, the end of the last
  int w_lo = 0x7FFFFFFF, w_hi = 0, all_lo = 0, all_hi = 0x7FFFFFFF;
#pragma unroll
  for (int j = 0; j < kQJ; ++j) {
    if (hi[j] > lo[j]) w_lo = min(w_lo, lo[j]), w_hi = max(w_hi, hi[j]);
    all_lo = max(all_lo, lo[j]), all_hi = min(all_hi, hi[j]);      // the keys that all of them see
  }
  auto over_rows = [&](int v, bool most) {
#define SMLM_STEP(J) { const int o = (int)xor_lane<J>((uint32_t)v); v = most ? max(v, o) : min(v, o); }
    SMLM_STEP(1) SMLM_STEP(2) SMLM_STEP(4) SMLM_STEP(8)
#undef SMLM_STEP
    return __builtin_amdgcn_readfirstlane(v);
  };
  w_lo = over_rows(w_lo, false), w_hi = over_rows(w_hi, true);
  all_lo = over_rows(all_lo, true), all_hi = over_rows(all_hi, false);
  if (lane == 0) s_range[0][wave] = w_lo, s_range[1][wave] = w_hi;
  __syncthreads();
  int begin = s_range[0][0], end = s_range[1][0];
#pragma unroll
  for (int i = 1; i < kNW; ++i) begin = min(begin, s_range[0][i]), end = max(end, s_range[1][i]);
  const int ntk = __builtin_amdgcn_readfirstlane(end > begin ? (end - begin + kBN - 1) / kBN : 0);
  begin = __builtin_amdgcn_readfirstlane(ntk ? begin : 0);

  float m[kQJ];     // finite: a query may see nothing of the first tiles
  const floatx4 zero4 = {0.f, 0.f, 0.f, 0.f};
  floatx4 lacc[kQJ];
#pragma unroll
  for (int j = 0; j < kQJ; ++j) m[j] = -3.0e38f, lacc[j] = zero4;
  const bf16x8 ones = __builtin_bit_cast(bf16x8, uint4{0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u});
  floatx4 oacc[MT][kQJ];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int j = 0; j < kQJ; ++j) oacc[mt][j] = zero4;

  // A tile goes straight into LDS (lane i of a wavefront's load writes bytes 16 i .. +15 of its 1 KB piece): LDS chunk
  // id = tid + 256 u is slot id % CPR of row id / CPR, which holds the row's chunk slot ^ (row % SW).  The descriptors
  // start at the tile's first row (64-bit) and end with row S - 1, behind which rows read as zeros.
  uint32_t koff[LPT], voff[LPT];
#pragma unroll
  for (int u = 0; u < LPT; ++u) {
    const int id = tid + 64 * kNW * u, row = id / CPR, c = (id % CPR) ^ (row % SW);
    koff[u] = (uint32_t)((row * A.ksn + 8 * c) * 2);
    voff[u] = (uint32_t)((row * A.vsn + 8 * c) * 2);
  }
  const uint32_t k_lds = (uint32_t)(uintptr_t)(lds_byte *)sK + wave * 1024, v_lds = (uint32_t)(uintptr_t)(lds_byte *)sV + wave * 1024;
  const uint16_t *kp = kb + begin * A.ksn, *vp = vb + begin * A.vsn;     // of the next tile
  const int64_t k_step = kBN * A.ksn, v_step = kBN * A.vsn;
  const int k_full = (int)(((kBN - 1) * A.ksn + HD) * 2), v_full = (int)(((kBN - 1) * A.vsn + HD) * 2);
  int left = ntk > 0 ? A.S - begin : 0, tiles_left = ntk;                // rows from there to the last; 0 behind the last tile
  // (Loads in inline assembly: behind the builtin's the compiler waits for them before every LDS read, so that they overlap
  // nothing.  Three tiles in LDS, a pipeline over half tiles, and 64 or 256 rows a workgroup were slower.)
  auto load_tile = [&](int buf) __attribute__((always_inline)) {
    intx4 krs{(int)(uint32_t)(uintptr_t)kp, (int)((uint64_t)(uintptr_t)kp >> 32), k_full, 0x00020000};
    intx4 vrs{(int)(uint32_t)(uintptr_t)vp, (int)((uint64_t)(uintptr_t)vp >> 32), v_full, 0x00020000};
    if (left < kBN) {
      krs[2] = left > 0 ? (int)(((left - 1) * A.ksn + HD) * 2) : 0;
      vrs[2] = left > 0 ? (int)(((left - 1) * A.vsn + HD) * 2) : 0;
    }
    kp += k_step, vp += v_step, left = --tiles_left > 0 ? left - kBN : 0;
#pragma unroll
    for (int u = 0; u < LPT; ++u) {
      mm_load_lds(krs, koff[u], k_lds + buf * (kBN * HD * 2) + u * (64 * kNW * 16));
      mm_load_lds(vrs, voff[u], v_lds + buf * (kBN * HD * 2) + u * (64 * kNW * 16));
    }
  };
  load_tile(0);

  for (int tk = 0; tk < ntk; ++tk) {
    const int kv0 = begin + tk * kBN, buf = tk & 1;
    mm_wait_barrier<0>();     // this tile has landed, and all have read the one before
    load_tile(buf ^ 1);

    if (kv0 < w_hi && kv0 + kBN > w_lo) {
      const bool masked = kv0 < all_lo || kv0 + kBN > all_hi;

      __builtin_amdgcn_s_setprio(1);
      // S^T: sacc[kt][j][i] = q(query 16 j + r) . k(key kv0 + 16 kt + 4 g + i)
      floatx4 sacc[4][kQJ];
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int j = 0; j < kQJ; ++j) sacc[kt][j] = zero4;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        bf16x8 a[4];
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) {
          const int row = 16 * kt + r;
          a[kt] = *(const bf16x8 *)((const char *)sK[buf] + row * RB + (((4 * s + g) ^ (row % SW)) * 16));
        }
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
          for (int j = 0; j < kQJ; ++j)
            sacc[kt][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[kt], bq[j][s], sacc[kt][j], 0, 0, 0);
      }

      __builtin_amdgcn_s_setprio(0);
      if (masked) {
#pragma unroll
        for (int j = 0; j < kQJ; ++j)
#pragma unroll
          for (int kt = 0; kt < 4; ++kt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int key = kv0 + 16 * kt + 4 * g + i;
              if ((uint32_t)(key - lo[j]) >= (uint32_t)(hi[j] - lo[j])) sacc[kt][j][i] = -__builtin_inff();
            }
      }
      // P^T as B fragments: 32-key step ks = key tiles 2 ks and 2 ks + 1, slots 4 g .. and 16 + 4 g .. of them.  Leaves the or
      // of their bits, in which 0x40004000 is set where one is 2 or more (an infinity or a NaN too).
      bf16x8 bp[kQJ][2];
      uint32_t bits[kQJ];
      auto probabilities = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < kQJ; ++j) {
          bits[j] = 0;
#pragma unroll
          for (int ks = 0; ks < 2; ++ks) {
            uint32_t u[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float p[2];
#pragma unroll
              for (int i = 0; i < 2; ++i)
                p[i] = __builtin_amdgcn_exp2f(sacc[2 * ks + e / 2][j][2 * (e % 2) + i] * A.scale_log2 - m[j]);
              u[e] = pack_bf16x2(p[0], p[1]);
              bits[j] |= u[e];
            }
            bp[j][ks] = __builtin_bit_cast(bf16x8, uint4{u[0], u[1], u[2], u[3]});
          }
        }
      };
      // Online softmax per query (lane), in the log2 domain, with a reference point m that starts 2^8 above the first tile's
      // maximum and moves, to 2^8 above a tile's, only when an exponential reaches 2: a test of the operands' bits stands in
      // for the maximum of every tile (head dim 64: 753 -> 800 TFLOP/s).  Each query by itself, whatever its neighbours do.
      probabilities();
      if (__builtin_amdgcn_ballot_w64(((bits[0] | bits[1]) & 0x40004000u) != 0)) {
        static_assert(kQJ == 2);
#pragma unroll
        for (int j = 0; j < kQJ; ++j) {
          uint32_t own = bits[j] & 0x40004000u;      // whether one of this query's is
          own |= xor_lane<16>(own);
          own |= xor_lane<32>(own);
          float a = -__builtin_inff();
#pragma unroll
          for (int i = 0; i < 16; ++i) a = fmaxf(a, sacc[i / 4][j][i % 4]);
          a = fmaxf(a, xor_lane_f<16>(a));
          a = fmaxf(a, xor_lane_f<32>(a)) * A.scale_log2;
          const float mnew = own && a - m[j] > 0.99f ? a + 8.f : m[j];
          const float alpha = __builtin_amdgcn_exp2f(m[j] - mnew);
          lacc[j] *= alpha;
          m[j] = mnew;
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) oacc[mt][j] *= alpha;
        }
        probabilities();
      }
#pragma unroll
      for (int j = 0; j < kQJ; ++j)
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
          lacc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, bp[j][ks], lacc[j], 0, 0, 0);

      // V^T fragment of dims 16 mt + r at the 32-key step's keys in the same slots, by transposing reads
      auto values = [&](int ks, int mt) {
        const int row = 32 * ks + 4 * g + r / 4, dim = 16 * mt + 4 * (r % 4);
        const char *src = (const char *)sV[buf] + row * RB + (((dim / 8) ^ (row % SW)) * 16) + (dim % 8) * 2;
        const uint2 a = read_tr16(src), b = read_tr16(src + 16 * RB);
        return uint4{a.x, a.y, b.x, b.y};
      };
      bool odd = false;
      if (masked) {
        floatx4 sums[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          sums[mt] = zero4;
#pragma unroll
          for (int ks = 0; ks < 2; ++ks)
            sums[mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, values(ks, mt)), ones, sums[mt], 0, 0, 0);
        }
        bool fine = true;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int i = 0; i < 4; ++i) fine = fine && fabsf(sums[mt][i]) < __builtin_inff();
        odd = __builtin_amdgcn_ballot_w64(!fine) != 0;
      }
      if (!odd) {
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            const bf16x8 a = __builtin_bit_cast(bf16x8, values(ks, mt));
#pragma unroll
            for (int j = 0; j < kQJ; ++j)
              oacc[mt][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, bp[j][ks], oacc[mt][j], 0, 0, 0);
          }
        __builtin_amdgcn_s_setprio(0);
      } else {
#pragma unroll 1
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            const uint4 w = values(ks, mt);
            const bf16x8 a = __builtin_bit_cast(bf16x8, uint4{w.x & ~not_finite(w.x), w.y & ~not_finite(w.y), w.z & ~not_finite(w.z),
                                                              w.w & ~not_finite(w.w)});
#pragma unroll
            for (int j = 0; j < kQJ; ++j)
              oacc[mt][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, ks ? bp[j][1] : bp[j][0], oacc[mt][j], 0, 0, 0);
          }
#pragma unroll 1
        for (int at = 0; at < kBN; ++at) {
          // the operand slot that holds key `at` of the tile: 16-bit half `slot % 2` of register slot / 2, in lane group `group`
          const int ks = at >> 5, group = (at >> 2) & 3, slot = (at & 3) + ((at >> 4) & 1) * 4;
          const uint32_t half = slot & 1 ? 0xFFFF0000u : 0x0000FFFFu;
          const bool mine = g == group;
          const uint4 keep{mine && slot / 2 == 0 ? half : 0u, mine && slot / 2 == 1 ? half : 0u,
                           mine && slot / 2 == 2 ? half : 0u, mine && slot / 2 == 3 ? half : 0u};
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            uint4 a = values(ks, mt);
            a = uint4{a.x & keep.x & not_finite(a.x), a.y & keep.y & not_finite(a.y), a.z & keep.z & not_finite(a.z),
                      a.w & keep.w & not_finite(a.w)};
#pragma unroll
            for (int j = 0; j < kQJ; ++j) {
              const uint4 p = __builtin_bit_cast(uint4, ks ? bp[j][1] : bp[j][0]);
              const bf16x8 b = __builtin_bit_cast(bf16x8, uint4{p.x & keep.x, p.y & keep.y, p.z & keep.z, p.w & keep.w});
              const floatx4 one = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), b, zero4, 0, 0, 0);
              const bool seen = kv0 + at >= lo[j] && kv0 + at < hi[j];
#pragma unroll
              for (int i = 0; i < 4; ++i) oacc[mt][j][i] = seen ? oacc[mt][j][i] + one[i] : oacc[mt][j][i];
            }
          }
        }
      }
    }
  }
  mm_finish();

  // y: lane (r, g) holds dims 16 mt + 4 g .. +3 of query row qw + 16 j + r
#pragma unroll
  for (int j = 0; j < kQJ; ++j) {
    const int t = qw + 16 * j + r;
    if (t >= A.N || (!owned[j] && !A.zero_rest)) continue;
    const float inv = hi[j] > lo[j] ? 1.0f / lacc[j][0] : 0.f;
    uint16_t *yr = A.y + t * A.ysn + h * A.ysh;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const floatx4 o = oacc[mt][j];
      uint2 out{pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv)};
      *(uint2 *)(yr + 16 * mt + 4 * g) = out;
    }
  }
}

template <int HD>
void launch(const PackedArgs &A, hipStream_t s) {
  constexpr int rows = kBM;
  hipLaunchKernelGGL((packed_attention_kernel<HD>), dim3((unsigned)((A.N + rows - 1) / rows * A.H)), dim3(64 * kNW), 0, s, A);
}

}  // namespace
}  // namespace smlm

extern "C" int smlm_packed_attention(const void *q, const int64_t *q_strides, const void *k, const int64_t *k_strides,
                                     const void *v, const int64_t *v_strides, const int *cu_q, const int *cu_k, int64_t B,
                                     int64_t N, int64_t S, int H, int kv_heads, int head_dim, float scale, void *y,
                                     const int64_t *y_strides, int zero_rest, void *stream) {
  using namespace smlm;
  const char *name = "smlm_packed_attention";
  if (!q || !y || !q_strides || !k_strides || !v_strides || !y_strides || !cu_q || !cu_k || (S > 0 && (!k || !v)))
    return fail(SMLM_EINVAL, "%s: null pointer argument", name);
  if (B < 0 || N < 0 || S < 0 || H < 1 || H > 65536 || kv_heads < 1 || H % kv_heads)
    return fail(SMLM_EINVAL, "%s: bad shape B=%lld N=%lld S=%lld H=%d kv_heads=%d", name, (long long)B, (long long)N,
                (long long)S, H, kv_heads);
  if (head_dim != 32 && head_dim != 64 && head_dim != 128)
    return fail(SMLM_EUNSUPPORTED, "%s: head_dim %d not in {32, 64, 128}", name, head_dim);
  // rows are numbered, and a tile's rows addressed, in 32 bits
  if (B > (1 << 30) || N > (1 << 30) || S > (1 << 30) || (N + 63) / 64 * H > 0x7FFFFFFFLL)
    return fail(SMLM_EUNSUPPORTED, "%s: more than 2^30 rows, or 2^31 workgroups", name);
  const int64_t *st[4] = {q_strides, k_strides, v_strides, y_strides};
  for (int a = 0; a < 4; ++a)
    for (int i = 0; i < 2; ++i)
      if (st[a][i] < 0 || st[a][i] % (a == 3 ? 4 : 8) || st[a][i] > (1 << 22))
        return fail(SMLM_EINVAL, "%s: strides must be multiples of 8 elements (4 for y) from 0 to 2^22; got %lld", name,
                    (long long)st[a][i]);
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v) % 16 || (uintptr_t)y % 8 || ((uintptr_t)cu_q | (uintptr_t)cu_k) % 4)
    return fail(SMLM_EINVAL, "%s: q, k, v must be 16-byte and y 8-byte aligned", name);
  if (!(scale > 0.f) || scale > 1e38f) return fail(SMLM_EINVAL, "%s: the scale must be positive, at most 1e38", name);
  if (N == 0 || (B == 0 && !zero_rest)) return SMLM_OK;
  const PackedArgs A{(const uint16_t *)q, (const uint16_t *)k, (const uint16_t *)v, (uint16_t *)y, q_strides[0], q_strides[1],
                     k_strides[0], k_strides[1], v_strides[0], v_strides[1], y_strides[0], y_strides[1], cu_q, cu_k, (int)N,
                     (int)S, (int)B, H, H / kv_heads, zero_rest, scale * 1.4426950408889634f};
  switch (head_dim) {
    case 32: launch<32>(A, (hipStream_t)stream); break;
    case 64: launch<64>(A, (hipStream_t)stream); break;
    default: launch<128>(A, (hipStream_t)stream); break;
  }
  return launch_status(name);
}
