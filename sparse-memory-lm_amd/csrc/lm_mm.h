// The K loop of the training step's products on the matrix cores (v_mfma_f32_16x16x32_bf16, fp32 sums): a tile of
// kT rows ("tokens") x kF columns ("features") from two bf16 operands, each of which may have the summed dimension k
// contiguous (rows of k: a linear layer's input and weight) or strided (rows of tokens or features, k the slow dimension:
// the operands of a weight's gradient).
//
// Workgroup = WF x WT wavefronts over the tile, 16 NI features x 16 NJ tokens each.  What bounds the loop is the way from
// the vector cache into LDS, 64 bytes per clock and CU: a chunk of 32 k takes (kF + kT) clocks of it and kF kT / 64 of the
// matrix cores.  Hence tiles of 256 x 256 or 384 x 128 where there are enough of them (half and two thirds of the products'
// time; 128 x 128 takes all of it), by eight wavefronts, two per SIMD, one workgroup a CU; and rows of 64 k, whole cache
// lines, where k is contiguous (rows of 32 k: 900 TFLOP/s on 8,192 cubed with both operands so, 1,260 with neither).
//
// k streams through LDS, loaded straight from memory (buffer_load ... lds, no registers in between), in stages of 64 k (two
// of them) or 32 (three, for products without long contiguous rows on both sides), and is multiplied in steps of 32.  While
// a step's products run, the next step's fragments are read into a second set of registers; behind the barrier before a
// stage's last step, by which all wavefronts have read the stage, a later one is loaded into it, the loads spread between
// the step's products.  Neither LDS nor memory latency stands between two steps' products.
//
// LDS layouts (16-byte pieces; 64 banks, 256 bytes; ds_read_b128 serves lanes 0-3, 12-15 and 20-27 of each 32 together,
// then the others):
//   k contiguous: 128-byte rows, piece c of row R at c ^ swz(R), so that the lanes served together fall on distinct banks.
//     Feature rows may be read permuted (mm_feature): row groups 2 p and 2 p + 1 then leave each lane 8 consecutive features
//     of a token in its accumulators, and the four lanes of a token 32: stores of 16 bytes a lane, 64 a token.
//   k strided: rows of kF or kT, piece c of row k at c ^ vsw(k), read with ds_read_b64_tr_b16, which gives lane r four k of
//     column r.  Lane group g takes k = 8 g .. 8 g + 7 of a step in both layouts.
// Out of range rows and k read as zeros (the buffer's record count; the k beyond the end of contiguous rows by an offset
// out of range), so tails need no other care than not storing what lies outside.
#pragma once

#include "pkm_common.h"

#include <atomic>

namespace smlm {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef int intx4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) unsigned char lds_byte;

constexpr int kMmStep = 32, kMmUnit = 64, kMmXcds = 8;    // k of a step; sums are padded with zeros to whole units
constexpr int kMmMaxStride = 1 << 21;         // elements: a tile's byte offsets stay below 2^31

// 16 bytes per lane from a buffer straight into LDS at lds + 16 * lane (wave-uniform lds).  Inline assembly, so that the
// compiler adds no wait for it before every LDS read; the kernels wait themselves (mm_wait_barrier).
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void mm_load_lds(intx4 rsrc, uint32_t voff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(voff), "s"(rsrc), "s"(lds)
               : "m0");
}
#pragma clang diagnostic pop

// At most N vector memory operations on their way and every LDS read done; then the barrier.  Loads complete in order:
// with N = the loads issued after a stage's, that stage has landed.
template <int N>
__device__ __forceinline__ void mm_wait_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | ((N >> 4) << 14));
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
// No load is on its way into LDS when the workgroup ends.
__device__ __forceinline__ void mm_finish() { __builtin_amdgcn_s_waitcnt(0x0F70); }

constexpr uint32_t kMmOutside = 0xFFFFFFF0u;  // an offset that no record count reaches

template <int WF_, int WT_, int NI_, int NJ_>
struct MmShape {
  static constexpr int WF = WF_, WT = WT_, NI = NI_, NJ = NJ_;
  static constexpr int kThreads = 64 * WF * WT, kF = 16 * WF * NI, kT = 16 * WT * NJ;
  // the wavefront's first feature and token in the tile
  static __device__ __forceinline__ int feature(int wave) { return wave % WF * 16 * NI; }
  static __device__ __forceinline__ int token(int wave) { return wave / WF * 16 * NJ; }
};

// First of the four features of row group i in lane group g's accumulators.
template <bool PERM>
__device__ __forceinline__ constexpr int mm_feature(int i, int g) {
  return PERM ? 32 * (i / 2) + 8 * g + 4 * (i % 2) : 16 * i + 4 * g;
}

// One operand's LDS tile of ROWS rows (tokens or features) x K k (32 or 64).  PERM: its fragments are permuted.
template <int ROWS, bool KC, bool PERM, int THREADS, int K>
struct MmTile {
  static constexpr bool kContiguous = KC;
  static constexpr int kK = K, kRows = ROWS, kBytes = ROWS * K * 2, kPerLoad = THREADS * 16;
  static constexpr int kLoads = kBytes / kPerLoad;                   // per thread and stage
  static constexpr int kRowBytes = KC ? K * 2 : ROWS * 2;
  static_assert(kBytes % kPerLoad == 0, "a whole number of loads");

  static __device__ __forceinline__ int swz(int row) {               // KC
    if constexpr (K == 32) return -(PERM ? row / 8 : row / 4) & 3;
    else return PERM ? (row >> 1 & 1) | (row / 8 & 3) << 1 : row >> 1 & 7;
  }
  static __device__ __forceinline__ int vsw(int k) {                 // k strided
    return ROWS % 128 == 0 ? 2 * ((k & 3) | (k >> 3 & 1) << 2) : 2 * ((k >> 1 & 1) | (k >> 3 & 1) << 1);
  }

  // Loads whose offsets are kept: contiguous rows have one, the loads' rows are kRowStep apart with one swizzle, and the
  // step goes into the (wave-uniform) descriptor.
  static constexpr int kRowStep = KC ? kPerLoad / kRowBytes : 0, kOffsets = KC ? 1 : kLoads;
  static_assert(!KC || (kRowStep % 32 == 0), "one swizzle for all loads");
  // This thread's byte offset of load u (KC: 0) from the stage's (the load's) first byte in memory; its first k (KC).
  static __device__ __forceinline__ uint32_t offset(int u, int tid, int64_t ld) {
    const int at = u * kPerLoad + tid * 16, row = at / kRowBytes, c = at % kRowBytes / 16;
    if constexpr (KC) return (uint32_t)(row * ld * 2 + (c ^ swz(row)) * 16);
    else return (uint32_t)(row * ld * 2 + (c ^ vsw(row)) * 16);
  }
  static __device__ __forceinline__ int first_k(int tid) {
    const int at = tid * 16;
    return 8 * (at % kRowBytes / 16 ^ swz(at / kRowBytes));
  }

  // LDS address (from the tile's base) that lane (r, g) reads the wavefront's row group i from, its rows starting at w0,
  // in step h (0, 1) of the stage.  KC: i only adds to it; k strided: h does.
  static __device__ __forceinline__ uint32_t at_contiguous(int w0, int h, int r, int g) {
    const int R = PERM ? w0 + 8 * (r / 4) + r % 4 : w0 + r;          // w0 a multiple of 32 or 16
    return R * kRowBytes + (((K == 32 ? 0 : 4 * h) + g) ^ swz(R)) * 16;
  }
  static __device__ __forceinline__ uint32_t at_strided(int w0, int i, int r, int g) {
    const int k = 8 * g + r / 4;
    const int col = w0 + mm_feature<PERM>(i, r % 4);
    return k * kRowBytes + (col / 8 ^ vsw(k)) * 16 + col % 8 * 2;
  }
  template <int N>
  static __device__ __forceinline__ void addresses(uint32_t (&a)[N], uint32_t base, int w0, int r, int g) {
#pragma unroll
    for (int i = 0; i < N; ++i) a[i] = base + (KC ? at_contiguous(w0, i & 1, r, g) : at_strided(w0, i, r, g));
  }
  // Row group i, step h, of the stage at byte `stage`, from the addresses above (KC uses the first two).
  template <int N>
  static __device__ __forceinline__ bf16x8 frag(const uint32_t (&a)[N], int i, int h, uint32_t stage) {
    if constexpr (KC) {
      return *(const __attribute__((address_space(3))) bf16x8 *)(uintptr_t)(a[h] + stage + mm_feature<PERM>(i, 0) * kRowBytes);
    } else {
      typedef __attribute__((address_space(3))) bf16x4 *p4;
      const uint32_t at = a[i] + stage + h * 32 * kRowBytes;
      const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((p4)(uintptr_t)at);
      const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((p4)(uintptr_t)(at + 4 * kRowBytes));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
};

// Where an operand's next stage comes from: wave-uniform, stepped from stage to stage.  `left` is exact: the bytes from the
// stage's first to the operand's last, which the record count of its loads is clipped to: past the end they read zeros.
template <class O>
struct MmSource {
  const uint16_t *p;
  int64_t left, step, k, rows_step;                      // steps in bytes; k: what is left of the sum
  // rows from row0 (< rows) on and k from k0 (< K) on of an operand of `rows` rows and K
  __device__ __forceinline__ void init(const uint16_t *base, int64_t ld, int64_t rows, int64_t K, int64_t row0, int64_t k0) {
    const int64_t major = O::kContiguous ? row0 : k0, minor = O::kContiguous ? k0 : row0;
    p = base + major * ld + minor;
    left = (((O::kContiguous ? rows : K) - 1 - major) * ld + (O::kContiguous ? K : rows) - minor) * 2;
    step = O::kContiguous ? O::kK * 2 : O::kK * 2 * ld;
    rows_step = O::kRowStep * ld * 2;
    k = K - k0;
  }
  // Descriptor of load u.
  __device__ __forceinline__ intx4 rsrc(int u) const {
    const uint64_t a = (uint64_t)p + u * rows_step;
    const int64_t more = left - u * rows_step;
    const uint32_t n = more >> 32 ? 0xFFFFFFF0u : (uint32_t)more;
    return intx4{(int)(uint32_t)a, (int)(uint32_t)(a >> 32), (int)(more <= 0 ? 0u : n), 0x00020000};
  }
  __device__ __forceinline__ void next() {
    p += step / 2;
    left -= step;
    k -= O::kK;
  }
};

template <int NI, int NJ>
struct MmFrags {
  bf16x8 a[NI], b[NJ];
};

// The loop's state of one thread for a feature tile F and a token tile T: a stage holds F, then T.
template <class F, class T, int NI, int NJ>
struct MmLoop {
  static_assert(F::kK == T::kK, "one stage");
  static constexpr int kK = F::kK, kStages = kK == 32 ? 3 : 2;
  static constexpr int kStage = F::kBytes + T::kBytes, kLoads = F::kLoads + T::kLoads, kLds = kStages * kStage;
  static constexpr int kFa = F::kContiguous ? 2 : NI, kTa = T::kContiguous ? 2 : NJ;
  typedef MmFrags<NI, NJ> Frags;
  uint32_t fo[F::kOffsets], to[T::kOffsets], fa[kFa], ta[kTa], lds;

  __device__ __forceinline__ void offsets(int64_t ldf, int64_t ldt) {
#pragma unroll
    for (int u = 0; u < F::kOffsets; ++u) fo[u] = F::offset(u, threadIdx.x, ldf);
#pragma unroll
    for (int u = 0; u < T::kOffsets; ++u) to[u] = T::offset(u, threadIdx.x, ldt);
  }
  // wf, wt: first feature and token row of this wavefront in the tile
  __device__ __forceinline__ void init(const unsigned char *smem, int64_t ldf, int64_t ldt, int wf, int wt) {
    const int lane = threadIdx.x % kWave, r = lane & 15, g = lane >> 4;
    const uint32_t base = (uint32_t)(uintptr_t)(lds_byte *)smem;
    offsets(ldf, ldt);
    F::addresses(fa, base, wf, r, g);
    T::addresses(ta, base + F::kBytes, wt, r, g);
    lds = base + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave) * 1024;
  }

  // The last stage of contiguous rows: the pieces from the sum's end on come from outside, as zeros, from now on.
  template <class O>
  static __device__ __forceinline__ void clip(const MmSource<O> &s, uint32_t *off) {
    if (O::kContiguous && s.k < O::kK)                   // wave-uniform
      off[0] = O::first_k(threadIdx.x) < s.k ? off[0] : kMmOutside;
  }
  // Load u of an operand's next stage to `at`, the place of its first.
  template <class O>
  static __device__ __forceinline__ void load_one(const MmSource<O> &s, const uint32_t *off, int u, uint32_t at) {
    mm_load_lds(s.rsrc(u), off[O::kContiguous ? 0 : u], at + u * O::kPerLoad);
  }
  // Load l of the sources' next stage (F's first) into `stage`.
  __device__ __forceinline__ void load(int l, const MmSource<F> &f, const MmSource<T> &t, uint32_t stage) const {
    if (l < F::kLoads) load_one(f, fo, l, lds + stage);
    else load_one(t, to, l - F::kLoads, lds + stage + F::kBytes);
  }
  __device__ __forceinline__ void issue(MmSource<F> &f, MmSource<T> &t, uint32_t stage) {
    clip(f, fo);
    clip(t, to);
#pragma unroll
    for (int l = 0; l < kLoads; ++l) load(l, f, t, stage);
    f.next();
    t.next();
  }
  // Part i of NI of step h's fragments.
  __device__ __forceinline__ void read_part(Frags &x, uint32_t stage, int h, int i) const {
    x.a[i] = F::frag(fa, i, h, stage);
#pragma unroll
    for (int j = 0; j < NJ; ++j)
      if (j >= i * NJ / NI && j < (i + 1) * NJ / NI) x.b[j] = T::frag(ta, j, h, stage);
  }
  __device__ __forceinline__ void read(Frags &x, uint32_t stage, int h) const {
#pragma unroll
    for (int i = 0; i < NI; ++i) read_part(x, stage, h, i);
  }
  // The products of `cur`, with between(i), i < NI, spread between them.
  template <class BETWEEN>
  static __device__ __forceinline__ void products(const Frags &cur, floatx4 (&acc)[NI][NJ], BETWEEN between) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      between(i);
#pragma unroll
      for (int j = 0; j < NJ; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(cur.a[i], cur.b[j], acc[i][j], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  // Fills the stages and reads the first step's fragments.
  __device__ __forceinline__ void start(MmSource<F> &f, MmSource<T> &t, Frags &x) {
#pragma unroll
    for (int q = 0; q < kStages; ++q) issue(f, t, q * kStage);
    mm_wait_barrier<(kStages - 1) * kLoads>();
    read(x, 0, 0);
  }
  static __device__ __forceinline__ uint32_t after(uint32_t stage) {
    return stage == (kStages - 1) * kStage ? 0 : stage + kStage;
  }
  // The last step of the stage at `here`, its fragments in `cur`: reads the first step of the stage behind it into `next`
  // and loads the sources' next stage into its own place.
  __device__ __forceinline__ void last_step(MmSource<F> &f, MmSource<T> &t, const Frags &cur, Frags &next, uint32_t here,
                                            floatx4 (&acc)[NI][NJ]) {
    mm_wait_barrier<(kStages - 2) * kLoads>();           // the next stage has landed, all have read this one
    clip(f, fo);
    clip(t, to);
    const uint32_t there = after(here);
    products(cur, acc, [&](int i) {
#pragma unroll
      for (int l = 0; l < kLoads; ++l)
        if (l >= i * kLoads / NI && l < (i + 1) * kLoads / NI) load(l, f, t, here);
      read_part(next, there, 0, i);
    });
    f.next();
    t.next();
  }
  // The products of a unit of 64 k from the stage at `stage` on, whose first step's fragments are in x: leaves the next
  // unit's in x.
  __device__ __forceinline__ void multiply(MmSource<F> &f, MmSource<T> &t, Frags &x, Frags &y, uint32_t &stage,
                                           floatx4 (&acc)[NI][NJ]) {
    if constexpr (kK == 32) {
      last_step(f, t, x, y, stage, acc);
      stage = after(stage);
    } else {
      products(x, acc, [&](int i) { read_part(y, stage, 1, i); });
    }
    last_step(f, t, y, x, stage, acc);
    stage = after(stage);
  }
};

template <int NI, int NJ>
__device__ __forceinline__ void mm_zero(floatx4 (&acc)[NI][NJ]) {
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
}

// Tile t of `n`, so that each XCD (workgroup id % 8) walks neighbours; -1 for the padding of the grid (mm_grid).
__device__ __forceinline__ int mm_tile_of(unsigned id, unsigned n) {
  const unsigned per = (n + kMmXcds - 1) / kMmXcds, t = id % kMmXcds * per + id / kMmXcds;
  return id / kMmXcds < per && t < n ? (int)t : -1;
}
inline int64_t mm_grid(int64_t n) { return (n + kMmXcds - 1) / kMmXcds * kMmXcds; }

__device__ __forceinline__ int mm_units(int64_t k) { return (int)((k + kMmUnit - 1) / kMmUnit); }
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Lets a kernel use `bytes` of dynamic LDS, more than the 64 KB that need no permission: once per kernel and device (the
// call costs as much as a launch).  done: the kernel's own, a bit per device.
inline int mm_allow_lds(const void *kernel, int bytes, std::atomic<uint64_t> &done, const char *what) {
  if (bytes <= 65536) return SMLM_OK;
  int device = 0;
  hipError_t e = hipGetDevice(&device);
  const uint64_t bit = 1ull << (device & 63);
  if (e == hipSuccess && !(device < 64 && (done.load(std::memory_order_relaxed) & bit))) {
    e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == hipSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  }
  return e == hipSuccess ? SMLM_OK : fail(SMLM_EHIP, "%s: %s", what, hipGetErrorString(e));
}

// Terms that an operand formed on the way (the activation, the logits' gradient) is held in: bf16, and for few tokens a
// second bf16 with what the first leaves, 16 bits of mantissa together.  Over many tokens the first's roundings average out
// in the sums (a result's error is 1.4 of its own rounding's); of a few tokens single values carry a result, whose error
// would be up to twice that, and the products are bound by the weights' bytes and the launches: the second terms cost the
// loss of 64 tokens 56 -> 61 us and an FFN block of 48 tokens 36 -> 41, both less than the calls take on the host; at 512 tokens
// the loss' two products would take twice as long.
constexpr int64_t kMmFewTokens = 128;
inline int mm_terms(int64_t tokens) { return tokens <= kMmFewTokens ? 2 : 1; }
__device__ __forceinline__ uint4 mm_pack(const float *v) {
  return uint4{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
}
// v - bf16(v), exact: the second term.  What is not finite stays in the first alone.
__device__ __forceinline__ float mm_rest(float v) {
  const float rest = v - round_bf16_hw(v);
  return fabsf(rest) < __builtin_inff() ? rest : 0.f;
}

// ---- plain products (lm_mm.hip) ----------------------------------------------------------------------------------------
// out[t, f] = sum_k tok[t, k] feat[f, k]; an operand with *_kc = false is stored [k][row].  Rows and strides in elements,
// rows of 16-byte pieces.  nsplit > 1 or f32: fp32 parts [nsplit][T][F] (with accumulate added to what is there), split s
// summing k_per (whole units) from s * k_per on; otherwise bf16 out [T][ldo], times *scale where scale is given.
// F a multiple of 8; K one too where an operand has k contiguous, that operand's k from the sum's end up to it zeros; a k
// strided tok has rows of at least T rounded up to 8.  Kf: the k that a k strided feat has (the last of K may lack).
// feat_rest, tok_rest: where not 0, the operand's second term is so many elements on (mm_terms).
struct MmArgs {
  const uint16_t *feat, *tok;
  int64_t feat_rest, tok_rest;
  int64_t ldf, ldt, F, T, K, Kf;
  void *out;
  int64_t ldo;
  int64_t nsplit, k_per;
  const float *scale;
  int f32, accumulate;
};
// A product's tile shape (an index of lm_mm.hip's) and the splits of its k.
struct MmPlan {
  int shape;
  int64_t splits;
  int64_t part_bytes(int64_t T, int64_t F) const { return splits > 1 ? splits * T * F * 4 : 0; }
};
MmPlan mm_plan(int64_t T, int64_t F, int64_t K, bool may_split);
// One launch of it: the parts (a.f32) or, with one split, the result.  a.nsplit and a.k_per are set from the plan.
// Refuses feat_kc without tok_kc, which no operator needs.
int mm_launch(MmArgs a, bool feat_kc, bool tok_kc, const MmPlan &plan, hipStream_t stream, const char *what);
// The product into bf16 a.out [T][a.ldo]: parts (part_bytes of the plan) and their sum where k is split.
int mm_run(MmArgs a, bool feat_kc, bool tok_kc, const MmPlan &plan, float *parts, hipStream_t stream, const char *what);
// out bf16 [T][ldo] = scale * sum of `parts` fp32 [nsplit][T][F] in order
int mm_reduce_launch(const float *parts, int64_t nsplit, int64_t T, int64_t F, const float *scale, void *out, int64_t ldo,
                     hipStream_t stream, const char *what);

}  // namespace smlm
