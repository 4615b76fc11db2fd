// The K loop of the training step's products on the matrix cores (v_mfma_f32_16x16x32_bf16, fp32 sums): a tile of
// TT rows ("tokens") x FT columns ("features") from two bf16 operands, each of which may have the summed dimension k
// contiguous (rows of k: a linear layer's input and weight) or strided (rows of tokens or features, k the slow dimension:
// the operands of a weight's gradient).
//
// Workgroup = 4 wavefronts, WF x WT of them over the tile, 16 NI features x 16 NJ tokens each.  At the matrix cores' rate a
// wavefront's tile of 64 features x 128 tokens reads 96 of the 128 bytes per clock that the LDS has, one of 64 x 64 all
// of them: hence 128 x 256 tiles where there are enough of them.
// k streams through three LDS stages of 32, loaded straight from memory into LDS (buffer_load ... lds, no registers in
// between).  While a chunk is multiplied, the next one's fragments are read into a second set of registers and the chunk
// three ahead is loaded into the stage that the first came from (which all wavefronts have read by the barrier that opens
// the step), the reads and loads spread between the products: neither LDS nor memory latency stands between two chunks'
// products.  The number of chunks is even, so that the two register sets alternate without copies.  A stage takes 24 KB for
// 128 x 256, so that two workgroups fit a CU: one's epilogue runs under the other's products.
//
// LDS layouts (16-byte pieces; banks repeat every 256 bytes):
//   k contiguous: 64-byte rows, piece c of row R at c ^ swz(R), so that the 16 rows of a fragment read fall on distinct
//     banks; read with ds_read_b128.  Feature rows are read permuted (lane r of tile i takes row 4 NI (r / 4) + 4 i +
//     r % 4), which leaves each lane 4 NI consecutive features of a token in its accumulators: 32-byte stores.
//   k strided: rows of 32 k, piece c of row k at c ^ v(k), read with ds_read_b64_tr_b16, which gives lane r four k of
//     column r.  Lane group g takes k = 8 g .. 8 g + 7 in both layouts.
// Out of range rows and k read as zeros (the buffer's record count; the k beyond the end of contiguous rows by an offset
// out of range), so tails need no other care than not storing what lies outside.
#pragma once

#include "pkm_common.h"

namespace smlm {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef int intx4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) unsigned char lds_byte;

constexpr int kMmThreads = 256, kMmK = 32, kMmStages = 3, kMmXcds = 8;

// 16 bytes per lane from a buffer straight into LDS at lds + 16 * lane (wave-uniform lds).  Inline assembly, so that the
// compiler adds no wait for it before every LDS read; the kernels wait themselves (mm_wait).
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void mm_load_lds(intx4 rsrc, uint32_t voff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(voff), "s"(rsrc), "s"(lds)
               : "m0");
}
#pragma clang diagnostic pop

// At most N vector memory operations on their way and every LDS read done; then the barrier.  Loads complete in order:
// with N = the loads issued after a chunk's, that chunk has landed.
template <int N>
__device__ __forceinline__ void mm_wait_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | ((N >> 4) << 14));
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

constexpr uint32_t kMmOutside = 0xFFFFFFF0u;  // an offset that no record count reaches

// One operand's LDS tile of ROWS rows (tokens or features) x 32 k.  PERM: features per lane group (4 NI) of a permuted
// fragment, 0 for a plain one.
template <int ROWS, bool KC, int PERM>
struct MmTile {
  static constexpr bool kContiguous = KC;
  static constexpr int kRows = ROWS, kBytes = ROWS * kMmK * 2;
  static constexpr int kLoads = kBytes / 4096;                       // per thread and chunk
  static constexpr int kRowBytes = KC ? kMmK * 2 : ROWS * 2;
  static constexpr int kRowsPerLoad = 4096 / kRowBytes;              // LDS rows that one load of the workgroup fills
  static_assert(kBytes % 4096 == 0, "a whole number of loads");

  static __device__ __forceinline__ int swz(int row) {               // KC
    return -(PERM ? row / PERM : row / 4) & 3;
  }
  static __device__ __forceinline__ int vsw(int k) {                 // k strided
    return ROWS >= 128 ? 2 * ((k & 3) | ((k >> 3 & 1) << 2)) : 2 * ((k >> 1 & 1) | ((k >> 3 & 1) << 1));
  }

  // This thread's byte offset of load u from the chunk's first byte.
  static __device__ __forceinline__ uint32_t offset(int u, int tid, int64_t ld) {
    if constexpr (KC) {
      return (uint32_t)((u * kRowsPerLoad + tid / 4) * ld * 2 + first_k(tid) * 2);
    } else {
      const int per = kRowBytes / 16, k = u * kRowsPerLoad + tid / per;
      return (uint32_t)(k * ld * 2 + (((tid % per) ^ vsw(k)) * 16));
    }
  }
  static __device__ __forceinline__ int first_k(int tid) { return 8 * ((tid % 4) ^ swz(tid / 4)); }   // KC
  // LDS address (from the tile's base) that lane (r, g) reads the wavefront's row group i from, its rows starting at w0.
  static __device__ __forceinline__ uint32_t frag_at(int w0, int i, int r, int g) {
    if constexpr (KC) {                       // w0 a multiple of 4 * PERM or 16: the swizzle is that of i = 0
      const int R = PERM ? w0 + PERM * (r / 4) + r % 4 : w0 + r;
      return R * kRowBytes + ((g ^ swz(R)) * 16) + i * (PERM ? 4 : 16) * kRowBytes;
    } else {
      const int k = 8 * g + r / 4;
      const int col = PERM ? w0 + PERM * (r % 4) + 4 * i : w0 + 16 * i + 4 * (r % 4);
      return k * kRowBytes + (((col / 8) ^ vsw(k)) * 16) + (col % 8) * 2;
    }
  }
  static __device__ __forceinline__ bf16x8 frag(uint32_t at) {
    if constexpr (KC) {
      return *(const __attribute__((address_space(3))) bf16x8 *)(uintptr_t)at;
    } else {
      typedef __attribute__((address_space(3))) bf16x4 *p4;
      const bf16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((p4)(uintptr_t)at);
      const bf16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((p4)(uintptr_t)(at + 4 * kRowBytes));
      return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
};

// Where an operand's next chunk comes from: wave-uniform, stepped from chunk to chunk.  `left` is exact: the bytes from the
// chunk's first to the operand's last, which the record count of its loads is clipped to: past the end they read zeros.
template <class O>
struct MmSource {
  const uint16_t *p;
  int64_t left, step, k;                                 // step in bytes; k: what is left of the sum
  // rows from row0 (< rows) on and k from k0 (< K) on of an operand of `rows` rows and K
  __device__ __forceinline__ void init(const uint16_t *base, int64_t ld, int64_t rows, int64_t K, int64_t row0, int64_t k0) {
    const int64_t major = O::kContiguous ? row0 : k0, minor = O::kContiguous ? k0 : row0;
    p = base + major * ld + minor;
    left = (((O::kContiguous ? rows : K) - 1 - major) * ld + (O::kContiguous ? K : rows) - minor) * 2;
    step = O::kContiguous ? kMmK * 2 : kMmK * 2 * ld;
    k = K - k0;
  }
  __device__ __forceinline__ intx4 rsrc() const {
    const uint64_t a = (uint64_t)p;
    const uint32_t n = left >> 32 ? 0xFFFFFFF0u : (uint32_t)left;
    return intx4{(int)(uint32_t)a, (int)(uint32_t)(a >> 32), (int)(left <= 0 ? 0u : n), 0x00020000};
  }
  __device__ __forceinline__ void next() {
    p += step / 2;
    left -= step;
    k -= kMmK;
  }
};

template <int NI, int NJ>
struct MmFrags {
  bf16x8 a[NI], b[NJ];
};

// The loop's state of one thread for an F tile of features and a T tile of tokens: a stage holds F, then T.
template <class F, class T, int NI, int NJ>
struct MmLoop {
  static constexpr int kStage = F::kBytes + T::kBytes, kLoads = F::kLoads + T::kLoads;
  typedef MmFrags<NI, NJ> Frags;
  uint32_t fo[F::kLoads], to[T::kLoads], fa[NI], ta[NJ], lds;

  __device__ __forceinline__ void offsets(int64_t ldf, int64_t ldt) {
#pragma unroll
    for (int u = 0; u < F::kLoads; ++u) fo[u] = F::offset(u, threadIdx.x, ldf);
#pragma unroll
    for (int u = 0; u < T::kLoads; ++u) to[u] = T::offset(u, threadIdx.x, ldt);
  }
  // wf, wt: first feature and token row of this wavefront in the tile
  __device__ __forceinline__ void init(const unsigned char *smem, int64_t ldf, int64_t ldt, int wf, int wt) {
    const int lane = threadIdx.x % kWave, r = lane & 15, g = lane >> 4;
    const uint32_t base = (uint32_t)(uintptr_t)(lds_byte *)smem;
    offsets(ldf, ldt);
#pragma unroll
    for (int i = 0; i < NI; ++i) fa[i] = base + F::frag_at(wf, i, r, g);
#pragma unroll
    for (int j = 0; j < NJ; ++j) ta[j] = base + F::kBytes + T::frag_at(wt, j, r, g);
    lds = base + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave) * 1024;
  }

  // The last chunks of contiguous rows: the pieces from the sum's end on come from outside, as zeros, from now on.
  template <class O>
  static __device__ __forceinline__ void clip(const MmSource<O> &s, uint32_t *off) {
    if (O::kContiguous && s.k < kMmK) {                  // wave-uniform
      const bool inside = O::first_k(threadIdx.x) < s.k;
#pragma unroll
      for (int u = 0; u < O::kLoads; ++u) off[u] = inside ? off[u] : kMmOutside;
    }
  }
  // Load l of the sources' next chunk (F's first) into `stage`.
  __device__ __forceinline__ void load(int l, intx4 frsrc, intx4 trsrc, uint32_t stage) const {
    mm_load_lds(l < F::kLoads ? frsrc : trsrc, l < F::kLoads ? fo[l] : to[l - F::kLoads], lds + stage + l * 4096);
  }
  __device__ __forceinline__ void issue(MmSource<F> &f, MmSource<T> &t, uint32_t stage) {
    clip(f, fo);
    clip(t, to);
    const intx4 fr = f.rsrc(), tr = t.rsrc();
#pragma unroll
    for (int l = 0; l < kLoads; ++l) load(l, fr, tr, stage);
    f.next();
    t.next();
  }
  __device__ __forceinline__ void read(Frags &x, uint32_t stage) const {
#pragma unroll
    for (int i = 0; i < NI; ++i) x.a[i] = F::frag(fa[i] + stage);
#pragma unroll
    for (int j = 0; j < NJ; ++j) x.b[j] = T::frag(ta[j] + stage);
  }
  // The products of `cur`, with load(i) and read(i), i < NI, spread between them.
  template <class LOAD, class READ>
  static __device__ __forceinline__ void products(const Frags &cur, floatx4 (&acc)[NI][NJ], LOAD load, READ read) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      load(i);
      read(i);
#pragma unroll
      for (int j = 0; j < NJ; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(cur.a[i], cur.b[j], acc[i][j], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  __device__ __forceinline__ void read_part(Frags &x, uint32_t stage, int i) const {
    x.a[i] = F::frag(fa[i] + stage);
#pragma unroll
    for (int j = 0; j < NJ; ++j)
      if (j >= i * NJ / NI && j < (i + 1) * NJ / NI) x.b[j] = T::frag(ta[j] + stage);
  }
  // One step: the products of `cur` (chunk ch, whose stage is `stage`), while `next` is read from chunk ch + 1's stage and
  // the sources' chunk ch + 3 is loaded into chunk ch's.  On the way at its start: the loads of chunks ch + 1 and ch + 2.
  __device__ __forceinline__ void step(MmSource<F> &f, MmSource<T> &t, const Frags &cur, Frags &next, uint32_t &stage,
                                       floatx4 (&acc)[NI][NJ]) {
    mm_wait_barrier<kLoads>();
    const uint32_t here = stage;
    stage = stage == 2 * kStage ? 0 : stage + kStage;
    clip(f, fo);
    clip(t, to);
    const intx4 fr = f.rsrc(), tr = t.rsrc();
    products(
        cur, acc,
        [&](int i) {
#pragma unroll
          for (int l = 0; l < kLoads; ++l)
            if (l >= i * kLoads / NI && l < (i + 1) * kLoads / NI) load(l, fr, tr, here);
        },
        [&](int i) { read_part(next, stage, i); });
    f.next();
    t.next();
  }
  // Fills the three stages and reads the first chunk's fragments.
  __device__ __forceinline__ void start(MmSource<F> &f, MmSource<T> &t, Frags &x) {
    issue(f, t, 0);
    issue(f, t, kStage);
    issue(f, t, 2 * kStage);
    mm_wait_barrier<2 * kLoads>();
    read(x, 0);
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

// Chunks of a sum over k, an even number.
__device__ __forceinline__ int mm_chunks(int64_t k) { return (int)((k + 2 * kMmK - 1) / (2 * kMmK)) * 2; }

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// ---- plain products (lm_mm.hip) ----------------------------------------------------------------------------------------
// out[t, f] = sum_k tok[t, k] feat[f, k]; an operand with *_kc = false is stored [k][row].  Rows and strides in elements,
// rows of 16-byte pieces.  nsplit > 1 or f32: fp32 parts [nsplit][T][F] (with accumulate added to what is there), split s
// summing k_per (a multiple of 64) from s * k_per on; otherwise bf16 out [T][ldo], times *scale where scale is given.
// F a multiple of 8; K one too where an operand has k contiguous, that operand's k from the sum's end up to it zeros; a k
// strided tok has rows of at least T rounded up to 8.  Kf: the k that a k strided feat has (the last of K may lack).
struct MmArgs {
  const uint16_t *feat, *tok;
  int64_t ldf, ldt, F, T, K, Kf;
  void *out;
  int64_t ldo;
  int64_t nsplit, k_per;
  const float *scale;
  int f32, accumulate;
};
int mm_launch(const MmArgs &a, bool feat_kc, bool tok_kc, hipStream_t stream, const char *what);
// Splits of k for T x F outputs over K: as many as fill the card, each of at least min_k.
int64_t mm_splits(int64_t T, int64_t F, int64_t K, int64_t min_k);
int64_t mm_k_per(int64_t K, int64_t nsplit);
// out bf16 [T][ldo] = scale * sum of `parts` fp32 [nsplit][T][F] in order
int mm_reduce_launch(const float *parts, int64_t nsplit, int64_t T, int64_t F, const float *scale, void *out, int64_t ldo,
                     hipStream_t stream, const char *what);

}  // namespace smlm
