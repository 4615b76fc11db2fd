// Keys and values of one attention layer in pages: appended with the position rotation on the way, and read back.
//
// Append, per token n and head: q and k heads rotated by the token's position, one pair (a, b) of the first `rot` dims at a time,
//   a' = a cos - b sin,  b' = b cos + a sin      (half layout: b = dim i + rot / 2; interleaved: dims 2 i, 2 i + 1)
// in fp32, every operation rounded (no fused multiply-adds, so that the same operations elsewhere give the same bits), q
// rounded to bf16 into its own rows, k and v into row slots[n] % page of page slots[n] / page.  bf16 pages hold the rows as they
// are; 4-bit pages hold, per row, lo = bf16(min), step = bf16((max - lo) / 15) and the codes clamp(rint((x - lo) / step), 0, 15).
// What they stand for is within half a step of x and, towards the row's ends, what the roundings of lo and step leave out: 2^-8 of
// the lowest value (of keys; values are bf16 before) and 2^-8 of the row's range.  So a row of keys whose range is small against
// them loses more: 100.3 .. 100.9 begins at 100.5.  A row that is not finite throughout, or whose range is not, reads back as NaN.
//
// Bound by memory (every value read and written once).  One lane takes 8 dims of one row, 16 bytes of bf16: consecutive lanes
// read consecutive 16-byte pieces of the projection's row.  In the half layout a lane also loads its partner's piece, which the
// partner loads too (the second read hits the L1); so no lane exchange is needed, and a row's minimum and maximum are a
// reduction over HD / 8 lanes.  Measured, 6 heads of 64: 16 tokens 3 us (6 the whole call), 11,540 tokens 12 (4.6 TB/s).  32 and
// 2 x 8 heads of 128 into 4 bits, 2,036 tokens: 12 us (query heads leave before the rounding to codes, whose quotients come
// from a reciprocal: 15.6 without either); reading 17,134 tokens of them back as bf16 (gather) 17.7, 5.0 TB/s.
#include "lm_paged.h"

namespace smlm {
namespace {

__device__ __forceinline__ void unpack8(const uint4 v, float *f) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    f[2 * e] = __uint_as_float(u[e] << 16);
    f[2 * e + 1] = __uint_as_float(u[e] & 0xFFFF0000u);
  }
}

__device__ __forceinline__ uint4 pack8(const float *f) {
  return uint4{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7])};
}

// W values of a rotation table
template <bool F32, int W>
__device__ __forceinline__ void load_table(const void *t, int64_t i, float *f) {
  if constexpr (F32) {
#pragma unroll
    for (int e = 0; e < W; e += 4) {
      const float4 v = *(const float4 *)((const float *)t + i + e);
      f[e] = v.x, f[e + 1] = v.y, f[e + 2] = v.z, f[e + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int e = 0; e < W; e += 4) {
      const uint2 v = *(const uint2 *)((const uint16_t *)t + i + e);
      f[e] = __uint_as_float(v.x << 16), f[e + 1] = __uint_as_float(v.x & 0xFFFF0000u);
      f[e + 2] = __uint_as_float(v.y << 16), f[e + 3] = __uint_as_float(v.y & 0xFFFF0000u);
    }
  }
}

// min (or max) over the aligned groups of L lanes, on every lane
template <int L, bool MAX>
__device__ __forceinline__ float group_extreme(float v) {
  auto step = [&](float o) { v = MAX ? fmaxf(v, o) : fminf(v, o); };
  step(__uint_as_float(xor_lane<1>(__float_as_uint(v))));
  step(__uint_as_float(xor_lane<2>(__float_as_uint(v))));
  if constexpr (L >= 8) step(__uint_as_float(xor_lane<4>(__float_as_uint(v))));
  if constexpr (L >= 16) step(__uint_as_float(xor_lane<8>(__float_as_uint(v))));
  return v;
}

struct AppendArgs {
  const uint16_t *qkv;
  int64_t qkv_stride;
  const void *cos, *sin;
  int64_t rope_len;
  int rot, interleaved, H, heads;          // heads: of a projection's row, H + 2 kv_heads
  const int64_t *positions, *slots;
  uint16_t *q_out, *k_out;
  uint32_t rows;                           // N * heads
};

// this lane's 8 dims 8 c .. 8 c + 7 of a head, rotated
template <bool F32>
__device__ __forceinline__ void rotate8(const AppendArgs &A, const uint16_t *head, int c, int64_t pos, float *x) {
#pragma clang fp contract(off)
  const int d = 8 * c, half = A.rot / 2;
  float cs[8], sn[8];
  if (A.interleaved) {
    load_table<F32, 4>(A.cos, pos * half + d / 2, cs);
    load_table<F32, 4>(A.sin, pos * half + d / 2, sn);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = x[2 * i], b = x[2 * i + 1];
      x[2 * i] = a * cs[i] - b * sn[i];
      x[2 * i + 1] = b * cs[i] + a * sn[i];
    }
    return;
  }
  const bool second = d >= half;
  const int at = second ? d - half : d;
  float o[8];
  unpack8(*(const uint4 *)(head + (second ? at : d + half)), o);
  load_table<F32, 8>(A.cos, pos * half + at, cs);
  load_table<F32, 8>(A.sin, pos * half + at, sn);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float t = o[i] * sn[i];
    x[i] = x[i] * cs[i] + (second ? t : -t);   // a cos - b sin, b cos + a sin: the sign is exact
  }
}

template <int HD, bool F32, bool Q4>
__global__ void __launch_bounds__(256) append_kernel(AppendArgs A, KVPages P) {
  constexpr int L = HD / 8;
  const uint32_t item = blockIdx.x * 256 + threadIdx.x, c = item % L;
  const bool in = item / L < A.rows;
  const uint32_t row = in ? item / L : A.rows - 1;
  const uint32_t n = row / A.heads, h = row - n * A.heads;
  const uint16_t *head = A.qkv + (int64_t)n * A.qkv_stride + h * HD;
  const int64_t pos = A.positions[n], slot = A.slots[n];
  const uint4 raw = *(const uint4 *)(head + 8 * c);
  const bool is_q = h < (uint32_t)A.H, is_v = h >= (uint32_t)(A.H + P.kv_heads);
  const bool known = pos >= 0 && pos < A.rope_len;
  float x[8];
  unpack8(raw, x);
  if (!is_v && 8 * (int)c < A.rot) {
    if (known) {
      rotate8<F32>(A, head, (int)c, pos, x);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = __builtin_nanf("");
    }
  }
  const uint4 packed = is_v ? raw : pack8(x);
  if (in && is_q) *(uint4 *)(A.q_out + ((int64_t)n * A.H + h) * HD + 8 * c) = packed;
  const uint32_t kh = is_v ? h - A.H - P.kv_heads : h - A.H;
  if (in && !is_q && !is_v && A.k_out) *(uint4 *)(A.k_out + ((int64_t)n * P.kv_heads + kh) * HD + 8 * c) = packed;
  const bool store = in && !is_q && known && slot >= 0 && slot < P.num_pages << P.page_shift;
  const int64_t at = store ? P.row(slot, kh) : 0;
  if constexpr (!Q4) {
    if (store) *(uint4 *)((uint16_t *)(is_v ? P.v : P.k) + at * HD + 8 * c) = packed;
  } else {
#pragma clang fp contract(off)
    if (is_q) return;   // whole heads: the lanes of a row stay together
    float lo = x[0], hi = x[0];
    bool finite = true;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      lo = fminf(lo, x[i]);
      hi = fmaxf(hi, x[i]);
      finite = finite && fabsf(x[i]) < __builtin_inff();
    }
    lo = group_extreme<L, false>(finite ? lo : -__builtin_inff());    // one value that is not makes the whole row's lo and step so
    hi = group_extreme<L, true>(finite ? hi : __builtin_inff());
    lo = round_bf16_hw(lo);
    const float step = round_bf16_hw((hi - lo) * (1.0f / 15.0f));
    // A reciprocal gives a quotient of up to 16 within 2^-18: it rounds to another code than the quotient
    // itself only within 2^-16 of halfway, and there the division is done.
    uint32_t codes = 0;
    if (step > 0.f) {
      const float inv = 1.0f / step;
      float away = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float t = (x[i] - lo) * inv, near = rintf(t);
        away = fmaxf(away, fabsf(t - near));
        codes |= (uint32_t)fminf(fmaxf(near, 0.f), 15.f) << (4 * i);
      }
      if (!(away < 0.5f - 0x1p-16f && inv > 0x1p-125f && inv < 0x1p125f)) {
        codes = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          codes |= (uint32_t)fminf(fmaxf(rintf((x[i] - lo) / step), 0.f), 15.f) << (4 * i);
      }
    }
    if (store) {
      ((uint32_t *)(is_v ? P.v : P.k))[at * L + c] = codes;
      if (c == 0) ((uint32_t *)(is_v ? P.v_scale : P.k_scale))[at] = pack_bf16x2(step, lo);
    }
  }
}

template <int HD, bool Q4>
__global__ void __launch_bounds__(256) gather_kernel(KVPages P, const int64_t *slots, uint32_t rows, uint16_t *k_out,
                                                     uint16_t *v_out) {
  constexpr int L = HD / 8;
  const uint32_t item = blockIdx.x * 256 + threadIdx.x, c = item % L, row = item / L;
  if (row >= rows) return;
  const uint32_t n = row / P.kv_heads, h = row - n * P.kv_heads;
  const int64_t slot = slots[n];
  uint4 k{0, 0, 0, 0}, v{0, 0, 0, 0};
  if (slot >= 0 && slot < P.num_pages << P.page_shift) {
    const int64_t at = P.row(slot, h);
    if constexpr (!Q4) {
      k = *(const uint4 *)((const uint16_t *)P.k + at * HD + 8 * c);
      v = *(const uint4 *)((const uint16_t *)P.v + at * HD + 8 * c);
    } else {
      const uint32_t code[2] = {((const uint32_t *)P.k)[at * L + c], ((const uint32_t *)P.v)[at * L + c]};
      const uint32_t scale[2] = {((const uint32_t *)P.k_scale)[at], ((const uint32_t *)P.v_scale)[at]};
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const float step = __uint_as_float(scale[w] << 16), lo = __uint_as_float(scale[w] & 0xFFFF0000u);
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = lo + step * (float)(code[w] >> (4 * i) & 15);   // the product is exact
        (w ? v : k) = pack8(x);
      }
    }
  }
  *(uint4 *)(k_out + (int64_t)row * HD + 8 * c) = k;
  *(uint4 *)(v_out + (int64_t)row * HD + 8 * c) = v;
}

__global__ void __launch_bounds__(256) step_kernel(const int *table, int64_t row_stride, int64_t M, const int *lengths, int64_t B,
                                                   int shift, int64_t max_len, int64_t *positions, int64_t *slots, int *next) {
  const int64_t b = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (b >= B) return;
  const int n = lengths[b], at = n >> shift;
  const int page = n >= 0 && n < max_len && at < M ? table[b * row_stride + at] : -1;
  positions[b] = n;
  slots[b] = page < 0 ? -1 : ((int64_t)page << shift) + (n & ((1 << shift) - 1));
  next[b] = n < 0x7FFFFFFF ? n + 1 : n;
}

}  // namespace

int kv_pages(const char *name, const smlm_kv_pages *p, KVPages *out) {
  if (!p || !p->k || !p->v) return fail(SMLM_EINVAL, "%s: null pointer argument", name);
  if (p->kind != SMLM_BF16 && p->kind != SMLM_Q4)
    return fail(SMLM_EINVAL, "%s: pages must be SMLM_BF16 or SMLM_Q4, got %d", name, p->kind);
  if (p->kind == SMLM_Q4 && (!p->k_scale || !p->v_scale))
    return fail(SMLM_EINVAL, "%s: 4-bit pages need their scales", name);
  if (p->head_dim != 32 && p->head_dim != 64 && p->head_dim != 128)
    return fail(SMLM_EUNSUPPORTED, "%s: head_dim %d not in {32, 64, 128}", name, p->head_dim);
  if (!is_pow2(p->page_size) || p->page_size < 16 || p->page_size > 4096)
    return fail(SMLM_EUNSUPPORTED, "%s: page size %d is not a power of two from 16 to 4096", name, p->page_size);
  if (p->num_pages < 1 || p->num_pages > 0x7FFFFFFF || p->kv_heads < 1 || p->kv_heads > 4096)
    return fail(SMLM_EINVAL, "%s: bad shape: %lld pages, %d kv heads", name, (long long)p->num_pages, p->kv_heads);
  if (((uintptr_t)p->k | (uintptr_t)p->v | (uintptr_t)p->k_scale | (uintptr_t)p->v_scale) % 16)
    return fail(SMLM_EINVAL, "%s: the pages and their scales must be 16-byte aligned", name);
  int shift = 0;
  while (1 << shift < p->page_size) ++shift;
  *out = KVPages{p->k, p->v, p->k_scale, p->v_scale, p->num_pages, shift, p->kv_heads};
  return SMLM_OK;
}

}  // namespace smlm

extern "C" int smlm_paged_append(const void *qkv, int64_t qkv_row_stride, const void *rope_cos, const void *rope_sin,
                                 int rope_dtype, int64_t rope_len, int rot, int interleaved, const int64_t *positions,
                                 const int64_t *slots, const smlm_kv_pages *pages, int64_t N, int H, void *q_out, void *k_out,
                                 void *stream) {
  using namespace smlm;
  const char *name = "smlm_paged_append";
  KVPages P;
  if (const int rc = kv_pages(name, pages, &P)) return rc;
  if (!qkv || !rope_cos || !rope_sin || !positions || !slots || !q_out)
    return fail(SMLM_EINVAL, "%s: null pointer argument", name);
  if (rope_dtype != SMLM_F32 && rope_dtype != SMLM_BF16)
    return fail(SMLM_EINVAL, "%s: rope tables must be SMLM_F32 or SMLM_BF16", name);
  const int hd = pages->head_dim;
  if (N < 0 || H < 1 || H > 65536 || rope_len < 0)
    return fail(SMLM_EINVAL, "%s: bad shape N=%lld H=%d rope_len=%lld", name, (long long)N, H, (long long)rope_len);
  if (rot < 16 || rot > hd || rot % 16)
    return fail(SMLM_EUNSUPPORTED, "%s: %d rotated dims are not a multiple of 16 from 16 to head_dim", name, rot);
  const int heads = H + 2 * pages->kv_heads;
  if (qkv_row_stride < (int64_t)heads * hd || qkv_row_stride % 8)
    return fail(SMLM_EINVAL, "%s: qkv_row_stride %lld must be >= (H + 2 kv_heads) * head_dim and a multiple of 8", name,
                (long long)qkv_row_stride);
  if (((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)k_out | (uintptr_t)rope_cos | (uintptr_t)rope_sin) % 16 ||
      ((uintptr_t)positions | (uintptr_t)slots) % 8)
    return fail(SMLM_EINVAL, "%s: qkv, the outputs and the rope tables must be 16-byte aligned", name);
  if (N > 0x7FFFFFFFLL / (heads * (hd / 8)))
    return fail(SMLM_EUNSUPPORTED, "%s: N=%lld tokens are more than 2^31 pieces of 8 dims", name, (long long)N);
  if (N == 0) return SMLM_OK;
  const AppendArgs A{(const uint16_t *)qkv, qkv_row_stride, rope_cos, rope_sin, rope_len, rot, interleaved != 0, H, heads,
                     positions, slots, (uint16_t *)q_out, (uint16_t *)k_out, (uint32_t)(N * heads)};
  const unsigned grid = (unsigned)((N * heads * (hd / 8) + 255) / 256);
  const bool f32 = rope_dtype == SMLM_F32, q4 = pages->kind == SMLM_Q4;
#define SMLM_APPEND(HD)                                                                                             \
  if (f32 && q4) hipLaunchKernelGGL((append_kernel<HD, true, true>), dim3(grid), dim3(256), 0, (hipStream_t)stream, A, P);    \
  else if (f32) hipLaunchKernelGGL((append_kernel<HD, true, false>), dim3(grid), dim3(256), 0, (hipStream_t)stream, A, P);    \
  else if (q4) hipLaunchKernelGGL((append_kernel<HD, false, true>), dim3(grid), dim3(256), 0, (hipStream_t)stream, A, P);     \
  else hipLaunchKernelGGL((append_kernel<HD, false, false>), dim3(grid), dim3(256), 0, (hipStream_t)stream, A, P)
  if (hd == 32) { SMLM_APPEND(32); }
  else if (hd == 64) { SMLM_APPEND(64); }
  else { SMLM_APPEND(128); }
#undef SMLM_APPEND
  return launch_status(name);
}

extern "C" int smlm_paged_step(const int *block_table, int64_t row_stride, int64_t M, const int *lengths, int64_t B, int page_size,
                               int64_t max_len, int64_t *positions, int64_t *slots, int *next, void *stream) {
  using namespace smlm;
  const char *name = "smlm_paged_step";
  if (!block_table || !lengths || !positions || !slots || !next) return fail(SMLM_EINVAL, "%s: null pointer argument", name);
  if (!is_pow2(page_size) || page_size < 16 || page_size > 4096)
    return fail(SMLM_EUNSUPPORTED, "%s: page size %d is not a power of two from 16 to 4096", name, page_size);
  if (B < 0 || B > 0x7FFFFFFF || M < 1 || row_stride < M || max_len < 0)
    return fail(SMLM_EINVAL, "%s: bad shape B=%lld M=%lld row_stride=%lld max_len=%lld", name, (long long)B, (long long)M,
                (long long)row_stride, (long long)max_len);
  if (((uintptr_t)block_table | (uintptr_t)lengths | (uintptr_t)next) % 4 || ((uintptr_t)positions | (uintptr_t)slots) % 8)
    return fail(SMLM_EINVAL, "%s: misaligned pointer", name);
  if (B == 0) return SMLM_OK;
  int shift = 0;
  while (1 << shift < page_size) ++shift;
  hipLaunchKernelGGL(step_kernel, dim3((unsigned)((B + 255) / 256)), dim3(256), 0, (hipStream_t)stream, block_table, row_stride, M,
                     lengths, B, shift, max_len, positions, slots, next);
  return launch_status(name);
}

extern "C" int smlm_paged_gather(const smlm_kv_pages *pages, const int64_t *slots, int64_t N, void *k_out, void *v_out,
                                 void *stream) {
  using namespace smlm;
  const char *name = "smlm_paged_gather";
  KVPages P;
  if (const int rc = kv_pages(name, pages, &P)) return rc;
  if (!slots || !k_out || !v_out) return fail(SMLM_EINVAL, "%s: null pointer argument", name);
  if (((uintptr_t)k_out | (uintptr_t)v_out) % 16 || (uintptr_t)slots % 8)
    return fail(SMLM_EINVAL, "%s: the outputs must be 16-byte aligned", name);
  const int hd = pages->head_dim;
  if (N < 0) return fail(SMLM_EINVAL, "%s: bad shape N=%lld", name, (long long)N);
  if (N > 0x7FFFFFFFLL / (pages->kv_heads * (hd / 8)))
    return fail(SMLM_EUNSUPPORTED, "%s: N=%lld tokens are more than 2^31 pieces of 8 dims", name, (long long)N);
  if (N == 0) return SMLM_OK;
  const uint32_t rows = (uint32_t)(N * pages->kv_heads);
  const unsigned grid = (unsigned)(((int64_t)rows * (hd / 8) + 255) / 256);
  const bool q4 = pages->kind == SMLM_Q4;
#define SMLM_GATHER(HD)                                                                                               \
  if (q4) hipLaunchKernelGGL((gather_kernel<HD, true>), dim3(grid), dim3(256), 0, (hipStream_t)stream, P, slots, rows,  \
                             (uint16_t *)k_out, (uint16_t *)v_out);                                                     \
  else hipLaunchKernelGGL((gather_kernel<HD, false>), dim3(grid), dim3(256), 0, (hipStream_t)stream, P, slots, rows,    \
                          (uint16_t *)k_out, (uint16_t *)v_out)
  if (hd == 32) { SMLM_GATHER(32); }
  else if (hd == 64) { SMLM_GATHER(64); }
  else { SMLM_GATHER(128); }
#undef SMLM_GATHER
  return launch_status(name);
}
