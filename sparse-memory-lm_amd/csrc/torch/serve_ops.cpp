// The operators of serving sequences of different lengths (smlm_hip.kernels.paged_append, paged_step, paged_gather, packed_attention,
// paged_attention and sample_tokens): argument checks, outputs and workspaces from torch's allocator, and the C entry points of
// include/smlm_pkm.h on torch's current stream of the inputs' device.  Forward only.
//
// In C++ because the smallest calls, 6 to 8 us whole, take as long as their argument checks and launches.
#include <array>

#include "common.h"

namespace {

constexpr int64_t kMaxStride = 1 << 22;      // of packed rows and heads, in elements (csrc/lm_packed_attention.hip)

Tensor aligned(const Tensor &t) {      // its last dimension dense and every row 16-byte aligned; a copy where it is not so
  bool fine = t.size(-1) == 0 || (t.stride(-1) == 1 && (uintptr_t)t.data_ptr() % 16 == 0);
  for (int64_t i = 0; i + 1 < t.dim(); ++i)
    fine = fine && (t.size(i) <= 1 || (t.stride(i) % 8 == 0 && t.stride(i) <= kMaxStride));
  return fine ? t : t.clone(at::MemoryFormat::Contiguous);
}

// Whether rows or heads of t (N, H, hd) lie on top of each other in memory: the smaller stride has to hold hd elements, the larger one
// all that the smaller one spans.
bool overlaps(const Tensor &t) {
  int64_t span = t.size(2);
  for (const int i : t.size(1) <= 1 || (t.size(0) > 1 && t.stride(0) < t.stride(1)) ? std::array{0, 1} : std::array{1, 0}) {
    if (t.size(i) <= 1) continue;
    if (t.stride(i) < span) return true;
    span += t.stride(i) * (t.size(i) - 1);
  }
  return false;
}

// strides over rows and heads; a dimension of one takes none
void row_strides(const Tensor &t, int64_t *s) {
  for (int i = 0; i < 2; ++i) s[i] = t.size(i) > 1 ? t.stride(i) : 0;
}

bool is_bf16(const Tensor &t) { return t.scalar_type() == at::kBFloat16; }

// There is no backward: inputs that autograd records would lose their gradients without a word.
void forward_only(const char *name, std::initializer_list<const Tensor *> inputs) {
  if (!at::GradMode::is_enabled()) return;
  for (const Tensor *t : inputs)
    TORCH_CHECK_VALUE(!t->defined() || !t->requires_grad(), name, " has no backward pass and an input requires grad: call it under "
                      "torch.no_grad() or detach the input");
}

// (k, v) of bf16 pages or (k, v, k_scale, v_scale) of 4-bit ones
smlm_kv_pages check_pages(const char *name, const Tensor &first, const std::vector<Tensor> &p) {
  TORCH_CHECK_VALUE(p.size() == 2 || p.size() == 4, name, ": pages are (k, v), or (k, v, k_scale, v_scale) in 4 bits; got ",
                    p.size(), " tensors");
  const bool q4 = p.size() == 4;
  for (const Tensor &t : p) {
    check_device(name, first, {&t});
    forward_only(name, {&t});
    TORCH_CHECK_VALUE(t.dim() == 4 && t.is_contiguous() && !t.is_neg(), name, ": pages must be contiguous and 4-dimensional, got ",
                      t.sizes());
  }
  TORCH_CHECK_VALUE(p[0].sizes() == p[1].sizes() && p[0].scalar_type() == p[1].scalar_type() &&
                        p[0].scalar_type() == (q4 ? at::kByte : at::kBFloat16),
                    name, ": k and v pages must both be (pages, kv_heads, page, head_dim) bf16, or (pages, kv_heads, page, "
                    "head_dim / 2) uint8 with scales; got ", p[0].sizes(), " ", p[0].scalar_type(), " and ", p[1].sizes(), " ",
                    p[1].scalar_type());
  const int64_t n = p[0].size(0), hk = p[0].size(1), page = p[0].size(2), hd = p[0].size(3) * (q4 ? 2 : 1);
  TORCH_CHECK_VALUE(n >= 1 && hk >= 1 && hk <= 4096 && page >= 16 && page <= 4096 && (page & (page - 1)) == 0 &&
                        (hd == 32 || hd == 64 || hd == 128),
                    name, ": pages must hold a power of two from 16 to 4096 tokens of up to 4096 heads of 32, 64 or 128 dims, got ",
                    n, " pages of ", page, " tokens, ", hk, " heads of ", hd);
  for (size_t i = 2; i < p.size(); ++i)
    TORCH_CHECK_VALUE(is_bf16(p[i]) && p[i].sizes() == at::IntArrayRef({n, hk, page, 2}), name, ": scales must be (", n, ", ", hk,
                      ", ", page, ", 2) bf16, got ", p[i].sizes(), " ", p[i].scalar_type());
  for (const Tensor &t : p) TORCH_CHECK_VALUE((uintptr_t)t.data_ptr() % 16 == 0, name, ": pages must be 16-byte aligned");
  return {p[0].data_ptr(), p[1].data_ptr(), q4 ? p[2].data_ptr() : nullptr, q4 ? p[3].data_ptr() : nullptr, n,
          q4 ? SMLM_Q4 : SMLM_BF16, (int)page, (int)hk, (int)hd};
}

Tensor check_slots(const char *name, const char *what, const Tensor &t, int64_t n) {
  TORCH_CHECK_VALUE(t.scalar_type() == at::kLong && t.dim() == 1 && (n < 0 || t.size(0) == n), name, ": ", what,
                    " must be int64, one a token, got ", t.sizes(), " ", t.scalar_type());
  return t.contiguous();
}

std::tuple<Tensor, std::optional<Tensor>> paged_append(const Tensor &qkv, const Tensor &cos, const Tensor &sin,
                                                       const Tensor &positions, const Tensor &slots,
                                                       const std::vector<Tensor> &pages, int64_t n_heads, bool interleaved,
                                                       bool keys) {
  const char *name = "paged_append";
  check_device(name, qkv, {&cos, &sin, &positions, &slots});
  forward_only(name, {&qkv, &cos, &sin});
  const c10::DeviceGuard guard(qkv.device());
  const smlm_kv_pages P = check_pages(name, qkv, pages);
  const int64_t heads = n_heads + 2 * P.kv_heads, hd = P.head_dim;
  TORCH_CHECK_VALUE(n_heads >= 1 && n_heads <= 65536 && is_bf16(qkv) && qkv.dim() >= 1 && qkv.size(-1) == heads * hd, name,
                    ": expected qkv (..., ", heads * hd, ") bf16 of ", n_heads, " query and 2 x ", P.kv_heads,
                    " key and value heads of ", hd, ", got ", qkv.sizes(), " ", qkv.scalar_type());
  const int64_t N = qkv.numel() / qkv.size(-1), half = cos.dim() == 2 ? cos.size(1) : 0;
  TORCH_CHECK_VALUE(cos.dim() == 2 && sin.sizes() == cos.sizes() && is_float_type(cos.scalar_type()) &&
                        sin.scalar_type() == cos.scalar_type() && half >= 8 && half % 8 == 0 && 2 * half <= hd,
                    name, ": rope tables must be (positions, rotated dims / 2) fp32 or bf16, the rotated dims a multiple of 16 up "
                    "to ", hd, ", got ", cos.sizes(), " ", cos.scalar_type(), " and ", sin.sizes(), " ", sin.scalar_type());
  const Tensor pos = check_slots(name, "positions", positions, N), at = check_slots(name, "slots", slots, N);
  const Tensor rows = plain(qkv).reshape({N, heads * hd});
  const Tensor x = N > 1 && rows.stride(0) < heads * hd ? rows.clone(at::MemoryFormat::Contiguous) : aligned(rows), c = aligned(plain(cos).contiguous()),
               s = aligned(plain(sin).contiguous());
  Tensor q = at::empty({N, n_heads, hd}, qkv.options());
  std::optional<Tensor> k;
  if (keys) k = at::empty({N, P.kv_heads, hd}, qkv.options());
  if (N == 0) return {q, k};
  check(smlm_paged_append(x.data_ptr(), N > 1 ? x.stride(0) : heads * hd, c.data_ptr(), s.data_ptr(), dtype_of(c.scalar_type()),
                          c.size(0), (int)(2 * half), interleaved, pos.data_ptr<int64_t>(), at.data_ptr<int64_t>(), &P, N,
                          (int)n_heads, q.data_ptr(), keys ? k->data_ptr() : nullptr, stream_of(qkv)),
        "smlm_paged_append");
  return {q, k};
}

std::tuple<Tensor, Tensor, Tensor> paged_step(const Tensor &block_table, const Tensor &lengths, int64_t page_size,
                                              int64_t max_len) {
  const char *name = "paged_step";
  check_device(name, block_table, {&lengths});
  const c10::DeviceGuard guard(block_table.device());
  TORCH_CHECK_VALUE(block_table.dim() == 2 && block_table.scalar_type() == at::kInt && lengths.dim() == 1 &&
                        lengths.scalar_type() == at::kInt && lengths.size(0) == block_table.size(0) && block_table.size(1) >= 1,
                    name, ": expected block_table (sequences, pages) and lengths (sequences,) int32, got ", block_table.sizes(), " ",
                    block_table.scalar_type(), " and ", lengths.sizes(), " ", lengths.scalar_type());
  TORCH_CHECK_VALUE(page_size >= 16 && page_size <= 4096 && (page_size & (page_size - 1)) == 0 && max_len >= 0, name,
                    ": a page holds a power of two from 16 to 4096 tokens, got ", page_size, ", and max_len ", max_len);
  const Tensor table = block_table.contiguous(), len = lengths.contiguous();
  const int64_t B = table.size(0);
  Tensor positions = at::empty({B}, len.options().dtype(at::kLong)), slots = at::empty_like(positions), next = at::empty_like(len);
  if (B)
    check(smlm_paged_step(table.data_ptr<int>(), table.size(1), table.size(1), len.data_ptr<int>(), B, (int)page_size, max_len,
                          positions.data_ptr<int64_t>(), slots.data_ptr<int64_t>(), next.data_ptr<int>(), stream_of(block_table)),
          "smlm_paged_step");
  return {positions, slots, next};
}

std::tuple<Tensor, Tensor> paged_gather(const std::vector<Tensor> &pages, const Tensor &slots) {
  const char *name = "paged_gather";
  check_device(name, slots, {});
  const c10::DeviceGuard guard(slots.device());
  const smlm_kv_pages P = check_pages(name, slots, pages);
  const Tensor at = check_slots(name, "slots", slots, -1);
  const auto bf16 = slots.options().dtype(at::kBFloat16);
  Tensor k = at::empty({at.size(0), P.kv_heads, P.head_dim}, bf16), v = at::empty({at.size(0), P.kv_heads, P.head_dim}, bf16);
  if (at.size(0) == 0) return {k, v};
  check(smlm_paged_gather(&P, at.data_ptr<int64_t>(), at.size(0), k.data_ptr(), v.data_ptr(), stream_of(slots)),
        "smlm_paged_gather");
  return {k, v};
}

float scale_of(const char *name, std::optional<double> scale, int64_t hd) {
  const double s = scale.value_or(1.0 / std::sqrt((double)hd));
  TORCH_CHECK_VALUE(s > 0 && s <= 1e38 && (float)s > 0, name, ": the scale must be positive, at most 1e38, got ", s);
  return (float)s;
}

Tensor packed_attention(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &cu_q, const std::optional<Tensor> &cu_k,
                        std::optional<double> scale, const std::optional<Tensor> &out) {
  const char *name = "packed_attention";
  const Tensor none;
  check_device(name, q, {&k, &v, &cu_q, cu_k ? &*cu_k : &none, out ? &*out : &none});
  forward_only(name, {&q, &k, &v, out ? &*out : &none});
  const c10::DeviceGuard guard(q.device());
  TORCH_CHECK_VALUE(is_bf16(q) && is_bf16(k) && is_bf16(v), name, ": q, k and v must be bf16, got ", q.scalar_type(), ", ",
                    k.scalar_type(), " and ", v.scalar_type());
  TORCH_CHECK_VALUE(q.dim() == 3 && k.dim() == 3 && v.sizes() == k.sizes() && k.size(2) == q.size(2) && k.size(1) >= 1 &&
                        q.size(1) >= 1 && q.size(1) % k.size(1) == 0,
                    name, ": expected q (N, heads, head_dim) and k, v (S, kv_heads, head_dim), the heads a multiple of the kv "
                    "heads, got ", q.sizes(), ", ", k.sizes(), " and ", v.sizes());
  const int64_t N = q.size(0), S = k.size(0), H = q.size(1), hd = q.size(2);
  TORCH_CHECK_VALUE(hd == 32 || hd == 64 || hd == 128, name, ": head_dim ", hd, " not in (32, 64, 128)");
  TORCH_CHECK_VALUE(cu_q.dim() == 1 && cu_q.size(0) >= 1 && cu_q.scalar_type() == at::kInt, name,
                    ": cu_q must be (sequences + 1,) int32, got ", cu_q.sizes(), " ", cu_q.scalar_type());
  TORCH_CHECK_VALUE(!cu_k || (cu_k->sizes() == cu_q.sizes() && cu_k->scalar_type() == at::kInt), name,
                    ": cu_k must be int32 of cu_q's size ", cu_q.sizes(), ", got ", cu_k ? cu_k->sizes() : cu_q.sizes(), " ",
                    cu_k ? cu_k->scalar_type() : at::kInt);
  TORCH_CHECK_VALUE(cu_k || S == N, name, ": ", S, " keys for ", N, " queries need cu_k");
  TORCH_CHECK_VALUE(!out || (out->sizes() == q.sizes() && is_bf16(*out) && !out->is_neg() && out->stride(2) == 1 &&
                             (N <= 1 || (out->stride(0) % 4 == 0 && out->stride(0) <= kMaxStride)) &&
                             (H <= 1 || (out->stride(1) % 4 == 0 && out->stride(1) <= kMaxStride)) && !overlaps(*out) &&
                             (uintptr_t)out->data_ptr() % 8 == 0),
                    name, ": out must be ", q.sizes(), " bf16 with a dense, 8-byte aligned last dimension, no element twice");
  const Tensor qa = aligned(plain(q)), ka = aligned(plain(k)), va = aligned(plain(v)), cq = cu_q.contiguous(),
               ck = cu_k ? cu_k->contiguous() : cq;
  Tensor y = out ? *out : at::empty({N, H, hd}, q.options());
  if (N == 0) return y;
  int64_t qs[2], ks[2], vs[2], ys[2];
  row_strides(qa, qs), row_strides(ka, ks), row_strides(va, vs), row_strides(y, ys);
  check(smlm_packed_attention(qa.data_ptr(), qs, ka.data_ptr(), ks, va.data_ptr(), vs, cq.data_ptr<int>(), ck.data_ptr<int>(),
                              cq.size(0) - 1, N, S, (int)H, (int)k.size(1), (int)hd, scale_of(name, scale, hd), y.data_ptr(), ys,
                              !out, stream_of(q)),
        "smlm_packed_attention");
  return y;
}

Tensor paged_attention(const Tensor &q, const std::vector<Tensor> &pages, const Tensor &block_table, const Tensor &lengths,
                       std::optional<double> scale) {
  const char *name = "paged_attention";
  check_device(name, q, {&block_table, &lengths});
  forward_only(name, {&q});
  const c10::DeviceGuard guard(q.device());
  const smlm_kv_pages P = check_pages(name, q, pages);
  TORCH_CHECK_VALUE(is_bf16(q) && q.dim() == 3 && q.size(2) == P.head_dim && q.size(1) >= 1 && q.size(1) % P.kv_heads == 0, name,
                    ": expected q (sequences, heads, ", P.head_dim, ") bf16, the heads a multiple of ", P.kv_heads, ", got ",
                    q.sizes(), " ", q.scalar_type());
  const int64_t B = q.size(0), H = q.size(1), hd = q.size(2);
  TORCH_CHECK_VALUE(block_table.dim() == 2 && block_table.size(0) == B && block_table.scalar_type() == at::kInt, name,
                    ": block_table must be (", B, ", pages of a sequence) int32, got ", block_table.sizes(), " ",
                    block_table.scalar_type());
  TORCH_CHECK_VALUE(lengths.dim() == 1 && lengths.size(0) == B && lengths.scalar_type() == at::kInt, name, ": lengths must be (",
                    B, ",) int32, got ", lengths.sizes(), " ", lengths.scalar_type());
  const int64_t M = block_table.size(1);
  Tensor y = at::empty({B, H, hd}, q.options());
  if (B == 0 || M == 0) return y.zero_();
  const Tensor x0 = plain(q);
  const bool dense = x0.stride(2) == 1 && (H == 1 || x0.stride(1) == hd) && (B == 1 || (x0.stride(0) % 8 == 0 && x0.stride(0) >= H * hd)) &&
                     (uintptr_t)x0.data_ptr() % 16 == 0;
  const Tensor x = dense ? x0 : x0.clone(at::MemoryFormat::Contiguous), len = lengths.contiguous();
  const bool rows = (M == 1 || block_table.stride(1) == 1) && (B == 1 || block_table.stride(0) >= M);
  const Tensor table = rows ? block_table : block_table.contiguous();
  const int64_t bytes = smlm_paged_attention_workspace(B, (int)H, P.kv_heads, (int)hd, P.page_size, M);
  const Tensor ws = bytes ? workspace(q, bytes) : Tensor();
  check(smlm_paged_attention(x.data_ptr(), B > 1 ? x.stride(0) : H * hd, &P, (const int *)table.data_ptr(),
                             B > 1 ? table.stride(0) : M, M, len.data_ptr<int>(), B, (int)H, scale_of(name, scale, hd),
                             y.data_ptr(), ptr(ws), bytes, stream_of(q)),
        "smlm_paged_attention");
  return y;
}

// one number for all rows, or a tensor of one a row
struct Setting {
  Tensor each;
  double all = 0;
  template <class T>
  const T *pointer() const { return each.defined() ? each.data_ptr<T>() : nullptr; }
};

Setting setting(const char *what, const py::object &v, const Tensor &logits, at::ScalarType type) {
  Setting s;
  if (THPVariable_Check(v.ptr())) {
    const Tensor &t = THPVariable_Unpack(v.ptr());
    check_device("sample_tokens", logits, {&t});
    TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == logits.size(0) && t.scalar_type() == type, "sample_tokens: ", what,
                      " must be a number or (", logits.size(0), ",) ", type, ", got ", t.sizes(), " ", t.scalar_type());
    s.each = plain(t).contiguous();
  } else {
    s.all = v.cast<double>();
    TORCH_CHECK_VALUE(s.all == s.all, "sample_tokens: ", what, " is not a number");
  }
  return s;
}

Tensor sample_tokens(const Tensor &logits, const Tensor &u, const py::object &temperature, const py::object &top_k,
                     const py::object &top_p, const py::object &min_p) {
  const char *name = "sample_tokens";
  check_device(name, logits, {&u});
  const c10::DeviceGuard guard(logits.device());
  TORCH_CHECK_VALUE(logits.dim() == 2 && is_float_type(logits.scalar_type()) && logits.size(1) >= 1 && logits.size(1) <= 1 << 18,
                    name, ": logits must be (rows, 1 to 2^18 tokens) fp32 or bf16, got ", logits.sizes(), " ",
                    logits.scalar_type());
  const int64_t B = logits.size(0), V = logits.size(1);
  TORCH_CHECK_VALUE(u.dim() == 1 && u.size(0) == B && u.scalar_type() == at::kFloat, name, ": u must be (", B, ",) fp32, got ",
                    u.sizes(), " ", u.scalar_type());
  const Setting T = setting("temperature", temperature, logits, at::kFloat), k = setting("top_k", top_k, logits, at::kInt),
                p = setting("top_p", top_p, logits, at::kFloat), m = setting("min_p", min_p, logits, at::kFloat);
  const Tensor x0 = plain(logits), x = (V == 1 || x0.stride(1) == 1) && (B <= 1 || x0.stride(0) >= V) ? x0 : x0.contiguous();
  const Tensor r = plain(u).contiguous();
  Tensor token = at::empty({B}, logits.options().dtype(at::kLong));
  if (B == 0) return token;
  const int64_t stride = B > 1 ? x.stride(0) : V;
  check(smlm_sample(x.data_ptr(), dtype_of(x.scalar_type()), stride, r.data_ptr<float>(), T.pointer<float>(), (float)T.all,
                    k.pointer<int>(), (int)std::min(std::max(k.all, 0.0), 1e9), p.pointer<float>(), (float)p.all,
                    m.pointer<float>(), (float)m.all, B, V, token.data_ptr<int64_t>(), stream_of(logits)),
        "smlm_sample");
  return token;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("paged_append", &paged_append);
  m.def("paged_step", &paged_step);
  m.def("paged_gather", &paged_gather);
  m.def("packed_attention", &packed_attention);
  m.def("paged_attention", &paged_attention);
  m.def("sample_tokens", &sample_tokens);
}
