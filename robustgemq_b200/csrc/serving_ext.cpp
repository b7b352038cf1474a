// Python entry points of the serving operators: argument checks, output and workspace
// tensors and the C ABI call in one step. The calls are short enough that on small inputs
// the host's part is their time (by way of Python checks and ctypes a one-token attention
// step took 17 us to issue, of which its two launches are 6).
#include <torch/extension.h>

#include <algorithm>

#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include "../../include/gemq_b200.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

// Raises what _lib.check raises for a status.
void check(int status) {
  if (status != GEMQ_OK) py::module_::import("robustgemq_b200._lib").attr("check")(status);
}

int code_of(at::ScalarType t) {
  return t == at::kHalf ? GEMQ_FP16 : t == at::kBFloat16 ? GEMQ_BF16 : t == at::kFloat ? GEMQ_FP32 : -1;
}

// The tensors' device made current (a model spread over several GPUs does not make a
// layer's GPU current), for the call's life.
struct OnDevice {
  explicit OnDevice(const at::Device& d) : guard(d), stream(at::cuda::getCurrentCUDAStream(d.index()).stream()) {}
  c10::cuda::CUDAGuard guard;
  void* stream;
};

Tensor bytes(size_t n, const at::Device& d) {
  return at::empty({static_cast<int64_t>(n)}, at::TensorOptions().dtype(at::kByte).device(d));
}

// The stride along axis i; an axis of one element may carry any, which does not count.
int64_t stride_of(const Tensor& t, int64_t i) {
  if (t.size(i) != 1) return t.stride(i);
  return i + 1 < t.dim() ? t.size(i + 1) * stride_of(t, i + 1) : 1;
}
bool same_strides(const Tensor& a, const Tensor& b) {
  for (int64_t i = 0; i < a.dim(); ++i)
    if (stride_of(a, i) != stride_of(b, i)) return false;
  return true;
}
bool on_16_bytes(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }
// A copy, also of what is contiguous as it is but starts off a 16-byte boundary.
Tensor copy_of(const Tensor& t) { return t.clone(at::MemoryFormat::Contiguous); }

struct Cache {
  Tensor k, v;
  OptTensor k_scale, v_scale;
  gemq_kv_cache_t c{};
  at::ScalarType dtype;

  Cache(Tensor k_, Tensor v_, OptTensor ks, OptTensor vs, at::ScalarType dtype_)
      : k(std::move(k_)), v(std::move(v_)), k_scale(std::move(ks)), v_scale(std::move(vs)), dtype(dtype_) {
    TORCH_CHECK_VALUE(k.is_cuda(), "k must be a CUDA tensor (no CPU path)");
    TORCH_CHECK_VALUE(k.dim() == 4 && v.sizes() == k.sizes() && same_strides(v, k) &&
                          v.scalar_type() == k.scalar_type() && v.device() == k.device(),
                      "k and v must be alike: [num_pages, num_kv_heads, page_size, head_dim] on one device");
    TORCH_CHECK_VALUE(dtype == at::kHalf || dtype == at::kBFloat16, "dtype must be float16 or bfloat16");
    TORCH_CHECK_VALUE(k.stride(3) == 1, "rows must be contiguous");
    const auto kind = k.scalar_type();
    c.bits = kind == at::kChar ? 8 : kind == at::kByte ? 4 : 16;
    c.dtype = code_of(dtype);
    if (c.bits == 16) {
      TORCH_CHECK_VALUE(kind == dtype, "a 16-bit cache holds its dtype");
      TORCH_CHECK_VALUE(!k_scale && !v_scale, "a 16-bit cache has no scales");
    } else {
      TORCH_CHECK_VALUE(k_scale && v_scale, "a quantised cache needs k_scale and v_scale");
      const Tensor &a = *k_scale, &b = *v_scale;
      bool ok = a.dim() == (c.bits == 8 ? 3 : 4) && a.sizes().slice(0, 3) == k.sizes().slice(0, 3) &&
                (c.bits == 8 || a.size(3) == 2);
      ok = ok && b.sizes() == a.sizes() && same_strides(b, a) && a.scalar_type() == at::kFloat &&
           b.scalar_type() == at::kFloat && a.device() == k.device() && b.device() == k.device();
      TORCH_CHECK_VALUE(ok, "k_scale and v_scale must be float32 [num_pages, num_kv_heads, page_size] (4 bits: [..., 2]) "
                            "with the same strides, beside k");
      TORCH_CHECK_VALUE(c.bits == 8 || a.stride(3) == 1, "a row's step and base must be neighbours");
      c.k_scale = a.data_ptr<float>();
      c.v_scale = b.data_ptr<float>();
      for (int i = 0; i < 3; ++i) c.scale_strides[i] = stride_of(a, i);
    }
    TORCH_CHECK_VALUE(k.size(0) <= INT32_MAX && k.size(1) <= INT32_MAX && k.size(2) <= INT32_MAX && k.size(3) < INT32_MAX / 2,
                      "sizes must be below 2^31");
    c.k = k.data_ptr();
    c.v = v.data_ptr();
    for (int i = 0; i < 3; ++i) c.strides[i] = stride_of(k, i) * static_cast<int64_t>(k.element_size());
    c.num_pages = static_cast<int32_t>(k.size(0));
    c.kv_heads = static_cast<int32_t>(k.size(1));
    c.page_size = static_cast<int32_t>(k.size(2));
    c.head_dim = static_cast<int32_t>(k.size(3)) * (c.bits == 4 ? 2 : 1);
  }

  Tensor slots_of(const Tensor& s) const {
    TORCH_CHECK_VALUE(s.scalar_type() == at::kLong && s.dim() == 1 && s.device() == k.device(),
                      "slots must be int64 [tokens] on the cache's device");
    return s.contiguous();
  }

  Tensor rows_of(const Tensor& t, const char* name, int64_t tokens) const {
    TORCH_CHECK_VALUE(t.scalar_type() == dtype && t.device() == k.device(), name, " must be ", dtype,
                      " on the cache's device");
    TORCH_CHECK_VALUE(t.dim() == 3 && t.size(0) == tokens && t.size(1) == c.kv_heads && t.size(2) == c.head_dim, name,
                      " must be [tokens, num_kv_heads, head_dim]");
    // rows of another layout (a transposed view, a start off 16 bytes) are copied once
    const bool fits = t.stride(2) == 1 && stride_of(t, 0) % 8 == 0 && stride_of(t, 1) % 8 == 0 && on_16_bytes(t);
    return fits ? t : copy_of(t);
  }

  void write(const Tensor& k_in, const Tensor& v_in, const Tensor& slots_in) const {
    const Tensor slots = slots_of(slots_in);
    const int64_t n = slots.size(0);
    const OnDevice on(k.device());
    const Tensor a = rows_of(k_in, "k", n), b = rows_of(v_in, "v", n);
    check(gemq_kv_cache_write(&c, a.data_ptr(), b.data_ptr(), stride_of(a, 0), stride_of(a, 1), stride_of(b, 0), stride_of(b, 1),
                              slots.data_ptr<int64_t>(), n, on.stream));
  }

  std::pair<Tensor, Tensor> read(const Tensor& slots_in) const {
    const Tensor slots = slots_of(slots_in);
    const int64_t n = slots.size(0);
    const OnDevice on(k.device());
    const auto opt = at::TensorOptions().dtype(dtype).device(k.device());
    Tensor a = at::empty({n, c.kv_heads, c.head_dim}, opt), b = at::empty({n, c.kv_heads, c.head_dim}, opt);
    check(gemq_kv_cache_read(&c, slots.data_ptr<int64_t>(), n, a.data_ptr(), b.data_ptr(), on.stream));
    return {std::move(a), std::move(b)};
  }
};

std::pair<Tensor, OptTensor> attention(Tensor q, const Cache& cache, Tensor page_table, Tensor kv_lens, OptTensor q_starts,
                                       int64_t max_q_len, int64_t max_kv_len, std::optional<double> scale, int64_t window,
                                       bool return_lse) {
  const auto dev = cache.k.device();
  TORCH_CHECK_VALUE(q.dim() == 3 && q.scalar_type() == cache.dtype && q.device() == dev && q.size(2) == cache.c.head_dim,
                    "q must be [tokens, q_heads, head_dim] of the cache's dtype and device");
  TORCH_CHECK_VALUE(page_table.dim() == 2 && page_table.scalar_type() == at::kInt && page_table.device() == dev,
                    "page_table must be int32 [seqs, pages] on the cache's device");
  const int64_t seqs = page_table.size(0), pages = page_table.size(1), tokens = q.size(0), heads = q.size(1);
  TORCH_CHECK_VALUE(kv_lens.scalar_type() == at::kInt && kv_lens.dim() == 1 && kv_lens.size(0) == seqs && kv_lens.device() == dev,
                    "kv_lens must be int32 [seqs] on the cache's device");
  if (q_starts) {
    TORCH_CHECK_VALUE(q_starts->scalar_type() == at::kInt && q_starts->dim() == 1 && q_starts->size(0) == seqs + 1 &&
                          q_starts->device() == dev,
                      "q_starts must be int32 [seqs + 1] on the cache's device");
    q_starts = q_starts->contiguous();
  }
  auto fits = [](int64_t x) { return x >= 0 && x <= INT32_MAX; };
  TORCH_CHECK_VALUE(fits(heads) && fits(seqs) && fits(pages) && fits(max_q_len) && fits(max_kv_len) && fits(window),
                    "sizes, bounds and window must be in [0, 2^31)");
  const OnDevice on(dev);
  kv_lens = kv_lens.contiguous();
  if (page_table.stride(1) != 1) page_table = page_table.contiguous();
  if (q.stride(2) != 1 || stride_of(q, 1) != q.size(2) || stride_of(q, 0) % 8 != 0 || !on_16_bytes(q)) q = copy_of(q);
  Tensor out = at::empty({tokens, heads, q.size(2)}, q.options());
  OptTensor lse;
  if (return_lse) lse = at::empty({tokens, heads}, q.options().dtype(at::kFloat));
  // without starts every sequence's tokens are as many as there are for it
  if (!q_starts && seqs > 0) max_q_len = std::min<int64_t>(tokens / seqs, INT32_MAX);
  const auto h = static_cast<int32_t>(heads), s = static_cast<int32_t>(seqs), p = static_cast<int32_t>(pages),
             mq = static_cast<int32_t>(max_q_len), mk = static_cast<int32_t>(max_kv_len);
  const size_t need = gemq_paged_attention_workspace_size(&cache.c, tokens, h, s, p, mq, mk);
  const Tensor ws = bytes(need, dev);
  const float factor = static_cast<float>(scale ? *scale : 1.0 / std::sqrt(static_cast<double>(q.size(2))));
  check(gemq_paged_attention(&cache.c, q.data_ptr(), stride_of(q, 0), tokens, h, page_table.data_ptr<int32_t>(),
                             page_table.stride(0), p, kv_lens.data_ptr<int32_t>(),
                             q_starts ? q_starts->data_ptr<int32_t>() : nullptr, s, mq, mk, factor,
                             static_cast<int32_t>(window), out.data_ptr(), lse ? lse->data_ptr<float>() : nullptr,
                             need ? ws.data_ptr() : nullptr, need, on.stream));
  return {std::move(out), std::move(lse)};
}

std::tuple<Tensor, Tensor, Tensor> verify(Tensor logits, Tensor drafts, Tensor uniforms, Tensor noise, OptTensor probs,
                                          OptTensor lens, OptTensor temperature) {
  TORCH_CHECK_VALUE(logits.is_cuda() && logits.dim() == 3 && code_of(logits.scalar_type()) >= 0,
                    "target_logits must be a CUDA tensor [seqs, drafts + 1, vocab] of float16, bfloat16 or float32");
  const auto dev = logits.device();
  const int64_t B = logits.size(0), n = logits.size(1) - 1, V = logits.size(2);
  auto is = [&](const Tensor& t, at::ScalarType kind, std::initializer_list<int64_t> shape) {
    return t.scalar_type() == kind && t.sizes() == at::IntArrayRef(shape) && t.device() == dev;
  };
  TORCH_CHECK_VALUE(is(drafts, at::kLong, {B, n}), "draft_tokens must be int64 [seqs, drafts] beside target_logits");
  TORCH_CHECK_VALUE(is(uniforms, at::kFloat, {B, n}), "uniforms must be float32 [seqs, drafts] beside target_logits");
  TORCH_CHECK_VALUE(is(noise, at::kFloat, {B, V}), "noise must be float32 [seqs, vocab] beside target_logits");
  TORCH_CHECK_VALUE(B <= INT32_MAX && n <= INT32_MAX && V <= INT32_MAX, "sizes must be below 2^31");
  const OnDevice on(dev);
  gemq_verify_t v{};
  if (logits.stride(2) != 1) logits = logits.contiguous();
  v.logits = logits.data_ptr();
  v.logits_seq_stride = logits.stride(0);
  v.logits_row_stride = logits.stride(1);
  v.logits_dtype = code_of(logits.scalar_type());
  if (probs) {
    TORCH_CHECK_VALUE(code_of(probs->scalar_type()) >= 0 && is(*probs, probs->scalar_type(), {B, n, V}),
                      "draft_probs must be [seqs, drafts, vocab] of float16, bfloat16 or float32 beside target_logits");
    if (probs->stride(2) != 1) probs = probs->contiguous();
    v.draft_probs = probs->data_ptr();
    v.probs_seq_stride = probs->stride(0);
    v.probs_row_stride = probs->stride(1);
    v.probs_dtype = code_of(probs->scalar_type());
  }
  if (lens) {
    TORCH_CHECK_VALUE(is(*lens, at::kInt, {B}), "draft_lens must be int32 [seqs] beside target_logits");
    lens = lens->contiguous();
    v.draft_lens = lens->data_ptr<int32_t>();
  }
  if (temperature) {
    TORCH_CHECK_VALUE(is(*temperature, at::kFloat, {B}), "temperature must be float32 [seqs] beside target_logits");
    temperature = temperature->contiguous();
    v.temperature = temperature->data_ptr<float>();
  }
  drafts = drafts.contiguous();
  uniforms = uniforms.contiguous();
  noise = noise.contiguous();
  v.draft_tokens = drafts.data_ptr<int64_t>();
  v.uniforms = uniforms.data_ptr<float>();
  v.noise = noise.data_ptr<float>();
  Tensor tokens = at::empty({B, n + 1}, drafts.options()), accepted = at::empty({B}, drafts.options().dtype(at::kInt)),
         logprobs = at::empty({B, n + 1}, noise.options());
  v.tokens = tokens.data_ptr<int64_t>();
  v.num_accepted = accepted.data_ptr<int32_t>();
  v.logprobs = logprobs.data_ptr<float>();
  const auto b = static_cast<int32_t>(B), d = static_cast<int32_t>(n), w = static_cast<int32_t>(V);
  const size_t need = gemq_verify_draft_workspace_size(b, d, w);
  const Tensor ws = bytes(need, dev);
  check(gemq_verify_draft(&v, b, d, w, need ? ws.data_ptr() : nullptr, need, on.stream));
  return {std::move(tokens), std::move(accepted), std::move(logprobs)};
}

}  // namespace

PYBIND11_MODULE(_serving_ext, m) {
  py::class_<Cache>(m, "Cache")
      .def(py::init<Tensor, Tensor, OptTensor, OptTensor, at::ScalarType>(), py::arg("k"), py::arg("v"), py::arg("k_scale"),
           py::arg("v_scale"), py::arg("dtype"))
      .def_readonly("k", &Cache::k)
      .def_readonly("v", &Cache::v)
      .def_readonly("k_scale", &Cache::k_scale)
      .def_readonly("v_scale", &Cache::v_scale)
      .def_property_readonly("dtype", [](const Cache& c) { return c.dtype; })
      .def_property_readonly("device", [](const Cache& c) { return c.k.device(); })
      .def_property_readonly("bits", [](const Cache& c) { return c.c.bits; })
      .def_property_readonly("num_pages", [](const Cache& c) { return c.c.num_pages; })
      .def_property_readonly("num_kv_heads", [](const Cache& c) { return c.c.kv_heads; })
      .def_property_readonly("page_size", [](const Cache& c) { return c.c.page_size; })
      .def_property_readonly("head_dim", [](const Cache& c) { return c.c.head_dim; })
      // the gemq_kv_cache_t, for callers of the C ABI; it lives as long as the cache
      .def_property_readonly("c_struct", [](const Cache& c) { return reinterpret_cast<uintptr_t>(&c.c); })
      .def("write", &Cache::write, py::arg("k"), py::arg("v"), py::arg("slots"))
      .def("read", &Cache::read, py::arg("slots"));
  m.def("attention", &attention);
  m.def("verify", &verify);
}
