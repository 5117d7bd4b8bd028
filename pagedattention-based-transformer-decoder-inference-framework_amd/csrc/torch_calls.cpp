// Module llm_torch: the calls of llm_capi.py whose arguments are many tensors (the quantised cache,
// drafted tokens, logit rules), checked and handed to the C ABI here.  From Python the checks of a
// call took 6 us of the host, twice its launch; here 1.
//
// The C entries are given by address (bind): the library that llm_capi.py has loaded is called.
#include <torch/csrc/utils/pybind.h>

#include <ATen/ATen.h>

#include <optional>
#include <sstream>

#include "llm_decoder.h"

namespace {

namespace py = pybind11;
using at::Tensor;
using MaybeTensor = std::optional<Tensor>;

decltype(&kv_quant_write) g_write;
decltype(&kv_quant_read) g_read;
decltype(&pa_tree) g_tree;
decltype(&pa_tree_workspace_bytes) g_tree_bytes;
decltype(&logits_adjust) g_adjust;

void bind(uintptr_t write, uintptr_t read, uintptr_t tree, uintptr_t tree_bytes, uintptr_t adjust) {
  g_write = reinterpret_cast<decltype(g_write)>(write);
  g_read = reinterpret_cast<decltype(g_read)>(read);
  g_tree = reinterpret_cast<decltype(g_tree)>(tree);
  g_tree_bytes = reinterpret_cast<decltype(g_tree_bytes)>(tree_bytes);
  g_adjust = reinterpret_cast<decltype(g_adjust)>(adjust);
}

[[noreturn]] void bad_value(const std::string& what) { throw py::value_error(what); }
[[noreturn]] void bad_type(const std::string& what) { throw py::type_error(what); }
void value(bool ok, const char* what) {
  if (!ok) bad_value(what);
}

// All tensors of a call are on one device, the current one (the Python side has seen to `dev`).
void on_device(const Tensor& t, int dev, const char* name) {
  if (t.get_device() != dev || !t.is_cuda())
    bad_value(std::string(name) + " is not on the device of the call's other tensors");
}

int value_dtype(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return LLM_F32;
    case at::kHalf: return LLM_F16;
    case at::kBFloat16: return LLM_BF16;
    default: bad_type(std::string(name) + " must be fp32, fp16 or bf16");
  }
}

// Address of an array that a call reads: of type and shape (empty: any), contiguous.
void* array(const Tensor& t, int dev, at::ScalarType type, at::IntArrayRef shape, const char* name) {
  on_device(t, dev, name);
  if (t.scalar_type() != type) bad_type(std::string(name) + " must be " + (type == at::kInt ? "int32" : "fp32"));
  if (!shape.empty() && t.sizes() != shape) {
    std::ostringstream s;
    s << name << " must have the shape " << shape << ", not " << t.sizes();
    bad_value(s.str());
  }
  if (!t.is_contiguous()) bad_value(std::string(name) + " must be contiguous");
  return t.data_ptr();
}
void* array(const MaybeTensor& t, int dev, at::ScalarType type, at::IntArrayRef shape, const char* name) {
  return t ? array(*t, dev, type, shape, name) : nullptr;
}
const int32_t* ints(const MaybeTensor& t, int dev, at::IntArrayRef shape, const char* name) {
  return static_cast<const int32_t*>(array(t, dev, at::kInt, shape, name));
}
const float* floats(const MaybeTensor& t, int dev, at::IntArrayRef shape, const char* name) {
  return static_cast<const float*>(array(t, dev, at::kFloat, shape, name));
}

// Elements from token to token of [B][N][H][D]: contiguous, or a view of wider tokens.
long long token_rows(const Tensor& t, const char* name) {
  const int64_t B = t.size(0), N = t.size(1), H = t.size(2), D = t.size(3);
  const int64_t step = N > 1 ? t.stride(1) : B > 1 ? t.stride(0) : H * D;
  if ((t.stride(3) != 1 && D > 1) || (t.stride(2) != D && H > 1) || (B > 1 && N > 1 && t.stride(0) != N * step) ||
      step < H * D)
    bad_value(std::string(name) + " must be [B][N][H][D] with one step between tokens and whole heads in them");
  return step;
}

pa_kv_view view_of(const Tensor& k, const Tensor& v, const Tensor& table, int dev) {
  on_device(k, dev, "k_pool");
  on_device(v, dev, "v_pool");
  if (k.scalar_type() != v.scalar_type()) bad_type("k_pool and v_pool must have the same dtype");
  value(k.dim() == 3 && v.sizes() == k.sizes(), "k_pool and v_pool must be [num_pages][ts][D], of one shape");
  const int64_t pages = k.size(0), ts = k.size(1), D = k.size(2);
  for (const Tensor& t : {k, v})
    value((t.stride(2) == 1 || D == 1) && (t.stride(1) == D || ts == 1), "pages must be contiguous");
  value(pages <= 1 || k.stride(0) == v.stride(0), "k_pool and v_pool must share one page stride");
  value(table.dim() == 3, "page_table must be [num_beams][num_heads][max_tiles]");
  value(pages <= INT32_MAX && ts <= INT32_MAX && D <= INT32_MAX && table.size(0) <= INT32_MAX &&
            table.size(1) <= INT32_MAX && table.size(2) <= INT32_MAX,
        "a dimension above 2^31 - 1");
  pa_kv_view view{};
  view.k_pool = k.data_ptr();
  view.v_pool = v.data_ptr();
  view.page_table = static_cast<int32_t*>(array(table, dev, at::kInt, {}, "page_table"));
  view.num_pages = (int32_t)pages;
  view.page_size = (int32_t)ts;
  view.head_dim = (int32_t)D;
  view.num_beams = (int32_t)table.size(0);
  view.num_heads = (int32_t)table.size(1);
  view.max_tiles = (int32_t)table.size(2);
  switch (k.scalar_type()) {
    case at::kHalf: view.kv_dtype = LLM_F16; break;
    case at::kBFloat16: view.kv_dtype = LLM_BF16; break;
    case at::kFloat: view.kv_dtype = LLM_F32; break;
    case at::kChar: view.kv_dtype = LLM_I8; break;
    case at::kFloat8_e4m3fn: view.kv_dtype = LLM_E4M3; break;
    default: bad_type("a KV pool's dtype must be fp16, bf16, fp32, int8 or float8_e4m3fn");
  }
  if (pages > 1 && k.stride(0) != ts * D) {
    value(k.stride(0) > 0, "pages must not overlap");
    view.page_stride = k.stride(0) * (int64_t)k.element_size();
  }
  return view;
}

pa_kv_scales scales_of(const Tensor& k, const Tensor& ks, const Tensor& vs, int dev) {
  const int64_t pages = k.size(0), ts = k.size(1);
  for (const Tensor& t : {ks, vs}) {
    on_device(t, dev, "a scale");
    if (t.scalar_type() != at::kFloat) bad_type("scales must be fp32");
    value(t.dim() == 2 && t.size(0) == pages && t.size(1) == ts && (t.stride(1) == 1 || ts == 1),
          "scales must be [num_pages][page_size] with contiguous pages");
  }
  value(pages <= 1 || ks.stride(0) == vs.stride(0), "k_scale and v_scale must share one page stride");
  value(pages <= 1 || ks.stride(0) > 0, "pages of scales must not overlap");
  return pa_kv_scales{ks.data_ptr<float>(), vs.data_ptr<float>(), pages > 1 ? ks.stride(0) : 0};
}

int quant(bool write, const Tensor& k, const Tensor& v, const Tensor& k_pool, const Tensor& v_pool,
          const Tensor& table, const Tensor& k_scale, const Tensor& v_scale, const Tensor& starts,
          const MaybeTensor& lens, const MaybeTensor& beam_ids, uintptr_t stream) {
  const int dev = k_pool.get_device();
  const pa_kv_view view = view_of(k_pool, v_pool, table, dev);
  const pa_kv_scales scales = scales_of(k_pool, k_scale, v_scale, dev);
  on_device(k, dev, "k");
  on_device(v, dev, "v");
  value(k.dim() == 4 && v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type() && k.size(2) == view.num_heads &&
            k.size(3) == view.head_dim,
        "k and v must be [B][N][num_heads][head_dim] of one type, as the pages are");
  const int64_t B = k.size(0), N = k.size(1);
  value(B <= INT32_MAX && N <= INT32_MAX, "too many tokens in one call");
  const int dtype = value_dtype(k, "k");
  const long long step = token_rows(k, "k");
  value(token_rows(v, "v") == step, "k and v must have one step between tokens");
  value(beam_ids || B <= view.num_beams, "more rows than page_table has beams");
  const int32_t* at = ints(starts, dev, {B}, "starts");
  const int32_t* n = ints(lens, dev, {B}, "lens");
  const int32_t* beams = ints(beam_ids, dev, {B}, "beam_ids");
  void* st = reinterpret_cast<void*>(stream);
  return write ? g_write(&view, &scales, k.data_ptr(), v.data_ptr(), dtype, step, beams, at, n, (int)B, (int)N, st)
               : g_read(&view, &scales, k.data_ptr(), v.data_ptr(), dtype, step, beams, at, n, (int)B, (int)N, st);
}

// A result's tensor, or the status of a call that failed.
py::object result(int rc, const Tensor& out) { return rc ? py::object(py::int_(rc)) : py::cast(out); }

py::object tree(const Tensor& q, const Tensor& k_pool, const Tensor& v_pool, const Tensor& table,
                const MaybeTensor& k_scale, const MaybeTensor& v_scale, const MaybeTensor& context_lens,
                const MaybeTensor& mask, const MaybeTensor& tree_lens, const MaybeTensor& beam_ids, int T,
                float sm_scale, const MaybeTensor& given, uintptr_t stream) {
  const int dev = k_pool.get_device();
  const pa_kv_view view = view_of(k_pool, v_pool, table, dev);
  pa_kv_scales scales{};
  value(k_scale.has_value() == v_scale.has_value(), "scales must be (k_scale, v_scale)");
  if (k_scale) scales = scales_of(k_pool, *k_scale, *v_scale, dev);
  on_device(q, dev, "q");
  value(q.dim() == 4, "q must be [B][N][H][D]");
  const int64_t B = q.size(0), N = q.size(1), H = q.size(2), D = q.size(3);
  value(B <= INT32_MAX && N <= INT32_MAX && H <= INT32_MAX && D <= INT32_MAX, "a dimension above 2^31 - 1");
  const int dtype = value_dtype(q, "q");
  const long long q_step = token_rows(q, "q");
  value(beam_ids || B <= view.num_beams, "more rows than page_table has beams");
  const int32_t* at = ints(context_lens, dev, {B}, "context_lens");
  const int32_t* n = ints(tree_lens, dev, {B}, "tree_lens");
  const int32_t* beams = ints(beam_ids, dev, {B}, "beam_ids");
  const int32_t* words = ints(mask, dev, {B, N, (N + 31) / 32}, "tree_mask");
  if (given)
    value(given->sizes() == q.sizes() && given->scalar_type() == q.scalar_type() && given->get_device() == dev,
          "out must have q's shape, type and device");
  const Tensor out = given       ? *given
                     : tree_lens ? at::zeros(q.sizes(), q.options())
                                 : at::empty(q.sizes(), q.options());
  const long long out_step = token_rows(out, "out");
  const size_t need = g_tree_bytes(&view, (int)B, (int)N, (int)H, T);
  const Tensor ws = need ? at::empty({(int64_t)need}, q.options().dtype(at::kByte)) : Tensor();
  return result(g_tree(&view, k_scale ? &scales : nullptr, q.data_ptr(), q_step, out.data_ptr(), out_step, dtype,
                       beams, at, reinterpret_cast<const uint32_t*>(words), n, (int)B, (int)N, (int)H, (int)D, T,
                       sm_scale, need ? ws.data_ptr() : nullptr, need, reinterpret_cast<void*>(stream)),
                out);
}

py::object adjust(const Tensor& logits, const MaybeTensor& history, const MaybeTensor& history_lens,
                  const MaybeTensor& prompt_lens, const MaybeTensor& repetition, const MaybeTensor& frequency,
                  const MaybeTensor& presence, const MaybeTensor& bias_ids, const MaybeTensor& bias,
                  const MaybeTensor& allowed, const MaybeTensor& allowed_rows, const MaybeTensor& given,
                  uintptr_t stream) {
  const int dev = logits.get_device();
  const int dtype = value_dtype(logits, "logits");
  on_device(logits, dev, "logits");
  value(logits.dim() == 2, "logits must be [R][V]");
  const int64_t R = logits.size(0), V = logits.size(1);
  value(R <= INT32_MAX && V <= INT32_MAX, "a dimension above 2^31 - 1");
  const int64_t step = R > 1 ? logits.stride(0) : V;
  value((logits.stride(1) == 1 || V <= 1) && step >= V, "logits must be [R][V] with contiguous rows");
  if (given)
    value(given->sizes() == logits.sizes() && given->scalar_type() == logits.scalar_type() &&
              given->get_device() == dev && (given->stride(1) == 1 || V <= 1) && (R <= 1 || given->stride(0) == step),
          "out must have the logits' shape, type, strides and device");
  // entries of a row in [R][n] or [n], and from row to row
  auto entries = [&](const Tensor& t, const char* name, long long& stride) -> int {
    value(t.dim() == 1 || (t.dim() == 2 && t.size(0) == R), name);
    const int64_t n = t.size(t.dim() - 1);
    value(n <= INT32_MAX, name);
    stride = t.dim() == 2 ? n : 0;
    return (int)n;
  };
  logits_rules r{};
  if (history) r.history_len = entries(*history, "history must be [R][n] or [n]", r.history_stride);
  r.history = ints(history, dev, {}, "history");
  r.history_lens = ints(history_lens, dev, {R}, "history_lens");
  r.prompt_lens = ints(prompt_lens, dev, {R}, "prompt_lens");
  r.repetition = floats(repetition, dev, {R}, "repetition");
  r.frequency = floats(frequency, dev, {R}, "frequency");
  r.presence = floats(presence, dev, {R}, "presence");
  if (history && !r.history_len) {  // (an empty list has no address)
    r.history = r.history_lens = r.prompt_lens = nullptr;
    r.repetition = r.frequency = r.presence = nullptr;
  }
  value(bias.has_value() == bias_ids.has_value() && (!bias || bias->sizes() == bias_ids->sizes()),
        "bias_ids and bias go together, of one shape");
  if (bias) r.bias_len = entries(*bias_ids, "bias_ids must be [R][n] or [n]", r.bias_stride);
  r.bias_ids = ints(bias_ids, dev, {}, "bias_ids");
  r.bias = floats(bias, dev, {}, "bias");
  if (bias && !r.bias_len) r.bias_ids = nullptr, r.bias = nullptr;
  if (allowed) {
    value(allowed->dim() == 2 && allowed->size(1) == (V + 31) / 32 && allowed->size(0) <= INT32_MAX,
          "allowed must be [masks][ceil(V / 32)]");
    // (a list of no masks has no address, by which the library would take it for none asked for)
    value(allowed_rows || allowed->size(0) >= R, "without allowed_rows every row needs a mask of its own in allowed");
    r.num_masks = (int)allowed->size(0);
  }
  r.allowed = reinterpret_cast<const uint32_t*>(ints(allowed, dev, {}, "allowed"));
  r.allowed_rows = ints(allowed_rows, dev, {R}, "allowed_rows");
  const Tensor out = given ? *given : at::empty_strided({R, V}, {step, 1}, logits.options());
  return result(g_adjust(logits.data_ptr(), out.data_ptr(), dtype, (int)R, (int)V, step, &r,
                         reinterpret_cast<void*>(stream)),
                out);
}

}  // namespace

PYBIND11_MODULE(llm_torch, m) {
  m.def("bind", &bind);
  m.def("quant", &quant);
  m.def("tree", &tree);
  m.def("adjust", &adjust);
}
