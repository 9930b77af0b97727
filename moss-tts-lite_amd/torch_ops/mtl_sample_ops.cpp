// torch dispatcher operators of drawing tokens over the C ABI in mtl_sample.h: mtl::sample and
// mtl::sample_logprob.  Host code only; meta kernels make the same checks and give the output
// shapes to tracing.
#include <cmath>

#include "mtl_op_checks.h"
#include "mtl_sample.h"

namespace {

using namespace mtl_ops;

constexpr const char* kWhat = "the draw of tokens";

// A setting of each row, or null.
template <class T>
const T* rows_of(const OptTensor& t, const at::Tensor& logits, at::ScalarType type,
                 const char* name) {
  if (!t.has_value()) return nullptr;
  TORCH_CHECK(t->scalar_type() == type && t->dim() == 1 && t->size(0) == logits.size(0) &&
                  t->is_contiguous(),
              name, " must be a number or contiguous ", type, " [", logits.size(0), "], got ",
              t->scalar_type(), " ", t->sizes());
  check_same_device(logits, {&*t}, kWhat);
  return ptr<T>(*t);
}

at::Tensor draw(const at::Tensor& logits, const at::Tensor& u, const OptTensor& temperature,
                const OptTensor& top_k, const OptTensor& top_p, const OptTensor& min_p,
                double temperature_all, int64_t top_k_all, double top_p_all, double min_p_all,
                at::Tensor* logprob) {
  TORCH_CHECK(logits.dim() == 2, "logits must be [rows, vocab], got ", logits.sizes());
  const bool f32 = logits.scalar_type() == at::kFloat;
  TORCH_CHECK(f32 || logits.scalar_type() == at::kBFloat16 || logits.scalar_type() == at::kHalf,
              "expected logits to be float32, bfloat16 or float16, got ", logits.scalar_type());
  const int64_t rows = logits.size(0), vocab = logits.size(1);
  TORCH_CHECK(vocab >= 1 && vocab <= (1 << 20) && rows <= 65535,
              "1 to 2^20 tokens and at most 65535 rows, got ", logits.sizes());
  TORCH_CHECK(u.scalar_type() == at::kFloat && u.dim() == 1 && u.size(0) == rows &&
                  u.is_contiguous(),
              "u must be contiguous float32 [", rows, "], got ", u.scalar_type(), " ", u.sizes());
  check_same_device(logits, {&u}, kWhat);
  TORCH_CHECK(std::isfinite(temperature_all) && !std::isnan(top_p_all) && !std::isnan(min_p_all),
              "temperature must be finite, top_p and min_p numbers");
  mtl_sample_settings s{};
  s.temperature = rows_of<float>(temperature, logits, at::kFloat, "temperature");
  s.top_k = rows_of<int32_t>(top_k, logits, at::kInt, "top_k");
  s.top_p = rows_of<float>(top_p, logits, at::kFloat, "top_p");
  s.min_p = rows_of<float>(min_p, logits, at::kFloat, "min_p");
  s.temperature_all = (float)temperature_all;
  s.top_k_all = (int32_t)std::min<int64_t>(std::max<int64_t>(top_k_all, 0), INT32_MAX);
  s.top_p_all = (float)top_p_all;
  s.min_p_all = (float)min_p_all;
  const int32_t type = f32 ? MTL_T_F32 : row_type(logits, "logits");
  at::Tensor token = at::empty({rows}, logits.options().dtype(at::kLong));
  if (logprob) *logprob = at::empty({rows}, logits.options().dtype(at::kFloat));
  if (logits.is_meta() || rows == 0) return token;
  const c10::DeviceGuard guard(logits.device());
  // a row's tokens lie side by side: any other view is copied
  const at::Tensor x = vocab == 1 || logits.stride(1) == 1 ? logits : logits.contiguous();
  const Workspace ws(x, mtl_sample_workspace_bytes(rows, vocab, type, &s));
  check_status(mtl_sample(x.data_ptr(), step(x, 0), rows, vocab, type, ptr<float>(u), &s,
                          ptr<int64_t>(token), logprob ? ptr<float>(*logprob) : nullptr, ws.get(),
                          ws.bytes, stream_of(x)),
               "mtl_sample");
  return token;
}

at::Tensor sample(const at::Tensor& logits, const at::Tensor& u, const OptTensor& temperature,
                  const OptTensor& top_k, const OptTensor& top_p, const OptTensor& min_p,
                  double temperature_all, int64_t top_k_all, double top_p_all, double min_p_all) {
  return draw(logits, u, temperature, top_k, top_p, min_p, temperature_all, top_k_all, top_p_all,
              min_p_all, nullptr);
}

std::tuple<at::Tensor, at::Tensor> sample_logprob(
    const at::Tensor& logits, const at::Tensor& u, const OptTensor& temperature,
    const OptTensor& top_k, const OptTensor& top_p, const OptTensor& min_p, double temperature_all,
    int64_t top_k_all, double top_p_all, double min_p_all) {
  at::Tensor logprob;
  at::Tensor token = draw(logits, u, temperature, top_k, top_p, min_p, temperature_all, top_k_all,
                          top_p_all, min_p_all, &logprob);
  return {token, logprob};
}

}  // namespace

#define MTL_SAMPLE_ARGS                                                                        \
  "(Tensor logits, Tensor u, Tensor? temperature=None, Tensor? top_k=None, Tensor? top_p=None, " \
  "Tensor? min_p=None, float temperature_all=1.0, int top_k_all=0, float top_p_all=1.0, "      \
  "float min_p_all=0.0)"

TORCH_LIBRARY_FRAGMENT(mtl, m) {
  m.def("sample" MTL_SAMPLE_ARGS " -> Tensor");
  m.def("sample_logprob" MTL_SAMPLE_ARGS " -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(mtl, CUDA, m) {
  m.impl("sample", &sample);
  m.impl("sample_logprob", &sample_logprob);
}

TORCH_LIBRARY_IMPL(mtl, Meta, m) {
  m.impl("sample", &sample);
  m.impl("sample_logprob", &sample_logprob);
}
