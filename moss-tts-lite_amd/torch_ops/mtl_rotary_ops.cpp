// torch dispatcher operators of the rotation of queries and keys over the C ABI in mtl_rotary.h:
// mtl::qk_rotary and mtl::qk_rotary_ (in place).  Host code only; meta kernels make the same
// checks and give the output shapes to tracing.
#include "mtl_op_checks.h"
#include "mtl_rotary.h"

namespace {

using namespace mtl_ops;

constexpr const char* kWhat = "the rotation of queries and keys";

struct Call {
  int32_t type = 0, turned = 0;
  int64_t rows = 0, dim = 0;
};

Call check_call(const at::Tensor& q, const at::Tensor& k, const at::Tensor& positions,
                const at::Tensor& freqs, const OptTensor& q_norm, const OptTensor& k_norm) {
  Call c;
  c.type = row_type(q, "q");
  TORCH_CHECK(k.scalar_type() == q.scalar_type(), "q and k must have one type, got ",
              q.scalar_type(), " and ", k.scalar_type());
  TORCH_CHECK(q.dim() == 3 && k.dim() == 3, "q and k must be [rows, heads, head_dim], got ",
              q.sizes(), " and ", k.sizes());
  c.rows = q.size(0);
  c.dim = q.size(2);
  TORCH_CHECK(k.size(0) == c.rows && k.size(2) == c.dim, "q and k must have the same rows and "
              "head_dim, got ", q.sizes(), " and ", k.sizes());
  TORCH_CHECK(c.dim >= 8 && c.dim <= 512 && c.dim % 8 == 0, "head_dim must be a multiple of 8 "
              "from 8 to 512, got ", c.dim);
  TORCH_CHECK(c.rows <= (int64_t{1} << 25) && q.size(1) <= 65535 && k.size(1) <= 65535,
              "at most 2^25 rows and 65535 heads, got ", q.sizes(), " and ", k.sizes());
  check_same_device(q, {&k, &positions, &freqs}, kWhat);
  TORCH_CHECK(positions.scalar_type() == at::kLong && positions.dim() == 1 &&
                  positions.size(0) == c.rows && positions.is_contiguous(),
              "positions must be contiguous int64 [", c.rows, "]");
  TORCH_CHECK(freqs.scalar_type() == at::kDouble && freqs.dim() == 1 && freqs.is_contiguous() &&
                  2 * freqs.size(0) <= c.dim,
              "freqs must be contiguous float64 [turned / 2], turned at most ", c.dim, ", got ",
              freqs.scalar_type(), " ", freqs.sizes());
  c.turned = (int32_t)(2 * freqs.size(0));
  for (const OptTensor* w : {&q_norm, &k_norm}) {
    if (!w->has_value()) continue;
    TORCH_CHECK((*w)->scalar_type() == q.scalar_type() && (*w)->dim() == 1 &&
                    (*w)->size(0) == c.dim && (*w)->is_contiguous(),
                "norm weights must be contiguous ", q.scalar_type(), " [", c.dim, "]");
    check_same_device(q, {&**w}, kWhat);
  }
  return c;
}

// Whether the kernel takes t as it is: heads in 16-byte pieces.
bool fits(const at::Tensor& t) {
  return t.stride(2) == 1 && step(t, 0) % 8 == 0 && step(t, 1) % 8 == 0 &&
         (t.is_meta() || aligned16(t.data_ptr()));
}

at::Tensor whole(const at::Tensor& t) {
  return aligned16(t.data_ptr()) ? t : t.clone(at::MemoryFormat::Contiguous);
}

mtl_rotary_heads heads_of(const at::Tensor& x, const at::Tensor& out, const OptTensor& norm,
                          at::Tensor& keep) {
  if (norm.has_value()) keep = whole(*norm);
  return mtl_rotary_heads{ptr<void>(x), step(x, 0), step(x, 1), ptr<void>(out), step(out, 0),
                          step(out, 1), norm.has_value() ? keep.data_ptr() : nullptr,
                          (int32_t)x.size(1)};
}

void rotate(const Call& c, const at::Tensor& q, const at::Tensor& k, const at::Tensor& q_out,
            const at::Tensor& k_out, const at::Tensor& positions, const at::Tensor& freqs,
            const OptTensor& q_norm, const OptTensor& k_norm, double eps, bool interleaved,
            double amplitude) {
  at::Tensor keep[2];
  const mtl_rotary_heads a = heads_of(q, q_out, q_norm, keep[0]);
  const mtl_rotary_heads b = heads_of(k, k_out, k_norm, keep[1]);
  check_status(mtl_qk_rotary(&a, &b, c.rows, (int32_t)c.dim, ptr<int64_t>(positions),
                             ptr<double>(freqs), c.turned, interleaved, (float)amplitude,
                             (float)eps, c.type, stream_of(q)),
               "mtl_qk_rotary");
}

std::tuple<at::Tensor, at::Tensor> qk_rotary(const at::Tensor& q, const at::Tensor& k,
                                             const at::Tensor& positions, const at::Tensor& freqs,
                                             const OptTensor& q_norm, const OptTensor& k_norm,
                                             double eps, bool interleaved, double amplitude) {
  const Call c = check_call(q, k, positions, freqs, q_norm, k_norm);
  at::Tensor q_out = at::empty({c.rows, q.size(1), c.dim}, q.options());
  at::Tensor k_out = at::empty({c.rows, k.size(1), c.dim}, k.options());
  if (q.is_meta() || c.rows == 0) return {q_out, k_out};
  const c10::DeviceGuard guard(q.device());
  // heads come in 16-byte pieces: any other view is copied
  rotate(c, fits(q) ? q : whole(q.contiguous()), fits(k) ? k : whole(k.contiguous()), q_out, k_out,
         positions, freqs, q_norm, k_norm, eps, interleaved, amplitude);
  return {q_out, k_out};
}

// q and k that are written: whether they can be seen to lie apart.  Views of the rows of one
// matrix repeat with one stride; theirs are the columns they take of it.
bool apart(const at::Tensor& q, const at::Tensor& k) {
  if (!q.has_storage() || !k.has_storage() ||
      q.storage().unsafeGetStorageImpl() != k.storage().unsafeGetStorageImpl() ||
      q.numel() == 0 || k.numel() == 0)
    return true;
  auto reach = [](const at::Tensor& t, int64_t from) {
    int64_t n = 1;
    for (int64_t d = from; d < 3; ++d) n += (t.size(d) - 1) * t.stride(d);
    return n;
  };
  const int64_t a = q.storage_offset(), b = k.storage_offset();
  if (a + reach(q, 0) <= b || b + reach(k, 0) <= a) return true;
  const int64_t ld = q.stride(0);
  if (q.size(0) < 2 || k.stride(0) != ld) return false;
  const int64_t ahead = ((b - a) % ld + ld) % ld;           // k's columns from q's first on
  return reach(q, 1) <= ahead && ahead + reach(k, 1) <= ld;
}

void qk_rotary_(at::Tensor& q, at::Tensor& k, const at::Tensor& positions, const at::Tensor& freqs,
                const OptTensor& q_norm, const OptTensor& k_norm, double eps, bool interleaved,
                double amplitude) {
  const Call c = check_call(q, k, positions, freqs, q_norm, k_norm);
  for (const auto& [t, name] : {std::pair<const at::Tensor&, const char*>(q, "q"),
                                std::pair<const at::Tensor&, const char*>(k, "k")}) {
    TORCH_CHECK(t.numel() == 0 || fits(t), name, " must have unit last stride, other strides of "
                "multiples of 8 and a 16-byte aligned base to be rotated in place");
    check_apart(t, name);
  }
  TORCH_CHECK(apart(q, k), "q and k share memory");
  if (q.is_meta() || c.rows == 0) return;
  const c10::DeviceGuard guard(q.device());
  rotate(c, q, k, q, k, positions, freqs, q_norm, k_norm, eps, interleaved, amplitude);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(mtl, m) {
  m.def("qk_rotary(Tensor q, Tensor k, Tensor positions, Tensor freqs, Tensor? q_norm=None, "
        "Tensor? k_norm=None, float eps=1e-6, bool interleaved=False, float amplitude=1.0) "
        "-> (Tensor, Tensor)");
  m.def("qk_rotary_(Tensor(a!) q, Tensor(b!) k, Tensor positions, Tensor freqs, "
        "Tensor? q_norm=None, Tensor? k_norm=None, float eps=1e-6, bool interleaved=False, "
        "float amplitude=1.0) -> ()");
}

TORCH_LIBRARY_IMPL(mtl, CUDA, m) {
  m.impl("qk_rotary", &qk_rotary);
  m.impl("qk_rotary_", &qk_rotary_);
}

TORCH_LIBRARY_IMPL(mtl, Meta, m) {
  m.impl("qk_rotary", &qk_rotary);
  m.impl("qk_rotary_", &qk_rotary_);
}
