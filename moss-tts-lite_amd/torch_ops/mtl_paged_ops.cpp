// torch dispatcher operators of the paged key-value cache over the C ABI in mtl_paged.h:
// mtl::paged_attention(_lse), mtl::paged_attention_shared(_lse), mtl::paged_write,
// mtl::pages_extend, mtl::pages_fork, mtl::pages_truncate, mtl::pages_compact and
// mtl::pages_copy.
//
// Host code only, as mtl_torch_ops.cpp: each operator checks its tensors, takes outputs and
// workspaces from torch's caching allocator and calls the C entry on torch's current stream of
// the tensors' device.  A workspace belongs to one call, so calls on several streams and
// graphs captured from them share nothing.  Meta kernels make the same checks and give the
// output shapes to tracing.
#include "mtl_op_checks.h"

namespace {

using namespace mtl_ops;

void check_int32(const at::Tensor& t, int64_t dim, const char* name) {
  TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == dim, name, " must be a ", dim,
              "-D int32 tensor, got ", t.scalar_type(), " ", t.sizes());
  TORCH_CHECK(t.size(dim - 1) <= 1 || t.numel() == 0 || t.stride(dim - 1) == 1, name,
              " must have unit last stride");
}

void check_page_size(int64_t ps) {
  TORCH_CHECK(ps == 16 || ps == 32 || ps == 64 || ps == 128 || ps == 256,
              "page_size must be 16, 32, 64, 128 or 256, got ", ps);
}

void check_scale(const OptTensor& s, const at::Tensor& pages, const char* name) {
  if (!s.has_value()) return;
  TORCH_CHECK(pages.scalar_type() == at::kFloat8_e4m3fn, name, " goes with float8_e4m3fn pages");
  TORCH_CHECK(s->scalar_type() == at::kFloat && s->dim() == 1 && s->size(0) == pages.size(1) &&
                  s->is_contiguous(),
              name, " must be contiguous float32 [", pages.size(1), "]");
  check_same_device(pages, {&*s});
}

// Keys and values that are written, of one type: dense blocks of one storage must not meet.  Where
// both get the same bytes (`same`) they may be one.
void check_pools_apart(const at::Tensor& k, const at::Tensor& v, bool same) {
  if (!k.has_storage() || !v.has_storage() ||
      k.storage().unsafeGetStorageImpl() != v.storage().unsafeGetStorageImpl() ||
      !k.is_non_overlapping_and_dense() || !v.is_non_overlapping_and_dense() ||
      (same && k.storage_offset() == v.storage_offset() && k.strides() == v.strides()))
    return;
  TORCH_CHECK(k.storage_offset() + k.numel() <= v.storage_offset() ||
                  v.storage_offset() + v.numel() <= k.storage_offset(),
              "k_pages and v_pages share memory");
}

// One layer's pages [pages, kv_heads, page_size, head_dim] with any strides that keep the
// head_dim elements of a row adjacent and rows 16-byte aligned.
mtl_page_pool pool_of(const at::Tensor& k, const at::Tensor& v, const OptTensor& k_scale,
                      const OptTensor& v_scale, int32_t type) {
  for (const auto& [t, name] : {std::pair<const at::Tensor&, const char*>(k, "k_pages"),
                                std::pair<const at::Tensor&, const char*>(v, "v_pages")}) {
    TORCH_CHECK(t.dim() == 4, name, " must be [pages, kv_heads, page_size, head_dim], got ",
                t.sizes());
    const bool e4m3 = t.scalar_type() == at::kFloat8_e4m3fn;
    TORCH_CHECK(e4m3 || t.scalar_type() == (type == MTL_T_BF16 ? at::kBFloat16 : at::kHalf), name,
                " must have the rows' type or be float8_e4m3fn, got ", t.scalar_type());
    TORCH_CHECK(t.size(0) >= 1 && t.size(1) >= 1, name, " must hold at least one page and head");
    const int64_t piece = e4m3 ? 16 : 8;
    TORCH_CHECK(t.stride(3) != 1 || t.stride(2) >= t.size(3), name, "'s rows must not overlap");
    TORCH_CHECK(t.stride(3) == 1 && step(t, 0) % piece == 0 && step(t, 1) % piece == 0 &&
                    t.stride(2) % piece == 0 && (t.is_meta() || aligned16(t.data_ptr())),
                name, " must have unit last stride, other strides of multiples of 16 bytes and a "
                "16-byte aligned base");
  }
  TORCH_CHECK(k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type(),
              "k_pages and v_pages must have the same shape and type");
  check_same_device(k, {&v});
  TORCH_CHECK(k.size(0) <= INT32_MAX && k.size(1) <= 65535,
              "at most 2^31 - 1 pages and 65535 kv heads, got ", k.sizes());
  TORCH_CHECK(k.size(3) == 64 || k.size(3) == 128, "head_dim must be 64 or 128, got ", k.size(3));
  check_page_size(k.size(2));
  check_scale(k_scale, k, "k_scale");
  check_scale(v_scale, v, "v_scale");
  mtl_page_pool p{};
  p.k = ptr<void>(k);
  p.v = ptr<void>(v);
  p.pages = k.size(0);
  p.k_page = step(k, 0);
  p.k_head = step(k, 1);
  p.k_token = k.stride(2);
  p.v_page = step(v, 0);
  p.v_head = step(v, 1);
  p.v_token = v.stride(2);
  p.kv_heads = (int32_t)k.size(1);
  p.page_size = (int32_t)k.size(2);
  p.head_dim = (int32_t)k.size(3);
  p.type = k.scalar_type() == at::kFloat8_e4m3fn ? MTL_T_E4M3 : type;
  p.k_scale = k_scale.has_value() ? ptr<float>(*k_scale) : nullptr;
  p.v_scale = v_scale.has_value() ? ptr<float>(*v_scale) : nullptr;
  return p;
}

mtl_page_table table_of(const at::Tensor& table) {
  check_int32(table, 2, "table");
  mtl_page_table t{};
  t.table = ptr<int32_t>(table);
  t.ld = std::max(step(table, 0), table.size(1));
  t.width = table.size(1);
  t.seqs = table.size(0);
  TORCH_CHECK(t.seqs <= 1 || table.stride(0) >= t.width, "table rows must not overlap");
  return t;
}

// Which sequences share a prefix, and how much of it.
struct Groups {
  const at::Tensor& starts;
  const at::Tensor& shared;
};

// out, and where lse is not null the log-sum-exp
at::Tensor attend(const at::Tensor& q, const at::Tensor& k_pages, const at::Tensor& v_pages,
                  const at::Tensor& table, const at::Tensor& lens, double scale,
                  const OptTensor& k_scale, const OptTensor& v_scale, at::Tensor* lse,
                  const Groups* groups = nullptr) {
  TORCH_CHECK(q.dim() == 3, "q must be [sequences, heads, head_dim], got ", q.sizes());
  const int32_t type = row_type(q, "q");
  const mtl_page_pool pool = pool_of(k_pages, v_pages, k_scale, v_scale, type);
  const mtl_page_table tab = table_of(table);
  check_int32(lens, 1, "lens");
  check_same_device(q, {&k_pages, &table, &lens});
  const int64_t b = q.size(0), h = q.size(1);
  TORCH_CHECK(q.size(2) == pool.head_dim, "q has head_dim ", q.size(2), ", the pages ",
              pool.head_dim);
  TORCH_CHECK(h >= 1 && h % pool.kv_heads == 0, "q's ", h, " heads must be a multiple of the ",
              pool.kv_heads, " kv heads");
  TORCH_CHECK(h <= 65535 && b <= 65535, "at most 65535 heads and 65535 sequences, got ", q.sizes());
  TORCH_CHECK(tab.width <= (int64_t{1} << 30) / pool.page_size,
              "a sequence has at most 2^30 positions, the table ", tab.width, " pages of ",
              pool.page_size);
  TORCH_CHECK(tab.seqs == b && lens.size(0) == b, "q, table and lens must have the same number of "
              "sequences, got ", b, ", ", tab.seqs, " and ", lens.size(0));
  int64_t n_groups = 0;
  if (groups) {
    check_int32(groups->starts, 1, "groups");
    check_int32(groups->shared, 1, "shared");
    check_same_device(q, {&groups->starts, &groups->shared});
    n_groups = groups->shared.size(0);
    TORCH_CHECK(groups->starts.size(0) == n_groups + 1, "groups must be int32 [", n_groups + 1,
                "], one more than shared, got ", groups->starts.sizes());
    TORCH_CHECK(n_groups <= 65535, "at most 65535 groups, got ", n_groups);
    const int64_t columns = (h / pool.kv_heads + 15) / 16 + 2;
    TORCH_CHECK(b * h < (1 << 26) && (b * columns + n_groups) *
                        (tab.width * pool.page_size / 128 + 2) < (1 << 27),
                "too many sequences, groups or pages for one call: q ", q.sizes(), ", table ",
                table.sizes());
  }
  at::Tensor out = at::empty({b, h, q.size(2)}, q.options());
  if (lse) *lse = at::empty({b, h}, q.options().dtype(at::kFloat));
  if (q.is_meta() || b == 0) return out;
  const c10::DeviceGuard guard(q.device());
  // the kernel reads q in 16-byte pieces: any other view is copied
  at::Tensor q2 = q;
  if (q.stride(2) != 1 || step(q, 0) % 8 || step(q, 1) % 8 || !aligned16(q.data_ptr())) {
    q2 = q.contiguous();
    if (!aligned16(q2.data_ptr())) q2 = q2.clone();
  }
  if (groups) {
    const Workspace ws(q, mtl_paged_attention_shared_workspace_bytes(
                              b, n_groups, (int32_t)h, pool.kv_heads, pool.head_dim, tab.width,
                              pool.page_size));
    check_status(mtl_paged_attention_shared(
                     q2.data_ptr(), step(q2, 0), step(q2, 1), &pool, &tab, ptr<int32_t>(lens),
                     ptr<int32_t>(groups->starts), ptr<int32_t>(groups->shared), n_groups,
                     (int32_t)h, type, (float)scale, out.data_ptr(),
                     lse ? ptr<float>(*lse) : nullptr, ws.get(), ws.bytes, stream_of(q)),
                 "mtl_paged_attention_shared");
    return out;
  }
  const Workspace ws(q, mtl_paged_attention_workspace_bytes(
                            b, (int32_t)h, pool.kv_heads, pool.head_dim, tab.width,
                            pool.page_size));
  check_status(mtl_paged_attention(q2.data_ptr(), step(q2, 0), step(q2, 1), &pool, &tab,
                                   ptr<int32_t>(lens), (int32_t)h, type, (float)scale,
                                   out.data_ptr(), lse ? ptr<float>(*lse) : nullptr, ws.get(),
                                   ws.bytes, stream_of(q)),
               "mtl_paged_attention");
  return out;
}

at::Tensor paged_attention(const at::Tensor& q, const at::Tensor& k_pages,
                           const at::Tensor& v_pages, const at::Tensor& table,
                           const at::Tensor& lens, double scale, const OptTensor& k_scale,
                           const OptTensor& v_scale) {
  return attend(q, k_pages, v_pages, table, lens, scale, k_scale, v_scale, nullptr);
}

std::tuple<at::Tensor, at::Tensor> paged_attention_lse(
    const at::Tensor& q, const at::Tensor& k_pages, const at::Tensor& v_pages,
    const at::Tensor& table, const at::Tensor& lens, double scale, const OptTensor& k_scale,
    const OptTensor& v_scale) {
  at::Tensor lse;
  at::Tensor out = attend(q, k_pages, v_pages, table, lens, scale, k_scale, v_scale, &lse);
  return {out, lse};
}

at::Tensor paged_attention_shared(const at::Tensor& q, const at::Tensor& k_pages,
                                  const at::Tensor& v_pages, const at::Tensor& table,
                                  const at::Tensor& lens, const at::Tensor& groups,
                                  const at::Tensor& shared, double scale, const OptTensor& k_scale,
                                  const OptTensor& v_scale) {
  const Groups g{groups, shared};
  return attend(q, k_pages, v_pages, table, lens, scale, k_scale, v_scale, nullptr, &g);
}

std::tuple<at::Tensor, at::Tensor> paged_attention_shared_lse(
    const at::Tensor& q, const at::Tensor& k_pages, const at::Tensor& v_pages,
    const at::Tensor& table, const at::Tensor& lens, const at::Tensor& groups,
    const at::Tensor& shared, double scale, const OptTensor& k_scale, const OptTensor& v_scale) {
  const Groups g{groups, shared};
  at::Tensor lse;
  at::Tensor out = attend(q, k_pages, v_pages, table, lens, scale, k_scale, v_scale, &lse, &g);
  return {out, lse};
}

at::Tensor paged_write(const at::Tensor& qkv, const at::Tensor& k_pages, const at::Tensor& v_pages,
                       const at::Tensor& table, const at::Tensor& positions, const OptTensor& seqs,
                       const OptTensor& q_norm, const OptTensor& k_norm, const OptTensor& cos,
                       const OptTensor& sin, double eps, const OptTensor& k_scale,
                       const OptTensor& v_scale) {
  TORCH_CHECK(qkv.dim() == 2, "qkv must be [rows, (heads + 2 kv_heads) * head_dim], got ",
              qkv.sizes());
  const int32_t type = row_type(qkv, "qkv");
  const mtl_page_pool pool = pool_of(k_pages, v_pages, k_scale, v_scale, type);
  check_apart(k_pages, "k_pages");
  check_apart(v_pages, "v_pages");
  check_pools_apart(k_pages, v_pages, false);
  const mtl_page_table tab = table_of(table);
  const int64_t rows = qkv.size(0), d = pool.head_dim;
  const int64_t heads = qkv.size(1) / d - 2 * (int64_t)pool.kv_heads;
  TORCH_CHECK(qkv.size(1) % d == 0 && heads >= 1, "qkv has ", qkv.size(1),
              " columns: (heads + 2 * ", pool.kv_heads, ") * ", d, " are expected");
  TORCH_CHECK(heads + 2 * (int64_t)pool.kv_heads <= 65535 && rows <= UINT32_MAX / 256,
              "at most 65535 heads of q, k and v and 2^24 - 1 rows, got ", qkv.sizes());
  check_same_device(qkv, {&k_pages, &table, &positions});
  TORCH_CHECK(positions.scalar_type() == at::kLong && positions.dim() == 1 &&
                  positions.size(0) == rows && positions.is_contiguous(),
              "positions must be contiguous int64 [", rows, "]");
  if (seqs.has_value()) {
    check_int32(*seqs, 1, "seqs");
    TORCH_CHECK(seqs->size(0) == rows, "seqs must be int32 [", rows, "]");
    check_same_device(qkv, {&*seqs});
  } else {
    TORCH_CHECK(rows <= tab.seqs, "without seqs row r is sequence r: ", rows, " rows, ", tab.seqs,
                " sequences");
  }
  TORCH_CHECK(q_norm.has_value() == k_norm.has_value(), "give both q_norm and k_norm or neither");
  TORCH_CHECK(cos.has_value() == sin.has_value(), "give both cos and sin or neither");
  for (const OptTensor* w : {&q_norm, &k_norm}) {
    if (!w->has_value()) continue;
    TORCH_CHECK((*w)->scalar_type() == qkv.scalar_type() && (*w)->dim() == 1 &&
                    (*w)->size(0) == d && (*w)->is_contiguous(),
                "norm weights must be contiguous ", qkv.scalar_type(), " [", d, "]");
    check_same_device(qkv, {&**w});
  }
  int32_t rope_f32 = 0;
  int64_t rope_rows = 0;
  if (cos.has_value()) {
    rope_f32 = cos->scalar_type() == at::kFloat;
    rope_rows = cos->size(0);
    for (const OptTensor* c : {&cos, &sin}) {
      TORCH_CHECK(((*c)->scalar_type() == at::kFloat ||
                   (*c)->scalar_type() == qkv.scalar_type()) &&
                      (*c)->scalar_type() == cos->scalar_type() && (*c)->dim() == 2 &&
                      (*c)->size(0) == rope_rows && (*c)->size(1) == d && (*c)->is_contiguous(),
                  "cos and sin must be contiguous float32 or ", qkv.scalar_type(),
                  " [positions, ", d, "] of one type");
      check_same_device(qkv, {&**c});
    }
  }
  at::Tensor q = at::empty({rows, heads, d}, qkv.options());
  if (qkv.is_meta() || rows == 0) return q;
  const c10::DeviceGuard guard(qkv.device());
  // the kernel reads rows, tables and weights in 16-byte pieces: any other view is copied
  auto whole = [](const at::Tensor& t) {
    return aligned16(t.data_ptr()) ? t : t.clone(at::MemoryFormat::Contiguous);
  };
  at::Tensor x = qkv;
  if (x.stride(1) != 1 || step(x, 0) % 8 || (rows > 1 && x.stride(0) < x.size(1)) ||
      !aligned16(x.data_ptr()))
    x = whole(x.contiguous());
  std::array<at::Tensor, 4> keep;
  const void* side[4] = {nullptr, nullptr, nullptr, nullptr};
  const OptTensor* from[4] = {&q_norm, &k_norm, &cos, &sin};
  for (int i = 0; i < 4; ++i) {
    if (!from[i]->has_value()) continue;
    keep[i] = whole(**from[i]);
    side[i] = keep[i].data_ptr();
  }
  check_status(mtl_paged_write(x.data_ptr(), std::max(step(x, 0), x.size(1)), rows, &pool, &tab,
                               ptr<int64_t>(positions),
                               seqs.has_value() ? ptr<int32_t>(*seqs) : nullptr, side[0], side[1],
                               side[2], side[3], rope_f32, rope_rows, (float)eps, (int32_t)heads,
                               type, q.data_ptr(), stream_of(qkv)),
               "mtl_paged_write");
  return q;
}

mtl_page_state state_of(const at::Tensor& table, const OptTensor& lens, const at::Tensor& refs,
                        int64_t page_size) {
  const mtl_page_table t = table_of(table);
  check_int32(refs, 1, "refs");
  check_same_device(table, {&refs});
  TORCH_CHECK(t.seqs <= MTL_PAGES_MAX_SEQS, "at most ", MTL_PAGES_MAX_SEQS, " sequences, got ",
              t.seqs);
  TORCH_CHECK(t.width <= MTL_PAGES_MAX_WIDTH, "at most ", MTL_PAGES_MAX_WIDTH,
              " pages a sequence, got ", t.width);
  check_page_size(page_size);
  if (lens.has_value()) {
    check_int32(*lens, 1, "lens");
    check_same_device(table, {&*lens});
    TORCH_CHECK(lens->size(0) == t.seqs, "lens must be int32 [", t.seqs, "]");
  }
  mtl_page_state st{};
  st.table = const_cast<int32_t*>(t.table);
  st.ld = t.ld;
  st.width = t.width;
  st.seqs = t.seqs;
  st.lens = lens.has_value() ? ptr<int32_t>(*lens) : nullptr;
  st.refs = ptr<int32_t>(refs);
  st.pages = refs.size(0);
  st.page_size = (int32_t)page_size;
  return st;
}

int64_t check_call(const at::Tensor& a, const at::Tensor& b, const at::Tensor& table,
                   const char* na, const char* nb) {
  check_int32(a, 1, na);
  check_int32(b, 1, nb);
  check_same_device(table, {&a, &b});
  TORCH_CHECK(a.size(0) == b.size(0), na, " and ", nb, " must have the same length");
  TORCH_CHECK(a.size(0) <= MTL_PAGES_MAX_CALL, "at most ", MTL_PAGES_MAX_CALL,
              " sequences a call, got ", a.size(0));
  return a.size(0);
}

// How whole pages lie in a pool [layers,] pages, kv_heads, page_size, head_dim.
struct PageBlocks {
  int64_t layers, layer_bytes, page_stride, page_bytes, pages;
};

PageBlocks blocks_of(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.dim() == 4 || t.dim() == 5, name,
              " must be [pages, kv_heads, page_size, head_dim], with or without leading layers");
  TORCH_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf ||
                  t.scalar_type() == at::kFloat8_e4m3fn,
              name, " must be bfloat16, float16 or float8_e4m3fn, got ", t.scalar_type());
  check_apart(t, name);
  const int64_t e = t.element_size(), p = t.dim() - 4;
  // kv_heads, page_size and head_dim have to fill one block, in any order
  std::array<std::pair<int64_t, int64_t>, 3> dims;
  for (int i = 0; i < 3; ++i) dims[i] = {t.stride(p + 1 + i), t.size(p + 1 + i)};
  std::sort(dims.begin(), dims.end());
  int64_t block = 1;
  bool dense = true;
  for (const auto& [stride, size] : dims) {
    dense = dense && (size == 1 || stride == block);
    block *= size;
  }
  PageBlocks b{p ? t.size(0) : 1, p ? step(t, 0) * e : 0,
               t.size(p) > 1 ? t.stride(p) * e : block * e, block * e, t.size(p)};
  TORCH_CHECK(dense && b.page_stride >= b.page_bytes && b.page_bytes % 16 == 0 &&
                  b.page_stride % 16 == 0 && b.layer_bytes % 16 == 0 &&
                  (t.is_meta() || aligned16(t.data_ptr())),
              name, ": a page must be one block of memory, in multiples of 16 bytes");
  return b;
}

void check_pools(const at::Tensor& k, const at::Tensor& v, const PageBlocks& kb) {
  TORCH_CHECK(k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type(),
              "k_pages and v_pages must have the same shape and type");
  TORCH_CHECK(kb.layers <= 65535, "at most 65535 layers, got ", kb.layers);
  check_same_device(k, {&v});
  check_pools_apart(k, v, true);
}

void copy_blocks(const at::Tensor& k, const at::Tensor& v, const PageBlocks& kb,
                 const PageBlocks& vb, const int32_t* src, const int32_t* dst, int64_t n,
                 const int32_t* count) {
  check_status(mtl_pages_copy(k.data_ptr(), v.data_ptr(), kb.layers, kb.layer_bytes,
                              vb.layer_bytes, kb.page_stride, vb.page_stride, kb.page_bytes,
                              kb.pages, src, dst, n, count, stream_of(k)),
               "mtl_pages_copy");
}

at::Tensor pages_extend(at::Tensor& table, at::Tensor& lens, at::Tensor& refs,
                        const at::Tensor& seqs, const at::Tensor& counts, at::Tensor& k_pages,
                        at::Tensor& v_pages) {
  const PageBlocks kb = blocks_of(k_pages, "k_pages"), vb = blocks_of(v_pages, "v_pages");
  check_pools(k_pages, v_pages, kb);
  const mtl_page_state st = state_of(table, lens, refs, k_pages.size(-2));
  check_same_device(table, {&k_pages});
  TORCH_CHECK(st.pages == kb.pages, "refs counts ", st.pages, " pages, the pool has ", kb.pages);
  const int64_t n = check_call(seqs, counts, table, "seqs", "counts");
  at::Tensor status = at::empty({1}, table.options());
  if (table.is_meta()) return status;
  const c10::DeviceGuard guard(table.device());
  const int64_t bytes = (mtl_pages_workspace_bytes(n, st.pages) + 15) / 16 * 16;
  const Workspace ws(table, bytes + 4 * (2 * n + 1));
  int32_t* copies = reinterpret_cast<int32_t*>(static_cast<char*>(ws.get()) + bytes);
  int32_t* src = copies + 1;
  int32_t* dst = src + n;
  check_status(mtl_pages_extend(&st, ptr<int32_t>(seqs), ptr<int32_t>(counts), n, src, dst,
                                copies, ptr<int32_t>(status), ws.get(), bytes, stream_of(table)),
               "mtl_pages_extend");
  copy_blocks(k_pages, v_pages, kb, vb, src, dst, n, copies);
  return status;
}

at::Tensor pages_fork(at::Tensor& table, at::Tensor& lens, at::Tensor& refs,
                      const at::Tensor& parents, const at::Tensor& children, int64_t page_size) {
  const mtl_page_state st = state_of(table, lens, refs, page_size);
  const int64_t n = check_call(parents, children, table, "parents", "children");
  at::Tensor status = at::empty({1}, table.options());
  if (table.is_meta()) return status;
  const c10::DeviceGuard guard(table.device());
  const Workspace ws(table, mtl_pages_workspace_bytes(n, st.pages));
  check_status(mtl_pages_fork(&st, ptr<int32_t>(parents), ptr<int32_t>(children), n,
                              ptr<int32_t>(status), ws.get(), ws.bytes, stream_of(table)),
               "mtl_pages_fork");
  return status;
}

at::Tensor pages_truncate(at::Tensor& table, at::Tensor& lens, at::Tensor& refs,
                          const at::Tensor& seqs, const at::Tensor& new_lens, int64_t page_size) {
  const mtl_page_state st = state_of(table, lens, refs, page_size);
  const int64_t n = check_call(seqs, new_lens, table, "seqs", "new_lens");
  at::Tensor status = at::empty({1}, table.options());
  if (table.is_meta()) return status;
  const c10::DeviceGuard guard(table.device());
  const Workspace ws(table, mtl_pages_workspace_bytes(n, st.pages));
  check_status(mtl_pages_truncate(&st, ptr<int32_t>(seqs), ptr<int32_t>(new_lens), n,
                                  ptr<int32_t>(status), ws.get(), ws.bytes, stream_of(table)),
               "mtl_pages_truncate");
  return status;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> pages_compact(const at::Tensor& table,
                                                             const at::Tensor& refs,
                                                             at::Tensor& k_pages,
                                                             at::Tensor& v_pages) {
  const PageBlocks kb = blocks_of(k_pages, "k_pages"), vb = blocks_of(v_pages, "v_pages");
  check_pools(k_pages, v_pages, kb);
  mtl_page_state st = state_of(table, c10::nullopt, refs, k_pages.size(-2));
  check_same_device(table, {&k_pages});
  TORCH_CHECK(st.pages == kb.pages, "refs counts ", st.pages, " pages, the pool has ", kb.pages);
  at::Tensor new_table = at::empty({table.size(0), table.size(1)}, table.options());
  at::Tensor new_refs = at::empty({refs.size(0)}, refs.options());
  at::Tensor live = at::empty({1}, table.options());
  if (table.is_meta()) return {new_table, new_refs, live};
  const c10::DeviceGuard guard(table.device());
  const int64_t half = st.pages / 2;
  const int64_t bytes = (mtl_pages_workspace_bytes(0, st.pages) + 15) / 16 * 16;
  const Workspace ws(table, bytes + 4 * (2 * half + 1));
  int32_t* moves = reinterpret_cast<int32_t*>(static_cast<char*>(ws.get()) + bytes);
  int32_t* src = moves + 1;
  check_status(mtl_pages_compact(&st, ptr<int32_t>(new_table), table.size(1),
                                 ptr<int32_t>(new_refs), ptr<int32_t>(live), moves, src,
                                 src + half, ws.get(), bytes, stream_of(table)),
               "mtl_pages_compact");
  copy_blocks(k_pages, v_pages, kb, vb, src, src + half, half, moves);
  return {new_table, new_refs, live};
}

void pages_copy(at::Tensor& k_pages, at::Tensor& v_pages, const at::Tensor& src,
                const at::Tensor& dst) {
  const PageBlocks kb = blocks_of(k_pages, "k_pages"), vb = blocks_of(v_pages, "v_pages");
  check_pools(k_pages, v_pages, kb);
  check_int32(src, 1, "src");
  check_int32(dst, 1, "dst");
  check_same_device(k_pages, {&src, &dst});
  TORCH_CHECK(src.size(0) == dst.size(0), "src and dst must have the same length");
  if (k_pages.is_meta()) return;
  const c10::DeviceGuard guard(k_pages.device());
  copy_blocks(k_pages, v_pages, kb, vb, ptr<int32_t>(src), ptr<int32_t>(dst), src.size(0),
              nullptr);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(mtl, m) {
  m.def("paged_attention(Tensor q, Tensor k_pages, Tensor v_pages, Tensor table, Tensor lens, "
        "float scale, Tensor? k_scale=None, Tensor? v_scale=None) -> Tensor");
  m.def("paged_attention_lse(Tensor q, Tensor k_pages, Tensor v_pages, Tensor table, "
        "Tensor lens, float scale, Tensor? k_scale=None, Tensor? v_scale=None) "
        "-> (Tensor, Tensor)");
  m.def("paged_attention_shared(Tensor q, Tensor k_pages, Tensor v_pages, Tensor table, "
        "Tensor lens, Tensor groups, Tensor shared, float scale, Tensor? k_scale=None, "
        "Tensor? v_scale=None) -> Tensor");
  m.def("paged_attention_shared_lse(Tensor q, Tensor k_pages, Tensor v_pages, Tensor table, "
        "Tensor lens, Tensor groups, Tensor shared, float scale, Tensor? k_scale=None, "
        "Tensor? v_scale=None) -> (Tensor, Tensor)");
  m.def("paged_write(Tensor qkv, Tensor(a!) k_pages, Tensor(b!) v_pages, Tensor table, "
        "Tensor positions, Tensor? seqs=None, Tensor? q_norm=None, Tensor? k_norm=None, "
        "Tensor? cos=None, Tensor? sin=None, float eps=1e-6, Tensor? k_scale=None, "
        "Tensor? v_scale=None) -> Tensor");
  m.def("pages_extend(Tensor(a!) table, Tensor(b!) lens, Tensor(c!) refs, Tensor seqs, "
        "Tensor counts, Tensor(d!) k_pages, Tensor(e!) v_pages) -> Tensor");
  m.def("pages_fork(Tensor(a!) table, Tensor(b!) lens, Tensor(c!) refs, Tensor parents, "
        "Tensor children, int page_size) -> Tensor");
  m.def("pages_truncate(Tensor(a!) table, Tensor(b!) lens, Tensor(c!) refs, Tensor seqs, "
        "Tensor new_lens, int page_size) -> Tensor");
  m.def("pages_compact(Tensor table, Tensor refs, Tensor(a!) k_pages, Tensor(b!) v_pages) "
        "-> (Tensor, Tensor, Tensor)");
  m.def("pages_copy(Tensor(a!) k_pages, Tensor(b!) v_pages, Tensor src, Tensor dst) -> ()");
}

#define MTL_PAGED_IMPLS(m)                   \
  m.impl("paged_attention", &paged_attention); \
  m.impl("paged_attention_lse", &paged_attention_lse); \
  m.impl("paged_attention_shared", &paged_attention_shared); \
  m.impl("paged_attention_shared_lse", &paged_attention_shared_lse); \
  m.impl("paged_write", &paged_write);         \
  m.impl("pages_extend", &pages_extend);       \
  m.impl("pages_fork", &pages_fork);           \
  m.impl("pages_truncate", &pages_truncate);   \
  m.impl("pages_compact", &pages_compact);     \
  m.impl("pages_copy", &pages_copy)

TORCH_LIBRARY_IMPL(mtl, CUDA, m) { MTL_PAGED_IMPLS(m); }

TORCH_LIBRARY_IMPL(mtl, Meta, m) { MTL_PAGED_IMPLS(m); }
