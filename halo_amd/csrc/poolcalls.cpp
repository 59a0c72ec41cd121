// Host side of the block-pool operators' ordinary calls (host code): the
// arguments are checked, the outputs allocated and the library called in one
// step, at a third of what the same costs through Python attributes and
// ctypes (a call of halo_amd.commit_path: 12 us -> 5 us of host time).
//
// Every function returns None for a call that it does not take: tensors on
// another device than the current one, forms that need a copy, anything that
// the checks refuse.  The Python functions of the same names then run the call
// themselves, or say what is wrong with it.  A status below 0 of the
// library is returned as it is.
#include <c10/hip/HIPStream.h>
#include <torch/extension.h>

#include <cmath>
#include <optional>
#include <type_traits>
#include <vector>

#include "../../include/halo_hip.h"

namespace py = pybind11;
using at::Tensor;

namespace {

constexpr int kMaxNodes = 512, kMaxPath = 64, kPlanRequests = 4096;

struct Entries {
  decltype(&halo_update_block_tables) update;
  decltype(&halo_append_rows) append;
  decltype(&halo_tree_layout) layout;
  decltype(&halo_tree_workspace_size) workspace;
  decltype(&halo_tree_attn) attn;
  decltype(&halo_commit_path) commit;
  decltype(&halo_chunk_workspace_size) chunk_workspace;
  decltype(&halo_chunk_attn) chunk;
  decltype(&halo_verify_tree) verify;
  decltype(&halo_rotate_rows) rotate;
  decltype(&halo_fork_workspace_size) fork_workspace;
  decltype(&halo_fork_blocks) fork;
  decltype(&halo_compact_workspace_size) compact_workspace;
  decltype(&halo_compact_blocks) compact;
} lib;

// The library's entries, in the order of halo_amd/block_pool.py's list.
void bind(const std::vector<uintptr_t>& at) {
  size_t i = 0;
  auto next = [&](auto& entry) { entry = reinterpret_cast<std::decay_t<decltype(entry)>>(at.at(i++)); };
  next(lib.update);
  next(lib.append);
  next(lib.layout);
  next(lib.workspace);
  next(lib.attn);
  next(lib.commit);
  next(lib.chunk_workspace);
  next(lib.chunk);
  next(lib.verify);
  next(lib.rotate);
  next(lib.fork_workspace);
  next(lib.fork);
  next(lib.compact_workspace);
  next(lib.compact);
}

bool on(const Tensor& t, const at::Device& d) { return t.device() == d; }
// the current device's index, or -1 if `t` is not there
int here(const Tensor& t) {
  if (!t.is_cuda()) return -1;
  const int d = t.device().index();
  return d == c10::hip::current_device() ? d : -1;
}
void* stream_of(int device) { return c10::hip::getCurrentHIPStream(device).stream(); }

bool ints(const Tensor& t, int64_t n, const at::Device& d, at::ScalarType type = at::kInt) {
  return t.dim() == 1 && t.size(0) == n && t.scalar_type() == type && on(t, d) && t.is_contiguous();
}
bool table_ok(const Tensor& t, int64_t B, const at::Device& d) {
  return t.scalar_type() == at::kInt && on(t, d) && t.dim() == 2 && t.size(0) == B && t.stride(1) == 1 && t.size(1) >= 1 &&
         (B == 1 || t.stride(0) >= t.size(1));
}
int64_t table_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

bool apart(const Tensor& a, const Tensor& b) {  // whether the memory they span is
  auto span = [](const Tensor& t, uintptr_t& lo, uintptr_t& hi) {
    int64_t n = t.numel() != 0;
    if (n)
      for (int64_t i = 0; i < t.dim(); ++i) n += (t.size(i) - 1) * t.stride(i);
    lo = reinterpret_cast<uintptr_t>(t.data_ptr());
    hi = lo + n * t.element_size();
  };
  uintptr_t alo, ahi, blo, bhi;
  span(a, alo, ahi);
  span(b, blo, bhi);
  return ahi <= blo || bhi <= alo;
}

int dtype_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return HALO_F32;
    case at::kBFloat16: return HALO_BF16;
    case at::kHalf: return HALO_F16;
    default: return -1;
  }
}

bool pool_of(const Tensor& k, const Tensor& v, bool written, halo_block_pool* p) {
  const int64_t n = k.dim();
  const int dt = dtype_of(k);
  if (dt < 0 || v.scalar_type() != k.scalar_type() || (n != 4 && n != 5) || v.sizes() != k.sizes() ||
      v.strides() != k.strides() || v.device() != k.device() || k.stride(n - 1) != 1 || k.numel() == 0)
    return false;
  for (int64_t i = 0; i < n; ++i)
    if (k.size(i) > 0x7fffffff || (written && k.size(i) > 1 && k.stride(i) == 0)) return false;
  if (written && k.data_ptr() == v.data_ptr()) return false;
  p->k = k.data_ptr();
  p->v = v.data_ptr();
  p->stride_l = n == 5 ? k.stride(0) : 0;
  p->stride_b = k.stride(n - 4);
  p->stride_h = k.stride(n - 3);
  p->stride_r = k.stride(n - 2);
  p->layers = n == 5 ? (int32_t)k.size(0) : 1;
  p->blocks = (int32_t)k.size(n - 4);
  p->H_kv = (int32_t)k.size(n - 3);
  p->block_size = (int32_t)k.size(n - 2);
  p->D = (int32_t)k.size(n - 1);
  p->dtype = dt;
  return true;
}

Tensor empty(at::IntArrayRef size, at::ScalarType type, const at::Device& d) {
  return at::empty(size, at::TensorOptions().dtype(type).device(d));
}

py::object update_block_tables(const Tensor& table, const Tensor& n_blocks, const Tensor& free_blocks,
                               const Tensor& n_free, const Tensor& lengths, const Tensor& first, int64_t block_size,
                               int64_t max_rows) {
  const int dev = here(table);
  const at::Device d = table.device();
  const int64_t B = lengths.dim() == 1 ? lengths.size(0) : 0;
  if (dev < 0 || B < 1 || B > 0x7ffffff || !table_ok(table, B, d) || !ints(n_blocks, B, d) || !ints(lengths, B, d) ||
      !ints(first, B, d) || !ints(n_free, 1, d) || free_blocks.dim() != 1 ||
      !ints(free_blocks, free_blocks.size(0), d) || block_size < 1 || block_size > 0x7fffffff || max_rows < 0 ||
      max_rows > 0x7fffffff || free_blocks.size(0) > 0x7fffffff || table.size(1) > 0x7fffffff)
    return py::none();
  for (const Tensor* t : {&n_blocks, &n_free, &free_blocks, &table})
    if (!apart(*t, lengths) || !apart(*t, first)) return py::none();
  Tensor cu = empty({B + 1}, at::kInt, d), slots = empty({max_rows}, at::kLong, d), ok = empty({B}, at::kBool, d);
  const int rc = lib.update(table.data_ptr<int32_t>(), table_stride(table), n_blocks.data_ptr<int32_t>(), (int)B,
                            (int)table.size(1), free_blocks.data_ptr<int32_t>(), (int)free_blocks.size(0),
                            n_free.data_ptr<int32_t>(), lengths.data_ptr<int32_t>(), first.data_ptr<int32_t>(),
                            (int)block_size, (int)max_rows, cu.data_ptr<int32_t>(), slots.data_ptr<int64_t>(),
                            reinterpret_cast<uint8_t*>(ok.data_ptr<bool>()), stream_of(dev));
  if (rc != HALO_OK) return py::int_(rc);
  return py::make_tuple(cu, slots, ok);
}

py::object append_rows(const Tensor& k, const Tensor& v, const Tensor& slots, const Tensor& k_pool,
                       const Tensor& v_pool) {
  halo_block_pool pool;
  const int dev = here(k_pool);
  if (dev < 0 || slots.dim() != 1 || !pool_of(k_pool, v_pool, true, &pool)) return py::none();
  const at::Device d = k_pool.device();
  const int64_t n = k_pool.dim() - 1, N = slots.size(0);
  if (!ints(slots, N, d, at::kLong) || N > 0x7fffffff) return py::none();
  for (const Tensor* t : {&k, &v})
    if (t->dim() != n || !on(*t, d) || t->scalar_type() != k_pool.scalar_type() || t->size(n - 3) != N ||
        t->size(n - 2) != pool.H_kv || t->size(n - 1) != pool.D || t->stride(n - 1) != 1 ||
        (n == 4 && t->size(0) != pool.layers) || !apart(*t, k_pool) || !apart(*t, v_pool))
      return py::none();
  const int rc = lib.append(&pool, k.data_ptr(), n == 4 ? k.stride(0) : 0, k.stride(n - 3), k.stride(n - 2),
                            v.data_ptr(), n == 4 ? v.stride(0) : 0, v.stride(n - 3), v.stride(n - 2),
                            slots.data_ptr<int64_t>(), (int)N, stream_of(dev));
  return py::int_(rc);
}

py::object tree_layout(const Tensor& parents, const Tensor& cu, int64_t max_nodes) {
  const int dev = here(parents);
  const at::Device d = parents.device();
  if (dev < 0 || parents.dim() != 1 || cu.dim() != 1 || cu.size(0) < 2 || max_nodes < 1 || max_nodes > kMaxNodes)
    return py::none();
  const int64_t N = parents.size(0), B = cu.size(0) - 1, words = (max_nodes + 63) / 64;
  if (N < 1 || N > 0x7fffffff || B > 0x7ffffff || !ints(parents, N, d) || !ints(cu, B + 1, d)) return py::none();
  Tensor mask = empty({N, words}, at::kLong, d), depth = empty({N}, at::kInt, d);
  const int rc = lib.layout(parents.data_ptr<int32_t>(), cu.data_ptr<int32_t>(), (int)B, (int)N, (int)max_nodes,
                            mask.data_ptr<int64_t>(), words, depth.data_ptr<int32_t>(), stream_of(dev));
  if (rc != HALO_OK) return py::int_(rc);
  return py::make_tuple(mask, depth);
}

// Trees, or (chunk) causal chunks of any number of rows.
py::object attend(const Tensor& q, const Tensor& k_pool, const Tensor& v_pool, const Tensor& table, const Tensor& lengths,
                  const Tensor& cu, int64_t max_nodes, const std::optional<Tensor>& mask, bool chunk,
                  std::optional<double> scale, std::optional<Tensor> out, std::optional<Tensor> lse, bool return_lse) {
  halo_block_pool pool;
  const int dev = here(q);
  if (dev < 0 || q.dim() != 3 || k_pool.dim() != 4 || !pool_of(k_pool, v_pool, false, &pool)) return py::none();
  const at::Device d = q.device();
  const int64_t N = q.size(0), H = q.size(1), D = q.size(2), B = lengths.dim() == 1 ? lengths.size(0) : 0;
  if (!on(k_pool, d) || k_pool.scalar_type() != q.scalar_type() || pool.D != D || (D != 64 && D != 128) || H < 1 ||
      H > 0x7fffffff || H % pool.H_kv != 0 || N < 1 || N > 0x7fffffff || max_nodes < 1 || (!chunk && max_nodes > kMaxNodes) || B < 1 ||
      B > 0x7ffffff || !table_ok(table, B, d) || table.size(1) > 0x7fffffff || !ints(lengths, B, d) ||
      !ints(cu, B + 1, d))
    return py::none();
  if (max_nodes > N) max_nodes = chunk ? N : max_nodes;  // no request has more rows than there are
  // the plan of chunks holds kPlanRequests; rows of more are nodes of trees without masks
  if (B > kPlanRequests && max_nodes <= kMaxNodes) chunk = false;
  const int64_t per = 16 / q.element_size();
  if (q.stride(2) != 1 || q.stride(0) % per || q.stride(1) % per || reinterpret_cast<uintptr_t>(q.data_ptr()) % 16)
    return py::none();
  int64_t words = 0;
  if (mask) {
    const Tensor& m = *mask;
    if (m.scalar_type() != at::kLong || !on(m, d) || m.dim() != 2 || m.size(0) != N || m.size(1) * 64 < max_nodes ||
        !m.is_contiguous())
      return py::none();
    words = m.size(1);
  }
  const double s = scale ? *scale : 1.0 / std::sqrt((double)D);
  if (!(s > 0 && s < INFINITY)) return py::none();
  if (out) {
    const Tensor& o = *out;
    if (o.sizes() != q.sizes() || !on(o, d) || o.scalar_type() != q.scalar_type() || o.stride(2) != 1 || o.stride(0) % 4 ||
        o.stride(1) % 4 || reinterpret_cast<uintptr_t>(o.data_ptr()) % (4 * o.element_size()) || !apart(o, q) ||
        !apart(o, k_pool) || !apart(o, v_pool) || (N > 1 && o.stride(0) == 0) || (H > 1 && o.stride(1) == 0))
      return py::none();
  } else {
    out = empty({N, H, D}, q.scalar_type(), d);
  }
  if (lse) {
    const Tensor& z = *lse;
    if (z.dim() != 2 || z.size(0) != N || z.size(1) != H || z.scalar_type() != at::kFloat || !on(z, d) ||
        !z.is_contiguous() || !apart(z, q) || !apart(z, k_pool) || !apart(z, v_pool) || !apart(z, *out))
      return py::none();
  } else if (return_lse) {
    lse = empty({N, H}, at::kFloat, d);
  }
  const int64_t rows = table.size(1) * pool.block_size;
  const size_t bytes =
      chunk ? lib.chunk_workspace(pool.dtype, (int)B, (int)N, (int)H, pool.H_kv, (int)D, rows, (int)max_nodes)
            : lib.workspace(pool.dtype, (int)B, (int)H, pool.H_kv, (int)D, rows, (int)max_nodes);
  Tensor ws;
  if (bytes) ws = empty({(int64_t)bytes}, at::kByte, d);
  void* wp = bytes ? ws.data_ptr() : nullptr;
  float* lp = lse ? lse->data_ptr<float>() : nullptr;
  const int rc =
      chunk ? lib.chunk(&pool, q.data_ptr(), q.stride(0), q.stride(1), (int)N, (int)H, table.data_ptr<int32_t>(),
                        table_stride(table), (int)B, (int)table.size(1), lengths.data_ptr<int32_t>(), cu.data_ptr<int32_t>(),
                        (int)max_nodes, (float)s, out->data_ptr(), out->stride(0), out->stride(1), pool.dtype, lp, wp, bytes,
                        stream_of(dev))
            : lib.attn(&pool, q.data_ptr(), q.stride(0), q.stride(1), (int)N, (int)H, table.data_ptr<int32_t>(),
                       table_stride(table), (int)B, (int)table.size(1), lengths.data_ptr<int32_t>(), cu.data_ptr<int32_t>(),
                       (int)max_nodes, mask ? mask->data_ptr<int64_t>() : nullptr, words, (float)s, out->data_ptr(),
                       out->stride(0), out->stride(1), pool.dtype, lp, wp, bytes, stream_of(dev));
  if (rc != HALO_OK) return py::int_(rc);
  if (return_lse) return py::make_tuple(*out, *lse);
  return py::cast(*out);
}

py::object tree_attention(const Tensor& q, const Tensor& k_pool, const Tensor& v_pool, const Tensor& table,
                          const Tensor& lengths, const Tensor& cu, int64_t max_nodes, const std::optional<Tensor>& mask,
                          std::optional<double> scale, std::optional<Tensor> out, std::optional<Tensor> lse,
                          bool return_lse) {
  return attend(q, k_pool, v_pool, table, lengths, cu, max_nodes, mask, false, scale, out, lse, return_lse);
}

py::object chunk_attention(const Tensor& q, const Tensor& k_pool, const Tensor& v_pool, const Tensor& table,
                           const Tensor& lengths, const Tensor& cu, int64_t max_rows, std::optional<double> scale,
                           std::optional<Tensor> out, std::optional<Tensor> lse, bool return_lse) {
  return attend(q, k_pool, v_pool, table, lengths, cu, max_rows, std::nullopt, true, scale, out, lse, return_lse);
}

py::object commit_path(const Tensor& k_pool, const Tensor& v_pool, const Tensor& table, const Tensor& lengths,
                       const Tensor& path, const Tensor& n_path, std::optional<Tensor> out) {
  halo_block_pool pool;
  const int dev = here(k_pool);
  if (dev < 0 || lengths.dim() != 1 || path.dim() != 2 || !pool_of(k_pool, v_pool, true, &pool)) return py::none();
  const at::Device d = k_pool.device();
  const int64_t B = lengths.size(0), n = path.size(1);
  if (B < 1 || B > 0x7ffffff || n < 1 || n > kMaxPath || !table_ok(table, B, d) || table.size(1) > 0x7fffffff ||
      !ints(lengths, B, d) || path.scalar_type() != at::kInt || !on(path, d) || path.size(0) != B ||
      !path.is_contiguous() || !ints(n_path, B, d))
    return py::none();
  if (out) {
    if (!ints(*out, B, d)) return py::none();
    for (const Tensor* t : {&lengths, &path, &n_path, &table})
      if (!apart(*out, *t)) return py::none();
  } else {
    out = empty({B}, at::kInt, d);
  }
  const int rc = lib.commit(&pool, table.data_ptr<int32_t>(), table_stride(table), (int)B, (int)table.size(1),
                            lengths.data_ptr<int32_t>(), path.data_ptr<int32_t>(), n, (int)n,
                            n_path.data_ptr<int32_t>(), out->data_ptr<int32_t>(), stream_of(dev));
  if (rc != HALO_OK) return py::int_(rc);
  return py::cast(*out);
}

bool floats(const Tensor& t, int64_t n, const at::Device& d) { return ints(t, n, d, at::kFloat); }

py::object verify_tree(const Tensor& tokens, const Tensor& parents, const Tensor& cu, const Tensor& probs,
                       const Tensor& accept, const Tensor& sample, int64_t max_nodes, const std::optional<Tensor>& draft,
                       bool replacement, int64_t max_path) {
  const int dev = here(probs), dt = dtype_of(probs);
  const at::Device d = probs.device();
  if (dev < 0 || dt < 0 || probs.dim() != 2 || tokens.dim() != 1 || cu.dim() != 1 || cu.size(0) < 2) return py::none();
  const int64_t N = tokens.size(0), B = cu.size(0) - 1, V = probs.size(1);
  if (N > 0x7fffffff || B > 65535 || V < 1 || V > (1 << 24) || max_nodes < 1 || max_nodes > kMaxNodes || max_path < 1 ||
      max_path > kMaxPath || !ints(tokens, N, d, at::kLong) || !ints(parents, N, d) || !ints(cu, B + 1, d) ||
      !floats(accept, N, d) || !floats(sample, B, d) || probs.size(0) != N || (V > 1 && probs.stride(1) != 1))
    return py::none();
  if (draft && (draft->sizes() != probs.sizes() || draft->scalar_type() != probs.scalar_type() || !on(*draft, d) ||
                (V > 1 && draft->stride(1) != 1)))
    return py::none();
  Tensor path = empty({B, max_path}, at::kInt, d), n_path = empty({B}, at::kInt, d), token = empty({B}, at::kLong, d);
  const int rc = lib.verify(tokens.data_ptr<int64_t>(), parents.data_ptr<int32_t>(), cu.data_ptr<int32_t>(), (int)B, (int)N,
                            (int)max_nodes, (int)V, dt, probs.data_ptr(), probs.stride(0), draft ? draft->data_ptr() : nullptr,
                            draft ? draft->stride(0) : 0, replacement, accept.data_ptr<float>(), sample.data_ptr<float>(),
                            (int)max_path, path.data_ptr<int32_t>(), n_path.data_ptr<int32_t>(), token.data_ptr<int64_t>(),
                            stream_of(dev));
  if (rc != HALO_OK) return py::int_(rc);
  return py::make_tuple(path, n_path, token);
}

// Whether all 16-byte pieces of (N, H, D) rows lie on their bounds.
bool rows_aligned(const Tensor& t) {
  const int64_t per = 16 / t.element_size();
  return t.stride(2) == 1 && t.stride(0) % per == 0 && t.stride(1) % per == 0 &&
         reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
}

py::object rotate_rows(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& positions, const Tensor& cos,
                       const Tensor& sin, const Tensor& slots, const Tensor& k_pool, const Tensor& v_pool,
                       const std::optional<Tensor>& q_norm, const std::optional<Tensor>& k_norm, double eps, bool interleaved) {
  halo_block_pool pool;
  const int dev = here(k_pool);
  if (dev < 0 || k_pool.dim() != 4 || q.dim() != 3 || slots.dim() != 1 || !pool_of(k_pool, v_pool, true, &pool))
    return py::none();
  const at::Device d = k_pool.device();
  const int64_t N = slots.size(0), H = q.size(1), D = pool.D;
  if ((D != 64 && D != 128) || N > 0x7fffffff || H < 1 || H > 0x7fffffff || !ints(slots, N, d, at::kLong) || positions.dim() != 1 ||
      positions.size(0) != N || !on(positions, d) || !positions.is_contiguous() ||
      (positions.scalar_type() != at::kInt && positions.scalar_type() != at::kLong))
    return py::none();
  for (const Tensor* t : {&q, &k, &v})
    if (t->dim() != 3 || t->scalar_type() != k_pool.scalar_type() || !on(*t, d) || t->size(0) != N || t->size(2) != D ||
        (t != &q && t->size(1) != pool.H_kv) || !rows_aligned(*t) || !apart(*t, k_pool) || !apart(*t, v_pool))
      return py::none();
  if (cos.dim() != 2 || sin.sizes() != cos.sizes()) return py::none();
  const int64_t R = 2 * cos.size(1);
  for (const Tensor* t : {&cos, &sin})
    if (t->scalar_type() != at::kFloat || !on(*t, d) || !t->is_contiguous() || reinterpret_cast<uintptr_t>(t->data_ptr()) % 16)
      return py::none();
  if (cos.size(0) < 1 || R < 16 || R > D || R % 16 || !(eps >= 0 && eps < INFINITY)) return py::none();
  for (const auto* w : {&q_norm, &k_norm})
    if (*w && ((*w)->dim() != 1 || (*w)->size(0) != D || !on(**w, d) || !(*w)->is_contiguous() ||
               ((*w)->scalar_type() != at::kFloat && (*w)->scalar_type() != k_pool.scalar_type())))
      return py::none();
  Tensor out = empty({N, H, D}, q.scalar_type(), d);
  auto f32 = [](const std::optional<Tensor>& w) { return w && w->scalar_type() == at::kFloat; };
  const int rc = lib.rotate(&pool, q.data_ptr(), q.stride(0), q.stride(1), (int)H, k.data_ptr(), k.stride(0), k.stride(1),
                            v.data_ptr(), v.stride(0), v.stride(1), out.data_ptr(), out.stride(0), out.stride(1), (int)N,
                            positions.data_ptr(), positions.scalar_type() == at::kLong, cos.data_ptr<float>(),
                            sin.data_ptr<float>(), R / 2, cos.size(0), (int)R, interleaved, q_norm ? q_norm->data_ptr() : nullptr,
                            f32(q_norm), k_norm ? k_norm->data_ptr() : nullptr, f32(k_norm), (float)eps,
                            slots.data_ptr<int64_t>(), stream_of(dev));
  if (rc != HALO_OK) return py::int_(rc);
  return py::cast(out);
}

// The tables, free list and counts that a call changes: their forms, and that they share no memory.
bool owners_ok(const Tensor& table, const Tensor& n_blocks, const Tensor& free_blocks, const Tensor& n_free, const Tensor& shared,
               const Tensor& k_pool, const Tensor& v_pool, int64_t B, const halo_block_pool& pool) {
  const at::Device d = k_pool.device();
  if (B < 1 || B > 0x7ffffff || !table_ok(table, B, d) || table.size(1) > 0x7fffffff || !ints(n_blocks, B, d) ||
      free_blocks.dim() != 1 || free_blocks.size(0) > 0x7fffffff || !ints(free_blocks, free_blocks.size(0), d) ||
      !ints(n_free, 1, d) || !ints(shared, pool.blocks, d))
    return false;
  const Tensor* all[] = {&table, &n_blocks, &free_blocks, &n_free, &shared, &k_pool, &v_pool};
  for (int i = 0; i < 7; ++i)
    for (int j = i + 1; j < 7; ++j)
      if (!apart(*all[i], *all[j])) return false;
  return true;
}

py::object fork_blocks(const Tensor& table, const Tensor& n_blocks, const Tensor& free_blocks, const Tensor& n_free,
                       const Tensor& shared, const Tensor& lengths, const Tensor& source, const Tensor& k_pool,
                       const Tensor& v_pool) {
  halo_block_pool pool;
  const int dev = here(k_pool);
  if (dev < 0 || lengths.dim() != 1 || !pool_of(k_pool, v_pool, true, &pool)) return py::none();
  const at::Device d = k_pool.device();
  const int64_t B = lengths.size(0);
  if (B > 4096 || !owners_ok(table, n_blocks, free_blocks, n_free, shared, k_pool, v_pool, B, pool) || !ints(lengths, B, d) ||
      !ints(source, B, d))
    return py::none();
  for (const Tensor* t : {&table, &n_blocks, &free_blocks, &n_free, &shared, &k_pool, &v_pool})
    if (!apart(*t, lengths) || !apart(*t, source)) return py::none();
  Tensor lens = empty({B}, at::kInt, d), ok = empty({1}, at::kBool, d);
  const size_t bytes = lib.fork_workspace((int)B, (int)table.size(1), pool.blocks);
  Tensor ws = empty({(int64_t)bytes}, at::kByte, d);
  const int rc = lib.fork(&pool, table.data_ptr<int32_t>(), table_stride(table), n_blocks.data_ptr<int32_t>(), (int)B,
                          (int)table.size(1), free_blocks.data_ptr<int32_t>(), (int)free_blocks.size(0),
                          n_free.data_ptr<int32_t>(), shared.data_ptr<int32_t>(), lengths.data_ptr<int32_t>(),
                          source.data_ptr<int32_t>(), lens.data_ptr<int32_t>(), reinterpret_cast<uint8_t*>(ok.data_ptr<bool>()),
                          ws.data_ptr(), bytes, stream_of(dev));
  if (rc != HALO_OK) return py::int_(rc);
  return py::make_tuple(lens, ok);
}

py::object compact_blocks(const Tensor& table, const Tensor& n_blocks, const Tensor& free_blocks, const Tensor& n_free,
                          const Tensor& shared, const Tensor& k_pool, const Tensor& v_pool) {
  halo_block_pool pool;
  const int dev = here(k_pool);
  if (dev < 0 || n_blocks.dim() != 1 || !pool_of(k_pool, v_pool, true, &pool)) return py::none();
  const at::Device d = k_pool.device();
  const int64_t B = n_blocks.size(0);
  if (!owners_ok(table, n_blocks, free_blocks, n_free, shared, k_pool, v_pool, B, pool)) return py::none();
  Tensor new_id = empty({pool.blocks}, at::kInt, d), n_used = empty({1}, at::kInt, d);
  const size_t bytes = lib.compact_workspace(pool.blocks);
  Tensor ws = empty({(int64_t)bytes}, at::kByte, d);
  const int rc = lib.compact(&pool, table.data_ptr<int32_t>(), table_stride(table), n_blocks.data_ptr<int32_t>(), (int)B,
                             (int)table.size(1), free_blocks.data_ptr<int32_t>(), (int)free_blocks.size(0),
                             n_free.data_ptr<int32_t>(), shared.data_ptr<int32_t>(), new_id.data_ptr<int32_t>(),
                             n_used.data_ptr<int32_t>(), ws.data_ptr(), bytes, stream_of(dev));
  if (rc != HALO_OK) return py::int_(rc);
  return py::make_tuple(new_id, n_used);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("bind", &bind);
  m.def("update_block_tables", &update_block_tables);
  m.def("append_rows", &append_rows);
  m.def("tree_layout", &tree_layout);
  m.def("tree_attention", &tree_attention);
  m.def("commit_path", &commit_path);
  m.def("chunk_attention", &chunk_attention);
  m.def("verify_tree", &verify_tree);
  m.def("rotate_rows", &rotate_rows);
  m.def("fork_blocks", &fork_blocks);
  m.def("compact_blocks", &compact_blocks);
}
