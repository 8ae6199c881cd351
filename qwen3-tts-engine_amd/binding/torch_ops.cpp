// The 8-bit pool's and the tree attention's torch ops over the C ABI (include/q3attn.h).
//
// They check what the C entry points cannot see (types, shapes, devices, contiguous dims), allocate outputs and workspace
// through torch's caching allocator on the current stream of the tensors' device, launch there and return.  In C++ because a
// serving step makes a call per layer and the calls of a small batch are a few microseconds on the device: through Python (a
// custom op with its checks in Python and the C call through ctypes) a read of 77 tokens took 23.8 us on the host, of which
// the launch is 2.6.
#include <ATen/ATen.h>
#include <ATen/hip/EmptyTensor.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/VariableTypeUtils.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <tuple>

#include "../../include/q3attn.h"

namespace {

using at::Tensor;
using std::optional;

void* stream_of(const c10::Device& d) {
  return (void*)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(d.index()).stream();
}

// A contiguous tensor on d.  (Past the dispatcher: 0.7 us of a call's 10 a tensor.)
Tensor empty_on(const c10::Device& d, at::IntArrayRef shape, c10::ScalarType t) {
  return at::detail::empty_cuda(shape, t, d, std::nullopt);
}

void done(int rc, const char* what) { TORCH_CHECK(rc == Q3A_OK, what, " failed (", rc, "): ", q3a_last_error()); }

// A pool's two caches of type t with equal shapes and strides on device d.
void check_caches(const char* who, const c10::Device& d, const Tensor& k, const Tensor& v, c10::ScalarType t) {
  TORCH_CHECK(k.device() == d && v.device() == d, who, ": k_cache and v_cache must be on ", d);
  TORCH_CHECK(k.scalar_type() == t && v.scalar_type() == t, who, ": k_cache and v_cache must be ", t);
  TORCH_CHECK(k.dim() == 4 && k.sizes() == v.sizes() && k.strides() == v.strides() && k.stride(3) == 1, who,
              ": k_cache and v_cache must be [num_pages, page_size, kv_heads, head_dim] with equal strides and a contiguous head_dim");
  TORCH_CHECK(k.size(0) <= INT_MAX && k.size(1) <= INT_MAX && k.size(2) <= INT_MAX && k.size(3) <= INT_MAX, who,
              ": pool too large");
}

void check_fp8_pool(const char* who, const c10::Device& d, const Tensor& kc, const Tensor& vc, const Tensor& ks, const Tensor& vs) {
  check_caches(who, d, kc, vc, at::kFloat8_e4m3fn);
  TORCH_CHECK(ks.device() == d && vs.device() == d, who, ": k_scale and v_scale must be on ", d);
  TORCH_CHECK(ks.scalar_type() == at::kByte && vs.scalar_type() == at::kByte, who, ": k_scale and v_scale must be uint8");
  TORCH_CHECK(ks.dim() == 3 && ks.size(0) == kc.size(0) && ks.size(1) == kc.size(2) && ks.size(2) == kc.size(1) &&
                  ks.sizes() == vs.sizes() && ks.strides() == vs.strides() && ks.stride(2) == 1, who,
              ": k_scale and v_scale must be [num_pages, kv_heads, page_size] with equal strides and contiguous tokens");
}

// bf16 rows of the given shape, dim contiguous.
void check_rows(const char* who, const char* name, const c10::Device& d, const Tensor& t, at::IntArrayRef shape) {
  TORCH_CHECK(t.device() == d, who, ": ", name, " is on ", t.device(), ", not ", d);
  TORCH_CHECK(t.scalar_type() == at::kBFloat16, who, ": ", name, " must be bfloat16, got ", t.scalar_type());
  TORCH_CHECK(t.sizes() == shape && t.stride(-1) == 1, who, ": ", name, " must be ", shape, " with a contiguous head_dim, got ",
              t.sizes());
}

void check_slots(const char* who, const c10::Device& d, const Tensor& s) {
  TORCH_CHECK(s.device() == d && s.scalar_type() == at::kLong && s.dim() == 1 && s.is_contiguous(), who,
              ": slots must be a contiguous int64 [tokens] tensor on ", d);
}

void check_table(const char* who, const c10::Device& d, int64_t B, const Tensor& lens, const Tensor& bt) {
  TORCH_CHECK(lens.device() == d && bt.device() == d, who, ": cache_seqlens and block_table must be on ", d);
  TORCH_CHECK(lens.scalar_type() == at::kInt && lens.dim() == 1 && lens.size(0) == B && lens.is_contiguous(), who,
              ": cache_seqlens must be a contiguous int32 [batch] tensor");
  TORCH_CHECK(bt.scalar_type() == at::kInt && bt.dim() == 2 && bt.size(0) == B && bt.size(1) <= INT_MAX &&
                  (bt.stride(1) == 1 || bt.size(1) <= 1), who, ": block_table must be int32 [batch, max_pages] with contiguous rows");
}

void on_gpu(const char* who, const Tensor& t) {
  TORCH_CHECK(t.is_cuda(), who, ": tensors must be on a GPU (there is no CPU path)");
}

void paged_write_fp8(const Tensor& k, const Tensor& v, const Tensor& slots, const Tensor& kc, const Tensor& vc, const Tensor& ks,
                     const Tensor& vs) {
  const char* who = "q3attn.paged_write_fp8";
  on_gpu(who, kc);
  const c10::Device d = kc.device();
  check_fp8_pool(who, d, kc, vc, ks, vs);
  check_slots(who, d, slots);
  const int64_t T = slots.size(0), shape[3] = {T, kc.size(2), kc.size(3)};
  check_rows(who, "k", d, k, shape);
  check_rows(who, "v", d, v, shape);
  if (T == 0) return;
  const c10::DeviceGuard guard(d);
  done(q3a_paged_write_fp8(k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1),
                           slots.data_ptr<int64_t>(), kc.data_ptr(), vc.data_ptr(), kc.stride(0), kc.stride(1), kc.stride(2),
                           ks.data_ptr(), vs.data_ptr(), ks.stride(0), ks.stride(1), (int)kc.size(0), (int)kc.size(1), T,
                           (int)kc.size(2), (int)kc.size(3), stream_of(d)), "q3a_paged_write_fp8");
}

std::tuple<Tensor, Tensor> paged_read_fp8(const Tensor& kc, const Tensor& vc, const Tensor& ks, const Tensor& vs,
                                          const Tensor& slots) {
  const char* who = "q3attn.paged_read_fp8";
  on_gpu(who, kc);
  const c10::Device d = kc.device();
  check_fp8_pool(who, d, kc, vc, ks, vs);
  check_slots(who, d, slots);
  const int64_t T = slots.size(0);
  const c10::DeviceGuard guard(d);
  const int64_t shape[3] = {T, kc.size(2), kc.size(3)};
  Tensor k = empty_on(d, shape, at::kBFloat16), v = empty_on(d, shape, at::kBFloat16);
  if (T == 0) return {k, v};
  done(q3a_paged_read_fp8(kc.data_ptr(), vc.data_ptr(), kc.stride(0), kc.stride(1), kc.stride(2), ks.data_ptr(), vs.data_ptr(),
                          ks.stride(0), ks.stride(1), (int)kc.size(0), (int)kc.size(1), slots.data_ptr<int64_t>(), k.data_ptr(),
                          k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), T, (int)kc.size(2), (int)kc.size(3),
                          stream_of(d)), "q3a_paged_read_fp8");
  return {k, v};
}

// What every attention call takes beside its rows.
struct Call {
  c10::Device d;
  Tensor out, ws;
  size_t ws_bytes;
  int B, N, Hq, Hkv, D, pages, page, max_pages;

  // q [B, Hq, D] or [B, N, Hq, D]; the kernels' own limits are checked behind the C entry points.
  Call(const char* who, const Tensor& q, int64_t nodes, const Tensor& kc, const Tensor& lens, const Tensor& bt) : d(q.device()) {
    TORCH_CHECK(q.size(0) <= INT_MAX && nodes <= INT_MAX && q.size(-2) <= INT_MAX, who, ": q too large");
    check_table(who, d, q.size(0), lens, bt);
    B = (int)q.size(0);
    N = (int)nodes;
    Hq = (int)q.size(-2);
    D = (int)q.size(-1);
    pages = (int)kc.size(0);
    page = (int)kc.size(1);
    Hkv = (int)kc.size(2);
    max_pages = (int)bt.size(1);
    out = empty_on(d, q.sizes(), at::kBFloat16);
    ws_bytes = q.numel() ? q3a_paged_decode_tree_workspace_bytes(B, N, Hq, Hkv, D, max_pages, page) : 0;
    if (ws_bytes > 0) ws = empty_on(d, {(int64_t)ws_bytes}, at::kByte);
  }
  void* workspace() const { return ws_bytes > 0 ? ws.data_ptr() : nullptr; }
};

void check_decode(const char* who, const Tensor& q, const Tensor& kc, const Tensor& vc, const Tensor& ks, const Tensor& vs) {
  on_gpu(who, q);
  check_fp8_pool(who, q.device(), kc, vc, ks, vs);
  TORCH_CHECK(q.dim() == 3, who, ": q must be [batch, heads, head_dim], got ", q.sizes());
  const int64_t shape[3] = {q.size(0), q.size(1), kc.size(3)};
  check_rows(who, "q", q.device(), q, shape);
}

Tensor paged_decode_fp8(const Tensor& q, const Tensor& kc, const Tensor& vc, const Tensor& ks, const Tensor& vs, const Tensor& lens,
                        const Tensor& bt, double softmax_scale) {
  const char* who = "q3attn.paged_decode_fp8";
  check_decode(who, q, kc, vc, ks, vs);
  const c10::DeviceGuard guard(q.device());
  const Call c(who, q, 1, kc, lens, bt);
  if (c.B == 0) return c.out;
  done(q3a_paged_decode_fp8(q.data_ptr(), q.stride(0), q.stride(1), kc.data_ptr(), vc.data_ptr(), kc.stride(0), kc.stride(1),
                            kc.stride(2), ks.data_ptr(), vs.data_ptr(), ks.stride(0), ks.stride(1), c.pages, c.page,
                            lens.data_ptr<int>(), bt.data_ptr<int>(), bt.stride(0), c.max_pages, c.out.data_ptr(),
                            c.out.stride(0), c.out.stride(1), c.workspace(), c.ws_bytes, c.B, c.Hq, c.Hkv, c.D,
                            (float)softmax_scale, stream_of(c.d)), "q3a_paged_decode_fp8");
  return c.out;
}

Tensor paged_decode_fp8_append(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& kc, const Tensor& vc,
                               const Tensor& ks, const Tensor& vs, const Tensor& lens, const Tensor& bt, double softmax_scale) {
  const char* who = "q3attn.paged_decode_fp8_append";
  check_decode(who, q, kc, vc, ks, vs);
  const int64_t shape[3] = {q.size(0), kc.size(2), kc.size(3)};
  check_rows(who, "k", q.device(), k, shape);
  check_rows(who, "v", q.device(), v, shape);
  const c10::DeviceGuard guard(q.device());
  const Call c(who, q, 1, kc, lens, bt);
  if (c.B == 0) return c.out;
  done(q3a_paged_decode_fp8_append(q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(),
                                   v.stride(0), v.stride(1), kc.data_ptr(), vc.data_ptr(), kc.stride(0), kc.stride(1),
                                   kc.stride(2), ks.data_ptr(), vs.data_ptr(), ks.stride(0), ks.stride(1), c.pages, c.page,
                                   lens.data_ptr<int>(), bt.data_ptr<int>(), bt.stride(0), c.max_pages, c.out.data_ptr(),
                                   c.out.stride(0), c.out.stride(1), c.workspace(), c.ws_bytes, c.B, c.Hq, c.Hkv, c.D,
                                   (float)softmax_scale, stream_of(c.d)), "q3a_paged_decode_fp8_append");
  return c.out;
}

Tensor paged_decode_tree(const Tensor& q, const Tensor& k, const Tensor& v, const optional<Tensor>& tree_mask, const Tensor& kc,
                         const Tensor& vc, const Tensor& lens, const Tensor& bt, double softmax_scale,
                         const optional<Tensor>& k_scale, const optional<Tensor>& v_scale) {
  const char* who = "q3attn.paged_decode_tree";
  on_gpu(who, q);
  const c10::Device d = q.device();
  TORCH_CHECK(k_scale.has_value() == v_scale.has_value(), who, ": pass both k_scale and v_scale, or neither");
  const void *ks = nullptr, *vs = nullptr;
  int64_t ss_p = 0, ss_h = 0;
  if (k_scale.has_value()) {
    check_fp8_pool(who, d, kc, vc, *k_scale, *v_scale);
    ks = k_scale->data_ptr();
    vs = v_scale->data_ptr();
    ss_p = k_scale->stride(0);
    ss_h = k_scale->stride(1);
    TORCH_CHECK(ks != nullptr && vs != nullptr, who, ": empty scales");
  } else {
    check_caches(who, d, kc, vc, at::kBFloat16);
  }
  TORCH_CHECK(q.dim() == 4, who, ": q must be [batch, nodes, heads, head_dim], got ", q.sizes());
  const int64_t B = q.size(0), N = q.size(1);
  const int64_t qs[4] = {B, N, q.size(2), kc.size(3)}, kvs[4] = {B, N, kc.size(2), kc.size(3)};
  check_rows(who, "q", d, q, qs);
  check_rows(who, "k", d, k, kvs);
  check_rows(who, "v", d, v, kvs);
  const uint8_t* mask = nullptr;
  int64_t m_sb = 0, m_sn = 0;
  if (tree_mask.has_value()) {
    const Tensor& m = *tree_mask;
    TORCH_CHECK(m.device() == d && m.scalar_type() == at::kBool, who, ": tree_mask must be bool on ", d);
    TORCH_CHECK((m.dim() == 2 || (m.dim() == 3 && m.size(0) == B)) && m.size(-1) == N && m.size(-2) == N, who,
                ": tree_mask must be [batch, nodes, nodes] or [nodes, nodes], got ", m.sizes());
    TORCH_CHECK(m.stride(-1) == 1 || N <= 1, who, ": tree_mask rows must be contiguous");
    mask = (const uint8_t*)m.data_ptr();
    m_sb = m.dim() == 3 ? m.stride(0) : 0;
    m_sn = m.stride(-2);
  }
  const c10::DeviceGuard guard(d);
  const Call c(who, q, N, kc, lens, bt);
  if (c.out.numel() == 0) return c.out;
  done(q3a_paged_decode_tree(q.data_ptr(), q.stride(0), q.stride(1), q.stride(2), k.data_ptr(), k.stride(0), k.stride(1),
                             k.stride(2), v.data_ptr(), v.stride(0), v.stride(1), v.stride(2), mask, m_sb, m_sn, kc.data_ptr(),
                             vc.data_ptr(), kc.stride(0), kc.stride(1), kc.stride(2), ks, vs, ss_p, ss_h, c.pages, c.page,
                             lens.data_ptr<int>(), bt.data_ptr<int>(), bt.stride(0), c.max_pages, c.out.data_ptr(),
                             c.out.stride(0), c.out.stride(1), c.out.stride(2), c.workspace(), c.ws_bytes, c.B, c.N, c.Hq, c.Hkv,
                             c.D, (float)softmax_scale, stream_of(d)), "q3a_paged_decode_tree");
  return c.out;
}

// What autograd sees.  None of the ops has a backward: one that is asked for raises, instead of leaving gradients out.  And the ops
// that write into caches count as in-place operations on them, so that autograd notices a cache that it has saved.
//
// (Each form calls the op again below its own dispatch key, as dispatch modes and fake tensors have to see it there.)
template <class Op>
auto op_of(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Op>();
}

void no_backward(const char* name, const Tensor& out, torch::autograd::edge_list&& edges) {
  torch::autograd::set_history(
      out, std::shared_ptr<torch::autograd::Node>(new torch::autograd::NotImplemented(name, std::move(edges)), torch::autograd::deleteNode));
}

Tensor decode_autograd(const Tensor& q, const Tensor& kc, const Tensor& vc, const Tensor& ks, const Tensor& vs, const Tensor& lens,
                       const Tensor& bt, double softmax_scale) {
  static const auto op = op_of<decltype(paged_decode_fp8)>("q3attn::paged_decode_fp8");
  Tensor out;
  {
    const at::AutoDispatchBelowAutograd below;
    out = op.call(q, kc, vc, ks, vs, lens, bt, softmax_scale);
  }
  if (torch::autograd::compute_requires_grad(q, kc, vc))
    no_backward("q3attn::paged_decode_fp8", out, torch::autograd::collect_next_edges(q, kc, vc));
  return out;
}

Tensor decode_append_autograd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& kc, const Tensor& vc, const Tensor& ks,
                              const Tensor& vs, const Tensor& lens, const Tensor& bt, double softmax_scale) {
  static const auto op = op_of<decltype(paged_decode_fp8_append)>("q3attn::paged_decode_fp8_append");
  Tensor out;
  {
    const at::AutoDispatchBelowAutograd below;
    out = op.call(q, k, v, kc, vc, ks, vs, lens, bt, softmax_scale);
  }
  if (torch::autograd::compute_requires_grad(q, k, v))
    no_backward("q3attn::paged_decode_fp8_append", out, torch::autograd::collect_next_edges(q, k, v));
  return out;
}

std::tuple<Tensor, Tensor> read_autograd(const Tensor& kc, const Tensor& vc, const Tensor& ks, const Tensor& vs, const Tensor& slots) {
  static const auto op = op_of<decltype(paged_read_fp8)>("q3attn::paged_read_fp8");
  std::tuple<Tensor, Tensor> out;
  {
    const at::AutoDispatchBelowAutograd below;
    out = op.call(kc, vc, ks, vs, slots);
  }
  if (torch::autograd::compute_requires_grad(kc, vc)) {
    no_backward("q3attn::paged_read_fp8", std::get<0>(out), torch::autograd::collect_next_edges(kc, vc));
    no_backward("q3attn::paged_read_fp8", std::get<1>(out), torch::autograd::collect_next_edges(kc, vc));
  }
  return out;
}

Tensor tree_autograd(const Tensor& q, const Tensor& k, const Tensor& v, const optional<Tensor>& tree_mask, const Tensor& kc,
                     const Tensor& vc, const Tensor& lens, const Tensor& bt, double softmax_scale, const optional<Tensor>& k_scale,
                     const optional<Tensor>& v_scale) {
  static const auto op = op_of<decltype(paged_decode_tree)>("q3attn::paged_decode_tree");
  Tensor out;
  {
    const at::AutoDispatchBelowAutograd below;
    out = op.call(q, k, v, tree_mask, kc, vc, lens, bt, softmax_scale, k_scale, v_scale);
  }
  if (torch::autograd::compute_requires_grad(q, k, v, kc, vc))
    no_backward("q3attn::paged_decode_tree", out, torch::autograd::collect_next_edges(q, k, v, kc, vc));
  return out;
}

template <class... T>
void written(const T&... caches) {
  for (const Tensor& t : {caches...})
    if (!t.is_inference()) torch::autograd::increment_version(t);
}

void write_in_place(const Tensor& k, const Tensor& v, const Tensor& slots, const Tensor& kc, const Tensor& vc, const Tensor& ks,
                    const Tensor& vs) {
  static const auto op = op_of<decltype(paged_write_fp8)>("q3attn::paged_write_fp8");
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    op.call(k, v, slots, kc, vc, ks, vs);
  }
  written(kc, vc, ks, vs);
}

Tensor decode_append_in_place(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& kc, const Tensor& vc, const Tensor& ks,
                              const Tensor& vs, const Tensor& lens, const Tensor& bt, double softmax_scale) {
  static const auto op = op_of<decltype(paged_decode_fp8_append)>("q3attn::paged_decode_fp8_append");
  Tensor out;
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    out = op.call(q, k, v, kc, vc, ks, vs, lens, bt, softmax_scale);
  }
  written(kc, vc, ks, vs);
  return out;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(q3attn, m) {
  m.def("paged_write_fp8(Tensor k, Tensor v, Tensor slots, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) k_scale, "
        "Tensor(d!) v_scale) -> ()");
  m.def("paged_read_fp8(Tensor k_cache, Tensor v_cache, Tensor k_scale, Tensor v_scale, Tensor slots) -> (Tensor, Tensor)");
  m.def("paged_decode_fp8(Tensor q, Tensor k_cache, Tensor v_cache, Tensor k_scale, Tensor v_scale, Tensor cache_seqlens, "
        "Tensor block_table, float softmax_scale) -> Tensor");
  m.def("paged_decode_fp8_append(Tensor q, Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) k_scale, "
        "Tensor(d!) v_scale, Tensor cache_seqlens, Tensor block_table, float softmax_scale) -> Tensor");
  m.def("paged_decode_tree(Tensor q, Tensor k, Tensor v, Tensor? tree_mask, Tensor k_cache, Tensor v_cache, Tensor cache_seqlens, "
        "Tensor block_table, float softmax_scale, Tensor? k_scale=None, Tensor? v_scale=None) -> Tensor");
}

// One implementation for every backend: on CPU tensors it says that there is none.
TORCH_LIBRARY_IMPL(q3attn, CompositeExplicitAutograd, m) {
  m.impl("paged_write_fp8", &paged_write_fp8);
  m.impl("paged_read_fp8", &paged_read_fp8);
  m.impl("paged_decode_fp8", &paged_decode_fp8);
  m.impl("paged_decode_fp8_append", &paged_decode_fp8_append);
  m.impl("paged_decode_tree", &paged_decode_tree);
}

TORCH_LIBRARY_IMPL(q3attn, Autograd, m) {
  m.impl("paged_read_fp8", &read_autograd);
  m.impl("paged_decode_fp8", &decode_autograd);
  m.impl("paged_decode_fp8_append", &decode_append_autograd);
  m.impl("paged_decode_tree", &tree_autograd);
}

TORCH_LIBRARY_IMPL(q3attn, ADInplaceOrView, m) {
  m.impl("paged_write_fp8", &write_in_place);
  m.impl("paged_decode_fp8_append", &decode_append_in_place);
}
