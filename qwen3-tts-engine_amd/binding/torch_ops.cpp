// The 8- and 4-bit pools', the tree attention's and the page moves' torch ops over the C ABI (include/q3attn.h).
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

#include <algorithm>
#include <string>
#include <tuple>
#include <utility>

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

// The pools of 8- and 4-bit codes, which differ in their types and in the C entry points behind their ops.
template <int kBits>
constexpr const char* pick(const char* of8, const char* of4) {
  return kBits == 8 ? of8 : of4;
}

template <int kBits>
void check_pool(const char* who, const c10::Device& d, const Tensor& kc, const Tensor& vc, const Tensor& ks, const Tensor& vs) {
  check_caches(who, d, kc, vc, kBits == 8 ? at::kFloat8_e4m3fn : at::kByte);
  TORCH_CHECK(ks.device() == d && vs.device() == d, who, ": k_scale and v_scale must be on ", d);
  TORCH_CHECK(ks.scalar_type() == at::kByte && vs.scalar_type() == at::kByte, who, ": k_scale and v_scale must be uint8");
  TORCH_CHECK(ks.sizes() == vs.sizes() && ks.strides() == vs.strides(), who, ": k_scale and v_scale must have equal shapes and strides");
  if constexpr (kBits == 8) {
    TORCH_CHECK(ks.dim() == 3 && ks.size(0) == kc.size(0) && ks.size(1) == kc.size(2) && ks.size(2) == kc.size(1) && ks.stride(2) == 1,
                who, ": k_scale and v_scale must be [num_pages, kv_heads, page_size] with equal strides and contiguous tokens");
  } else {
    TORCH_CHECK(kc.size(3) == 64, who, ": k_cache and v_cache must be [num_pages, page_size, kv_heads, 64] (two codes a byte)");
    TORCH_CHECK(ks.dim() == 4 && ks.size(0) == kc.size(0) && ks.size(1) == kc.size(2) && ks.size(2) == 4 && ks.size(3) == kc.size(1) &&
                    ks.stride(3) == 1 && ks.stride(2) == ks.size(3), who,
                ": k_scale and v_scale must be [num_pages, kv_heads, 4, page_size] with equal strides and contiguous blocks");
  }
}
template <int kBits>
int64_t head_dim_of(const Tensor& kc) {
  return kBits == 8 ? kc.size(3) : 2 * kc.size(3);
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

template <int kBits>
void paged_write(const Tensor& k, const Tensor& v, const Tensor& slots, const Tensor& kc, const Tensor& vc, const Tensor& ks,
                 const Tensor& vs) {
  const char* who = pick<kBits>("q3attn.paged_write_fp8", "q3attn.paged_write_fp4");
  on_gpu(who, kc);
  const c10::Device d = kc.device();
  check_pool<kBits>(who, d, kc, vc, ks, vs);
  check_slots(who, d, slots);
  const int64_t T = slots.size(0), D = head_dim_of<kBits>(kc), shape[3] = {T, kc.size(2), D};
  check_rows(who, "k", d, k, shape);
  check_rows(who, "v", d, v, shape);
  if (T == 0) return;
  const c10::DeviceGuard guard(d);
  constexpr auto call = kBits == 8 ? &q3a_paged_write_fp8 : &q3a_paged_write_fp4;
  done(call(k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1),
            slots.data_ptr<int64_t>(), kc.data_ptr(), vc.data_ptr(), kc.stride(0), kc.stride(1), kc.stride(2), ks.data_ptr(),
            vs.data_ptr(), ks.stride(0), ks.stride(1), (int)kc.size(0), (int)kc.size(1), T, (int)kc.size(2), (int)D, stream_of(d)),
       pick<kBits>("q3a_paged_write_fp8", "q3a_paged_write_fp4"));
}

template <int kBits>
std::tuple<Tensor, Tensor> paged_read(const Tensor& kc, const Tensor& vc, const Tensor& ks, const Tensor& vs, const Tensor& slots) {
  const char* who = pick<kBits>("q3attn.paged_read_fp8", "q3attn.paged_read_fp4");
  on_gpu(who, kc);
  const c10::Device d = kc.device();
  check_pool<kBits>(who, d, kc, vc, ks, vs);
  check_slots(who, d, slots);
  const int64_t T = slots.size(0);
  const c10::DeviceGuard guard(d);
  const int64_t D = head_dim_of<kBits>(kc), shape[3] = {T, kc.size(2), D};
  Tensor k = empty_on(d, shape, at::kBFloat16), v = empty_on(d, shape, at::kBFloat16);
  if (T == 0) return {k, v};
  constexpr auto call = kBits == 8 ? &q3a_paged_read_fp8 : &q3a_paged_read_fp4;
  done(call(kc.data_ptr(), vc.data_ptr(), kc.stride(0), kc.stride(1), kc.stride(2), ks.data_ptr(), vs.data_ptr(), ks.stride(0),
            ks.stride(1), (int)kc.size(0), (int)kc.size(1), slots.data_ptr<int64_t>(), k.data_ptr(), k.stride(0), k.stride(1),
            v.data_ptr(), v.stride(0), v.stride(1), T, (int)kc.size(2), (int)D, stream_of(d)),
       pick<kBits>("q3a_paged_read_fp8", "q3a_paged_read_fp4"));
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

template <int kBits>
void check_decode(const char* who, const Tensor& q, const Tensor& kc, const Tensor& vc, const Tensor& ks, const Tensor& vs) {
  on_gpu(who, q);
  check_pool<kBits>(who, q.device(), kc, vc, ks, vs);
  TORCH_CHECK(q.dim() == 3, who, ": q must be [batch, heads, head_dim], got ", q.sizes());
  const int64_t shape[3] = {q.size(0), q.size(1), head_dim_of<kBits>(kc)};
  check_rows(who, "q", q.device(), q, shape);
}

template <int kBits>
Tensor paged_decode(const Tensor& q, const Tensor& kc, const Tensor& vc, const Tensor& ks, const Tensor& vs, const Tensor& lens,
                    const Tensor& bt, double softmax_scale) {
  const char* who = pick<kBits>("q3attn.paged_decode_fp8", "q3attn.paged_decode_fp4");
  check_decode<kBits>(who, q, kc, vc, ks, vs);
  const c10::DeviceGuard guard(q.device());
  const Call c(who, q, 1, kc, lens, bt);
  if (c.B == 0) return c.out;
  constexpr auto call = kBits == 8 ? &q3a_paged_decode_fp8 : &q3a_paged_decode_fp4;
  done(call(q.data_ptr(), q.stride(0), q.stride(1), kc.data_ptr(), vc.data_ptr(), kc.stride(0), kc.stride(1),
            kc.stride(2), ks.data_ptr(), vs.data_ptr(), ks.stride(0), ks.stride(1), c.pages, c.page,
            lens.data_ptr<int>(), bt.data_ptr<int>(), bt.stride(0), c.max_pages, c.out.data_ptr(),
            c.out.stride(0), c.out.stride(1), c.workspace(), c.ws_bytes, c.B, c.Hq, c.Hkv, c.D,
            (float)softmax_scale, stream_of(c.d)), pick<kBits>("q3a_paged_decode_fp8", "q3a_paged_decode_fp4"));
  return c.out;
}

template <int kBits>
Tensor paged_decode_append(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& kc, const Tensor& vc, const Tensor& ks,
                           const Tensor& vs, const Tensor& lens, const Tensor& bt, double softmax_scale) {
  const char* who = pick<kBits>("q3attn.paged_decode_fp8_append", "q3attn.paged_decode_fp4_append");
  check_decode<kBits>(who, q, kc, vc, ks, vs);
  const int64_t shape[3] = {q.size(0), kc.size(2), head_dim_of<kBits>(kc)};
  check_rows(who, "k", q.device(), k, shape);
  check_rows(who, "v", q.device(), v, shape);
  const c10::DeviceGuard guard(q.device());
  const Call c(who, q, 1, kc, lens, bt);
  if (c.B == 0) return c.out;
  constexpr auto call = kBits == 8 ? &q3a_paged_decode_fp8_append : &q3a_paged_decode_fp4_append;
  done(call(q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(),
            v.stride(0), v.stride(1), kc.data_ptr(), vc.data_ptr(), kc.stride(0), kc.stride(1),
            kc.stride(2), ks.data_ptr(), vs.data_ptr(), ks.stride(0), ks.stride(1), c.pages, c.page,
            lens.data_ptr<int>(), bt.data_ptr<int>(), bt.stride(0), c.max_pages, c.out.data_ptr(),
            c.out.stride(0), c.out.stride(1), c.workspace(), c.ws_bytes, c.B, c.Hq, c.Hkv, c.D,
            (float)softmax_scale, stream_of(c.d)), pick<kBits>("q3a_paged_decode_fp8_append", "q3a_paged_decode_fp4_append"));
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
    check_pool<8>(who, d, kc, vc, *k_scale, *v_scale);
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

// A cache [num_pages, ...] as its pages' memory: runs of it, in at most two more dimensions.
q3a_page_cache page_cache(const char* who, const c10::Device& d, const Tensor& t) {
  TORCH_CHECK(t.device() == d, who, ": all caches and page lists must be on ", d, ", got ", t.device());
  TORCH_CHECK(t.dim() >= 1 && t.size(0) <= INT_MAX, who, ": a cache must be [num_pages, ...], got ", t.sizes());
  const int64_t elem = t.element_size();
  q3a_page_cache c = {t.data_ptr(), t.stride(0) * elem, 0, 0, 1, 1, elem, (int)t.size(0)};
  c10::SmallVector<std::pair<int64_t, int64_t>, 8> dims;  // stride, size
  for (int64_t i = 1; i < t.dim(); ++i)
    if (t.size(i) > 1) dims.emplace_back(t.stride(i) * elem, t.size(i));
  std::sort(dims.begin(), dims.end());
  int more = 0;
  for (const auto& [stride, size] : dims) {
    if (more == 0 && stride == c.run_bytes) {
      c.run_bytes *= size;
    } else if (more == 1 && stride == c.stride_0 * c.n_0) {
      c.n_0 *= size;
    } else {
      TORCH_CHECK(stride > 0 && more < 2, who, ": a cache's pages must be made of runs of memory in at most two dimensions, got strides ",
                  t.strides());
      (more == 0 ? c.stride_0 : c.stride_1) = stride;
      (more == 0 ? c.n_0 : c.n_1) = size;
      ++more;
    }
  }
  return c;
}

void check_pages(const char* who, const char* name, const c10::Device& d, const Tensor& t) {
  TORCH_CHECK(t.device() == d && t.scalar_type() == at::kInt && t.dim() == 1 && t.is_contiguous(), who, ": ", name,
              " must be a contiguous int32 [pairs] tensor on ", d);
}

void paged_copy(at::TensorList caches, const Tensor& src, const Tensor& dst) {
  const char* who = "q3attn.paged_copy";
  TORCH_CHECK(!caches.empty(), who, ": at least one cache");
  on_gpu(who, caches[0]);
  const c10::Device d = caches[0].device();
  check_pages(who, "src", d, src);
  check_pages(who, "dst", d, dst);
  TORCH_CHECK(src.size(0) == dst.size(0), who, ": ", src.size(0), " source pages for ", dst.size(0));
  c10::SmallVector<q3a_page_cache, 64> list;
  c10::SmallVector<std::pair<const Tensor*, q3a_page_cache>, 4> known;  // (layers are alike: a shape is worked out once)
  size_t k = 0;                                                         // the last cache's
  const auto alike = [](const Tensor& t, const Tensor& u) {
    return t.element_size() == u.element_size() && t.sizes() == u.sizes() && t.strides() == u.strides();
  };
  for (const Tensor& t : caches) {
    if (known.empty() || !alike(t, *known[k].first)) {
      k = 0;
      while (k < known.size() && !alike(t, *known[k].first)) ++k;
    }
    if (k == known.size() || t.device() != d) {
      known.emplace_back(&t, page_cache(who, d, t));
      k = known.size() - 1;
    }
    if (t.numel() == 0) continue;
    list.push_back(known[k].second);
    list.back().base = t.data_ptr();
  }
  if (list.empty()) return;
  const c10::DeviceGuard guard(d);
  done(q3a_paged_copy(list.data(), (int)list.size(), src.data_ptr<int>(), dst.data_ptr<int>(), src.size(0), stream_of(d)), "q3a_paged_copy");
}

Tensor paged_compact(at::TensorList caches, const Tensor& keep, const Tensor& lens, const Tensor& bt, at::TensorList scales) {
  const char* who = "q3attn.paged_compact";
  TORCH_CHECK(!caches.empty(), who, ": at least one cache");
  const Tensor& first = caches[0];
  on_gpu(who, first);
  const c10::Device d = first.device();
  TORCH_CHECK(first.dim() == 4 && first.stride(3) == 1 && first.size(0) <= INT_MAX && first.size(1) <= INT_MAX && first.size(2) <= INT_MAX, who,
              ": a cache must be [num_pages, page_size, kv_heads, row] with contiguous rows, got ", first.sizes());
  TORCH_CHECK(first.numel() > 0, who, ": empty caches");
  const int64_t elem = first.element_size(), row = first.size(3) * elem;
  TORCH_CHECK((first.scalar_type() == at::kBFloat16 && row == 256) || (first.scalar_type() == at::kFloat8_e4m3fn && row == 128) ||
                  (first.scalar_type() == at::kByte && row == 64), who,
              ": caches must be a bf16 pool's, an 8-bit pool's or a 4-bit pool's, got ", first.scalar_type(), " ", first.sizes());
  const int64_t blocks = elem == 2 ? 0 : row == 128 ? 1 : 4;
  TORCH_CHECK(scales.size() == (blocks > 0 ? caches.size() : 0), who, ": ", caches.size(), " caches of this pool take ",
              blocks > 0 ? caches.size() : 0, " scales, got ", scales.size());
  c10::SmallVector<void*, 64> codes, exps;
  for (const Tensor& t : caches) {
    TORCH_CHECK(t.device() == d && t.scalar_type() == first.scalar_type() && t.sizes() == first.sizes() && t.strides() == first.strides(), who,
                ": all caches must be on ", d, " with one type, shape and strides");
    codes.push_back(t.data_ptr());
  }
  for (const Tensor& t : scales) {
    const Tensor& f = scales[0];
    TORCH_CHECK(t.device() == d && t.scalar_type() == at::kByte && t.sizes() == f.sizes() && t.strides() == f.strides(), who,
                ": all scales must be uint8 on ", d, " with one shape and strides");
    exps.push_back(t.data_ptr());
  }
  const int64_t P = first.size(0), page = first.size(1), H = first.size(2);
  if (blocks == 1) {
    const int64_t shape[3] = {P, H, page};
    TORCH_CHECK(scales[0].sizes() == at::IntArrayRef(shape) && scales[0].stride(2) == 1, who,
                ": scales must be [num_pages, kv_heads, page_size] with contiguous tokens");
  } else if (blocks == 4) {
    const int64_t shape[4] = {P, H, 4, page};
    TORCH_CHECK(scales[0].sizes() == at::IntArrayRef(shape) && scales[0].stride(3) == 1 && scales[0].stride(2) == page, who,
                ": scales must be [num_pages, kv_heads, 4, page_size] with contiguous blocks");
  }
  const int64_t B = lens.dim() == 1 ? lens.size(0) : 0;
  check_table(who, d, B, lens, bt);
  TORCH_CHECK(keep.device() == d && keep.scalar_type() == at::kBool && keep.dim() == 2 && keep.size(0) == B && keep.size(1) <= INT_MAX &&
                  (keep.stride(1) == 1 || keep.size(1) <= 1), who, ": keep must be bool [batch, tokens] with contiguous rows on ", d);
  const c10::DeviceGuard guard(d);
  Tensor out = empty_on(d, {B}, at::kInt);
  if (B == 0) return out;
  done(q3a_paged_compact(codes.data(), blocks > 0 ? exps.data() : nullptr, (int)codes.size(), (int)row, (int)blocks, first.stride(0) * elem,
                         first.stride(1) * elem, first.stride(2) * elem, blocks > 0 ? scales[0].stride(0) : 0,
                         blocks > 0 ? scales[0].stride(1) : 0, (int)P, (int)page, (const uint8_t*)keep.data_ptr(), keep.stride(0),
                         (int)keep.size(1), lens.data_ptr<int>(), bt.data_ptr<int>(), bt.stride(0), (int)bt.size(1), out.data_ptr<int>(), (int)B,
                         (int)H, stream_of(d)), "q3a_paged_compact");
  return out;
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

template <int kBits>
Tensor decode_autograd(const Tensor& q, const Tensor& kc, const Tensor& vc, const Tensor& ks, const Tensor& vs, const Tensor& lens,
                       const Tensor& bt, double softmax_scale) {
  constexpr const char* name = pick<kBits>("q3attn::paged_decode_fp8", "q3attn::paged_decode_fp4");
  static const auto op = op_of<decltype(paged_decode<kBits>)>(name);
  Tensor out;
  {
    const at::AutoDispatchBelowAutograd below;
    out = op.call(q, kc, vc, ks, vs, lens, bt, softmax_scale);
  }
  if (torch::autograd::compute_requires_grad(q, kc, vc))
    no_backward(name, out, torch::autograd::collect_next_edges(q, kc, vc));
  return out;
}

template <int kBits>
Tensor decode_append_autograd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& kc, const Tensor& vc, const Tensor& ks,
                              const Tensor& vs, const Tensor& lens, const Tensor& bt, double softmax_scale) {
  constexpr const char* name = pick<kBits>("q3attn::paged_decode_fp8_append", "q3attn::paged_decode_fp4_append");
  static const auto op = op_of<decltype(paged_decode_append<kBits>)>(name);
  Tensor out;
  {
    const at::AutoDispatchBelowAutograd below;
    out = op.call(q, k, v, kc, vc, ks, vs, lens, bt, softmax_scale);
  }
  if (torch::autograd::compute_requires_grad(q, k, v))
    no_backward(name, out, torch::autograd::collect_next_edges(q, k, v));
  return out;
}

template <int kBits>
std::tuple<Tensor, Tensor> read_autograd(const Tensor& kc, const Tensor& vc, const Tensor& ks, const Tensor& vs, const Tensor& slots) {
  constexpr const char* name = pick<kBits>("q3attn::paged_read_fp8", "q3attn::paged_read_fp4");
  static const auto op = op_of<decltype(paged_read<kBits>)>(name);
  std::tuple<Tensor, Tensor> out;
  {
    const at::AutoDispatchBelowAutograd below;
    out = op.call(kc, vc, ks, vs, slots);
  }
  if (torch::autograd::compute_requires_grad(kc, vc)) {
    no_backward(name, std::get<0>(out), torch::autograd::collect_next_edges(kc, vc));
    no_backward(name, std::get<1>(out), torch::autograd::collect_next_edges(kc, vc));
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
  for (const Tensor* t : {&caches...})
    if (!t->is_inference()) torch::autograd::increment_version(*t);
}

template <int kBits>
void write_in_place(const Tensor& k, const Tensor& v, const Tensor& slots, const Tensor& kc, const Tensor& vc, const Tensor& ks,
                    const Tensor& vs) {
  static const auto op = op_of<decltype(paged_write<kBits>)>(pick<kBits>("q3attn::paged_write_fp8", "q3attn::paged_write_fp4"));
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    op.call(k, v, slots, kc, vc, ks, vs);
  }
  written(kc, vc, ks, vs);
}

template <int kBits>
Tensor decode_append_in_place(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& kc, const Tensor& vc, const Tensor& ks,
                              const Tensor& vs, const Tensor& lens, const Tensor& bt, double softmax_scale) {
  static const auto op =
      op_of<decltype(paged_decode_append<kBits>)>(pick<kBits>("q3attn::paged_decode_fp8_append", "q3attn::paged_decode_fp4_append"));
  Tensor out;
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    out = op.call(q, k, v, kc, vc, ks, vs, lens, bt, softmax_scale);
  }
  written(kc, vc, ks, vs);
  return out;
}

void copy_in_place(at::TensorList caches, const Tensor& src, const Tensor& dst) {
  static const auto op = op_of<decltype(paged_copy)>("q3attn::paged_copy");
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    op.call(caches, src, dst);
  }
  for (const Tensor& t : caches) written(t);
}

Tensor compact_in_place(at::TensorList caches, const Tensor& keep, const Tensor& lens, const Tensor& bt, at::TensorList scales) {
  static const auto op = op_of<decltype(paged_compact)>("q3attn::paged_compact");
  Tensor out;
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    out = op.call(caches, keep, lens, bt, scales);
  }
  for (const Tensor& t : caches) written(t);
  for (const Tensor& t : scales) written(t);
  return out;
}

// The moves take bf16 caches, whose elements may have a history.  What they write over no longer follows from it, so the cache's history
// becomes a node that raises; a leaf is refused, as by torch's own in-place operations.
// Whether a cache has a history that the move ends.
bool check_moved(at::TensorList caches) {
  if (!at::GradMode::is_enabled()) return false;
  bool any = false;
  for (const Tensor& t : caches)
    if (t.requires_grad()) {
      torch::autograd::check_inplace(t, true);
      any = true;
    }
  return any;
}
void moved(const char* name, at::TensorList caches) {
  for (const Tensor& t : caches)
    if (t.requires_grad())
      torch::autograd::rebase_history(
          t, std::shared_ptr<torch::autograd::Node>(new torch::autograd::NotImplemented(name, torch::autograd::collect_next_edges(t)),
                                                    torch::autograd::deleteNode));
}

// (Straight to the in-place forms: another way through the dispatcher with lists of 56 caches takes 0.3 us.)
void copy_autograd(at::TensorList caches, const Tensor& src, const Tensor& dst) {
  const bool any = check_moved(caches);
  copy_in_place(caches, src, dst);
  if (any) moved("q3attn::paged_copy", caches);
}

Tensor compact_autograd(at::TensorList caches, const Tensor& keep, const Tensor& lens, const Tensor& bt, at::TensorList scales) {
  const bool any = check_moved(caches);
  const Tensor out = compact_in_place(caches, keep, lens, bt, scales);
  if (any) moved("q3attn::paged_compact", caches);
  return out;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(q3attn, m) {
  for (const std::string bits : {"8", "4"}) {
    const std::string pool = "Tensor k_cache, Tensor v_cache, Tensor k_scale, Tensor v_scale";
    const std::string written = "Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) k_scale, Tensor(d!) v_scale";
    const std::string rows = "Tensor cache_seqlens, Tensor block_table, float softmax_scale";
    m.def(("paged_write_fp" + bits + "(Tensor k, Tensor v, Tensor slots, " + written + ") -> ()").c_str());
    m.def(("paged_read_fp" + bits + "(" + pool + ", Tensor slots) -> (Tensor, Tensor)").c_str());
    m.def(("paged_decode_fp" + bits + "(Tensor q, " + pool + ", " + rows + ") -> Tensor").c_str());
    m.def(("paged_decode_fp" + bits + "_append(Tensor q, Tensor k, Tensor v, " + written + ", " + rows + ") -> Tensor").c_str());
  }
  m.def("paged_decode_tree(Tensor q, Tensor k, Tensor v, Tensor? tree_mask, Tensor k_cache, Tensor v_cache, Tensor cache_seqlens, "
        "Tensor block_table, float softmax_scale, Tensor? k_scale=None, Tensor? v_scale=None) -> Tensor");
  m.def("paged_copy(Tensor(a!)[] caches, Tensor src, Tensor dst) -> ()");
  m.def("paged_compact(Tensor(a!)[] caches, Tensor keep, Tensor cache_seqlens, Tensor block_table, Tensor(b!)[] scales) -> Tensor");
}

// One implementation for every backend: on CPU tensors it says that there is none.
TORCH_LIBRARY_IMPL(q3attn, CompositeExplicitAutograd, m) {
  m.impl("paged_write_fp8", &paged_write<8>);
  m.impl("paged_write_fp4", &paged_write<4>);
  m.impl("paged_read_fp8", &paged_read<8>);
  m.impl("paged_read_fp4", &paged_read<4>);
  m.impl("paged_decode_fp8", &paged_decode<8>);
  m.impl("paged_decode_fp4", &paged_decode<4>);
  m.impl("paged_decode_fp8_append", &paged_decode_append<8>);
  m.impl("paged_decode_fp4_append", &paged_decode_append<4>);
  m.impl("paged_decode_tree", &paged_decode_tree);
  m.impl("paged_copy", &paged_copy);
  m.impl("paged_compact", &paged_compact);
}

TORCH_LIBRARY_IMPL(q3attn, Autograd, m) {
  m.impl("paged_read_fp8", &read_autograd<8>);
  m.impl("paged_read_fp4", &read_autograd<4>);
  m.impl("paged_decode_fp8", &decode_autograd<8>);
  m.impl("paged_decode_fp4", &decode_autograd<4>);
  m.impl("paged_decode_fp8_append", &decode_append_autograd<8>);
  m.impl("paged_decode_fp4_append", &decode_append_autograd<4>);
  m.impl("paged_decode_tree", &tree_autograd);
  m.impl("paged_copy", &copy_autograd);
  m.impl("paged_compact", &compact_autograd);
}

TORCH_LIBRARY_IMPL(q3attn, ADInplaceOrView, m) {
  m.impl("paged_write_fp8", &write_in_place<8>);
  m.impl("paged_write_fp4", &write_in_place<4>);
  m.impl("paged_decode_fp8_append", &decode_append_in_place<8>);
  m.impl("paged_decode_fp4_append", &decode_append_in_place<4>);
  m.impl("paged_copy", &copy_in_place);
  m.impl("paged_compact", &compact_in_place);
}
