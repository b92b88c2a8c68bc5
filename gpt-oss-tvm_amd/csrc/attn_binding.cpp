// The wrappers of the trees' and beams' entry points (attn_native.py), in C++: their argument
// checks, the buffers that they allocate and the call.  A call's host time with its launches, us in
// Python and here: a tree 17, 9.4, a selection 17, 11, a page copy 8.1, 4.6, a commit 14, 6.5 (on
// another machine here 11.8, 13.5, 7.1, 8.6); a small one's kernels take 3 to 12.
//
// The rules are attn_native's: GPU tensors on the current device, dtype, shape and contiguity
// checked before anything is launched (TypeError, ValueError), torch's current stream,
// RuntimeError on a status that is not MOE_OK.
#include <c10/hip/HIPStream.h>
#include <torch/extension.h>

#include <initializer_list>
#include <string>
#include <tuple>

#include "../../include/attn_gfx950.h"

namespace {

using at::ScalarType;
using at::Tensor;

constexpr int64_t kHeadDim = 64, kQHeads = 64, kKvHeads = 8, kPage = 16;
constexpr int64_t kBf16PageBytes = 2 * kKvHeads * kPage * kHeadDim * 2;
constexpr int64_t kBeams = 64;
constexpr ScalarType kBf16 = at::kBFloat16, kInt = at::kInt, kFloat = at::kFloat, kByte = at::kByte;

std::string shape_text(at::IntArrayRef shape) {
  std::string s = "(";
  for (size_t i = 0; i < shape.size(); ++i)
    s += (i ? ", " : "") + std::to_string(shape[i]);
  return s + (shape.size() == 1 ? ",)" : ")");
}

struct Call {  // the current device and stream
  c10::hip::HIPStream stream = c10::hip::getCurrentHIPStream();
  void* handle() const { return (void*)stream.stream(); }
};

// a GPU tensor, before the current device is asked for
const Tensor& on_gpu(const Tensor& t, const char* name, ScalarType dtype) {
  if (t.scalar_type() != dtype)
    throw py::type_error(std::string(name) + ": expected dtype torch." +
                         (dtype == kBf16    ? "bfloat16"
                          : dtype == kInt   ? "int32"
                          : dtype == kFloat ? "float32"
                                            : "uint8") +
                         ", got " + c10::toString(t.scalar_type()));
  if (!t.is_cuda())
    throw py::value_error(std::string(name) + ": expected a GPU tensor, got device " +
                          t.device().str());
  return t;
}

void* need(const Call& call, const Tensor& t, const char* name, ScalarType dtype,
           std::initializer_list<int64_t> shape) {
  on_gpu(t, name, dtype);
  if (!t.is_contiguous())
    throw py::value_error(std::string(name) + ": expected a contiguous tensor");
  const at::IntArrayRef want(shape.begin(), shape.size());
  if (t.sizes() != want)
    throw py::value_error(std::string(name) + ": expected shape " + shape_text(want) + ", got " +
                          shape_text(t.sizes()));
  if (t.device().index() != call.stream.device_index())
    throw py::value_error(std::string(name) + ": on " + t.device().str() + ", expected cuda:" +
                          std::to_string(call.stream.device_index()) + ", the current device");
  return t.data_ptr();
}

int64_t rows_of(const Tensor& t, const char* name) {
  if (t.dim() == 0) throw py::value_error(std::string(name) + ": expected rows, got a single value");
  return t.size(0);
}

void check(int rc, const char* what) {
  if (rc != MOE_OK)
    throw std::runtime_error(std::string(what) + " failed: " + moe_status_string(rc) + " (" +
                             std::to_string(rc) + ")");
}

Tensor tree(const Tensor& q, const Tensor& q_indptr, int64_t max_q_len, const Tensor& tree_mask,
            const Tensor& positions, const Tensor& kv_cache, const Tensor& page_indptr,
            const Tensor& page_indices, const Tensor& kv_len, int64_t window, double sm_scale,
            const Tensor& sinks, const Tensor& out, int64_t max_kv_len, bool fp8) {
  const int64_t pages = rows_of(on_gpu(kv_cache, "kv_cache", fp8 ? kByte : kBf16), "kv_cache");
  const Call call;
  void* cache = fp8 ? need(call, kv_cache, "kv_cache", kByte, {pages, ATTN_FP8_PAGE_BYTES})
                    : need(call, kv_cache, "kv_cache", kBf16, {pages, 2, kKvHeads, kPage, kHeadDim});
  const int64_t n = rows_of(q, "q"), batch = rows_of(q_indptr, "q_indptr") - 1;
  const int64_t words = tree_mask.dim() ? tree_mask.size(-1) : 0;
  const auto* qp = (const uint16_t*)need(call, q, "q", kBf16, {n, kQHeads, kHeadDim});
  const auto* qi = (const int32_t*)need(call, q_indptr, "q_indptr", kInt, {batch + 1});
  const auto* mask = (const int32_t*)need(call, tree_mask, "tree_mask", kInt, {n, words});
  const auto* pos = (const int32_t*)need(call, positions, "positions", kInt, {n});
  const auto* pi = (const int32_t*)need(call, page_indptr, "page_indptr", kInt, {batch + 1});
  const auto* ids = (const int32_t*)need(call, page_indices, "page_indices", kInt,
                                         {page_indices.numel()});
  const auto* len = (const int32_t*)need(call, kv_len, "kv_len", kInt, {batch});
  const auto* sk = (const uint16_t*)need(call, sinks, "sinks", kBf16, {kQHeads});
  auto* o = (uint16_t*)need(call, out, "out", kBf16, {n, kQHeads, kHeadDim});
  if (window != (int32_t)window)
    throw py::value_error("window: " + std::to_string(window) + " does not fit 32 bits");
  const size_t bytes =
      attn_tree_workspace_bytes(batch, max_q_len, max_kv_len, (int32_t)window);
  const Tensor ws = bytes ? at::empty({(int64_t)bytes}, q.options().dtype(kByte)) : Tensor();
  check((fp8 ? attn_tree_fp8 : attn_tree)(
            qp, n, qi, batch, max_q_len, mask, words, pos, cache, pages, pi, ids, len, max_kv_len,
            (int32_t)window, (float)sm_scale, sk, o, bytes ? ws.data_ptr() : nullptr, bytes,
            call.handle()),
        fp8 ? "attn_tree_fp8" : "attn_tree");
  return out;
}

// all layers of a cache: [layers, pages, ...]
struct Layers {
  bool fp8;
  int64_t layers, pages;
  void* data;
  Layers(const Tensor& t, Call* call) {
    fp8 = t.scalar_type() == kByte;
    layers = t.dim() > 1 ? t.size(0) : 0;
    pages = t.dim() > 1 ? t.size(1) : 0;
    data = fp8 ? need(*call, t, "kv_cache", kByte, {layers, pages, ATTN_FP8_PAGE_BYTES})
               : need(*call, t, "kv_cache", kBf16, {layers, pages, 2, kKvHeads, kPage, kHeadDim});
  }
};
const Tensor& layers_on_gpu(const Tensor& t) {
  return on_gpu(t, "kv_cache", t.scalar_type() == kByte ? kByte : kBf16);
}

std::tuple<Tensor, Tensor, Tensor> tree_commit(
    const Tensor& kv_cache, const Tensor& page_indptr, const Tensor& page_indices,
    const Tensor& kv_len, const Tensor& q_indptr, int64_t max_q_len, const Tensor& tokens,
    const Tensor& parents, const Tensor& chosen) {
  layers_on_gpu(kv_cache);
  Call call;
  const Layers c(kv_cache, &call);
  const int64_t n = rows_of(tokens, "tokens"), batch = rows_of(q_indptr, "q_indptr") - 1;
  const auto* qi = (const int32_t*)need(call, q_indptr, "q_indptr", kInt, {batch + 1});
  const auto* pi = (const int32_t*)need(call, page_indptr, "page_indptr", kInt, {batch + 1});
  const auto* ids = (const int32_t*)need(call, page_indices, "page_indices", kInt,
                                         {page_indices.numel()});
  const auto* len = (const int32_t*)need(call, kv_len, "kv_len", kInt, {batch});
  const auto* tk = (const int32_t*)need(call, tokens, "tokens", kInt, {n});
  const auto* pa = (const int32_t*)need(call, parents, "parents", kInt, {n});
  const auto* ch = (const int32_t*)need(call, chosen, "chosen", kInt, {n});
  const at::AutoDispatchBelowADInplaceOrView below;  // (of integers: nothing to differentiate)
  const Tensor out = at::empty({n + 2 * batch}, tokens.options());
  auto* p = (int32_t*)out.data_ptr();
  check((c.fp8 ? attn_tree_commit_fp8 : attn_tree_commit)(
            c.data, c.layers, c.pages, pi, ids, len, qi, batch, n, max_q_len, tk, pa, ch, p, p + n,
            p + n + batch, call.handle()),
        c.fp8 ? "attn_tree_commit_fp8" : "attn_tree_commit");
  return {at::as_strided(out, {n}, {1}, 0), at::as_strided(out, {batch}, {1}, n),
          at::as_strided(out, {batch}, {1}, n + batch)};
}

Tensor kv_copy_pages(const Tensor& kv_cache, const Tensor& src_pages, const Tensor& dst_pages) {
  layers_on_gpu(kv_cache);
  Call call;
  const Layers c(kv_cache, &call);
  const int64_t n = rows_of(src_pages, "src_pages");
  const auto* src = (const int32_t*)need(call, src_pages, "src_pages", kInt, {n});
  const auto* dst = (const int32_t*)need(call, dst_pages, "dst_pages", kInt, {n});
  check(attn_kv_copy_pages(c.data, c.layers, c.pages, c.fp8 ? ATTN_FP8_PAGE_BYTES : kBf16PageBytes,
                           src, dst, n, call.handle()),
        "attn_kv_copy_pages");
  return kv_cache;
}

std::tuple<Tensor, Tensor, Tensor> beam_top_k(const Tensor& logits, const Tensor& scores,
                                              int64_t k) {
  const bool f32 = logits.scalar_type() == kFloat;
  on_gpu(logits, "logits", f32 ? kFloat : kBf16);
  const Call call;
  const int64_t batch = scores.dim() == 2 ? scores.size(0) : 0;
  const int64_t width = scores.dim() == 2 ? scores.size(1) : 0;
  const int64_t vocab = logits.dim() ? logits.size(-1) : 0;
  const auto* sc = (const float*)need(call, scores, "scores", kFloat, {batch, width});
  const void* x = need(call, logits, "logits", f32 ? kFloat : kBf16, {batch * width, vocab});
  Tensor moved;  // rows of bf16 from an odd element on: the entry point wants 4-byte words
  if ((uintptr_t)x & 3u) x = (moved = logits.clone()).data_ptr();
  if (k < 1 || k > kBeams || k > width * vocab || width > kBeams)
    throw py::value_error("k: " + std::to_string(k) + " of " + std::to_string(width) +
                          " beams and " + std::to_string(vocab) + " tokens; both up to " +
                          std::to_string(kBeams));
  const size_t bytes = attn_beam_workspace_bytes(batch, width, vocab, k);
  const Tensor ws = at::empty({(int64_t)bytes}, logits.options().dtype(kByte));
  const Tensor values = at::empty({batch, k}, scores.options());
  const Tensor beams = at::empty({batch, k}, scores.options().dtype(kInt));
  const Tensor tokens = at::empty({batch, k}, scores.options().dtype(kInt));
  check(attn_beam_top_k(x, f32, batch, width, vocab, sc, k, (float*)values.data_ptr(),
                        (int32_t*)beams.data_ptr(), (int32_t*)tokens.data_ptr(), ws.data_ptr(),
                        bytes, call.handle()),
        "attn_beam_top_k");
  return {values, beams, tokens};
}

}  // namespace

PYBIND11_MODULE(attn_binding, m) {
  m.def("tree", &tree);
  m.def("tree_commit", &tree_commit);
  m.def("kv_copy_pages", &kv_copy_pages);
  m.def("beam_top_k", &beam_top_k);
}
