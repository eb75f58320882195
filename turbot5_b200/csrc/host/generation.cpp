// Beam search and 8-bit caches: argument checks, outputs and launches, and their Python bindings.
#include "host.h"

#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <cstring>

#include "bindings.h"

namespace t5b_host {
namespace {

constexpr int64_t kMaxBeams = 16;

void check_on(const Tensor& t, at::Device dev, const char* name) {
  require_cuda(t);
  TORCH_CHECK_VALUE(t.device() == dev, name, " is on ", t.device(), ", expected ", dev);
}
// a contiguous tensor of this type and shape on this device
void check_plain(const Tensor& t, at::ScalarType dtype, at::IntArrayRef sizes, at::Device dev, const char* name) {
  TORCH_CHECK_TYPE(t.defined() && t.scalar_type() == dtype, name, " must be a ", c10::toString(dtype), " tensor");
  TORCH_CHECK_VALUE(t.sizes() == sizes, name, " must be of shape ", sizes, ", got ", t.sizes());
  check_on(t, dev, name);
  TORCH_CHECK_VALUE(t.is_contiguous(), name, " must be contiguous");
}
struct Dim { int64_t stride, size; };
// A tensor's dims with more than one index, widest stride first.
std::vector<Dim> dims_of(const Tensor& t) {
  std::vector<Dim> dims;
  for (int64_t d = 0; d < t.dim(); ++d)
    if (t.size(d) > 1) dims.push_back({t.stride(d), t.size(d)});
  std::sort(dims.begin(), dims.end(), [](const Dim& a, const Dim& b) { return a.stride > b.stride; });
  return dims;
}
// Tensors that are written in place: they do not overlap themselves (every stride reaches past what is inside it), have
// no part in gradients, and count the change.
void check_written(const Tensor& t, const char* name, bool grad) {
  int64_t inside = 0;
  bool apart = true;
  if (t.numel() > 0 && !t.is_non_overlapping_and_dense()) {
    const std::vector<Dim> dims = dims_of(t);
    for (size_t i = dims.size(); i-- > 0; inside += (dims[i].size - 1) * dims[i].stride) apart = apart && dims[i].stride > inside;
  }
  TORCH_CHECK_VALUE(apart, name, " is written and must not overlap itself");
  TORCH_CHECK_VALUE(!(grad && t.requires_grad()), name, " is written in place and must not require gradients");
}
void count_change(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
// The bytes from a tensor's first element to its last.
struct Span {
  uintptr_t from = 0, to = 0;
  explicit Span(const Tensor& t) {
    if (t.numel() == 0) return;
    int64_t last = 0;
    for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
    from = (uintptr_t)t.data_ptr(); to = from + (uintptr_t)(last + 1) * t.element_size();
  }
  bool meets(const Span& o) const { return from < o.to && o.from < to; }
};
// Whether two tensors of one shape and one set of strides, `delta` bytes apart, share a byte.  Dim by dim from the widest
// stride: where a dim's stride holds all that is inside it, only two distances of its index can make up for `delta`.
bool share_bytes(int64_t delta, const Dim* dims, size_t n, int64_t es) {
  if (n == 0) return std::abs(delta) < es;
  int64_t q = delta / dims->stride;
  if (q * dims->stride > delta) --q;
  for (int64_t c = q; c <= q + 1; ++c)
    if (std::abs(c) < dims->size && share_bytes(delta - c * dims->stride, dims + 1, n - 1, es)) return true;
  return false;
}
// Of tensors that are alike in shape and strides, with these first bytes: whether two share a byte.
bool any_share_bytes(const Tensor& like, uintptr_t* at, size_t n) {
  std::sort(at, at + n);
  const Span whole(like);
  std::vector<Dim> dims;
  for (size_t i = 0; i < n; ++i)
    for (size_t j = i + 1; j < n && at[j] - at[i] < whole.to - whole.from; ++j) {
      if (dims.empty()) {
        dims = dims_of(like);
        for (Dim& d : dims) d.stride *= like.element_size();
      }
      if (share_bytes((int64_t)(at[j] - at[i]), dims.data(), dims.size(), like.element_size())) return true;
    }
  return false;
}
// `n` lengths on the device
Tensor lengths_arg(PyObject* o, int64_t n, at::Device dev, const char* name) {
  const Tensor t = tensor_arg(o);
  if (!t.defined()) return t;
  TORCH_CHECK_TYPE(t.scalar_type() == at::kInt, name, " must be int32");
  TORCH_CHECK_VALUE(t.numel() == n, name, " must have one entry per row, ", n, ", got ", t.numel());
  check_on(t, dev, name);
  return t.contiguous();
}
int int32_size(int64_t n, const char* name) {
  TORCH_CHECK_VALUE(n >= 0 && n <= INT32_MAX, name, " is too large: ", n);
  return (int)n;
}
int int32_option(int64_t n, const char* name) {
  TORCH_CHECK_VALUE(n >= INT32_MIN && n <= INT32_MAX, name, " does not fit in 32 bits: ", n);
  return (int)n;
}

std::vector<Tensor> tensors_of(PyObject* o, const char* what) {
  std::vector<Tensor> r;
  PyObject* seq = PySequence_Fast(o, what);
  if (!seq) throw python_error();
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq);
  try {
    for (Py_ssize_t i = 0; i < n; ++i) r.push_back(tensor_arg(PySequence_Fast_GET_ITEM(seq, i)));
  } catch (...) {
    Py_DECREF(seq);
    throw;
  }
  Py_DECREF(seq);
  return r;
}

PyObject* tuple_of(const std::vector<Tensor>& ts) {
  PyObject* r = PyTuple_New((Py_ssize_t)ts.size());
  for (size_t i = 0; i < ts.size(); ++i) PyTuple_SET_ITEM(r, (Py_ssize_t)i, wrap(ts[i]));
  return r;
}

// beam_step(logits, scores, finished_scores, finished_steps, finished_beams, done, pos, eos, pad, length_penalty,
//           early_stopping, out, history) -> (tokens, parents, scores, finished_scores, finished_steps, finished_beams, done)
PyObject* py_beam_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 13);
  const bool grad = at::GradMode::is_enabled();
  at::AutoGradMode no_grad(false);
  Tensor logits = tensor_arg(a[0]);
  const Tensor scores = tensor_arg(a[1]);
  require_cuda(logits);
  TORCH_CHECK_TYPE(logits.defined() && scores.defined(), "logits and scores must be tensors");
  const int dtype = dtype_code(logits.scalar_type());
  TORCH_CHECK_VALUE(scores.dim() == 2, "scores must be (batch, num_beams), got ", scores.sizes());
  const int64_t B = scores.size(0), K = scores.size(1);
  TORCH_CHECK_VALUE(K >= 1 && K <= kMaxBeams, "between 1 and ", kMaxBeams, " beams, got ", K);
  TORCH_CHECK_VALUE(logits.dim() >= 2 && logits.size(-1) >= 2, "logits must be (batch * num_beams, vocab) with two tokens at least");
  const int64_t V = logits.size(-1);
  TORCH_CHECK_VALUE(V <= (1 << 27) && logits.numel() == B * K * V, "logits of shape ", logits.sizes(), " do not hold batch * num_beams = ",
                    B * K, " rows of at most 2^27 tokens");
  const at::Device dev = logits.device();
  const at::IntArrayRef bk = scores.sizes();
  const Tensor done = tensor_arg(a[5]), pos = tensor_arg(a[6]);
  const std::array<Tensor, 3> pool = {tensor_arg(a[2]), tensor_arg(a[3]), tensor_arg(a[4])};
  check_plain(scores, at::kFloat, bk, dev, "scores");
  check_plain(pool[0], at::kFloat, bk, dev, "finished_scores");
  check_plain(pool[1], at::kInt, bk, dev, "finished_steps");
  check_plain(pool[2], at::kInt, bk, dev, "finished_beams");
  check_plain(done, at::kBool, {B}, dev, "done");
  TORCH_CHECK_TYPE(pos.defined() && pos.scalar_type() == at::kLong && pos.numel() == 1, "pos must be one int64 on the device");
  check_on(pos, dev, "pos");
  const double length_penalty = float_arg(a[9]);
  TORCH_CHECK_VALUE(std::isfinite(length_penalty), "length_penalty must be finite");
  const at::ScalarType types[7] = {at::kLong, at::kInt, at::kFloat, at::kFloat, at::kInt, at::kInt, at::kBool};
  static const char* const names[7] = {"out[0] (tokens)", "out[1] (parents)", "out[2] (scores)", "out[3] (finished_scores)",
                                       "out[4] (finished_steps)", "out[5] (finished_beams)", "out[6] (done)"};
  std::vector<Tensor> out;
  if (a[11] == Py_None) {
    for (int i = 0; i < 7; ++i) out.push_back(empty_like_dense(i == 6 ? at::IntArrayRef({B}) : bk, types[i], dev));
  } else {
    out = tensors_of(a[11], "out must be a sequence of seven tensors");
    TORCH_CHECK_VALUE(out.size() == 7, "out must hold seven tensors, got ", out.size());
    for (int i = 0; i < 7; ++i) {
      if (i == 6) check_plain(out[i], types[i], {B}, dev, names[i]);
      else check_plain(out[i], types[i], bk, dev, names[i]);
    }
  }
  std::vector<Tensor> history;
  int64_t steps = 0;
  if (a[12] != Py_None) {
    history = tensors_of(a[12], "history must be (tokens, parents)");
    TORCH_CHECK_VALUE(history.size() == 2 && history[0].defined() && history[0].dim() == 3, "history must be two (steps, batch, num_beams) tensors");
    steps = history[0].size(0);
    check_plain(history[0], at::kInt, {steps, B, K}, dev, "history[0] (tokens)");
    check_plain(history[1], at::kInt, {steps, B, K}, dev, "history[1] (parents)");
  }
  if (a[11] != Py_None || !history.empty()) {
    // what is written may be the matching input; it overlaps nothing else
    std::vector<Span> written;
    for (const Tensor& t : out) written.emplace_back(t);
    for (const Tensor& t : history) written.emplace_back(t);
    const Span read[7] = {Span(logits), Span(pos), Span(scores), Span(pool[0]), Span(pool[1]), Span(pool[2]), Span(done)};
    for (size_t i = 0; i < written.size(); ++i)
      for (size_t j = 0; j < i; ++j)
        TORCH_CHECK_VALUE(!written[i].meets(written[j]), "two of the tensors in out and history are the same or overlap");
    for (size_t i = 0; i < written.size(); ++i) {
      for (size_t j = 0; j < 7; ++j)
        TORCH_CHECK_VALUE(!written[i].meets(read[j]) || (i == j && i >= 2 && written[i].from == read[j].from), i < 7 ? names[i] : "history",
                          " overlaps an input that it does not replace");
    }
    for (size_t i = 0; i < written.size(); ++i) {
      const Tensor& t = i < 7 ? out[i] : history[i - 7];
      check_written(t, i < 7 ? names[i] : "history", grad);
      count_change(t);
    }
  }
  if (logits.dim() != 2) logits = logits.reshape({B * K, V});
  if (logits.stride(1) != 1) logits = logits.contiguous();
  t5b_beam_step_args g;
  g.logits = logits.data_ptr(); g.scores = (const float*)scores.data_ptr();
  g.finished_scores = (const float*)pool[0].data_ptr(); g.finished_steps = (const int32_t*)pool[1].data_ptr();
  g.finished_beams = (const int32_t*)pool[2].data_ptr(); g.done = (const uint8_t*)done.data_ptr();
  g.pos = (const int64_t*)pos.data_ptr();
  g.tokens_out = (int64_t*)out[0].data_ptr(); g.parents_out = (int32_t*)out[1].data_ptr(); g.scores_out = (float*)out[2].data_ptr();
  g.finished_scores_out = (float*)out[3].data_ptr(); g.finished_steps_out = (int32_t*)out[4].data_ptr();
  g.finished_beams_out = (int32_t*)out[5].data_ptr(); g.done_out = (uint8_t*)out[6].data_ptr();
  g.history_tokens = history.empty() ? nullptr : (int32_t*)history[0].data_ptr();
  g.history_parents = history.empty() ? nullptr : (int32_t*)history[1].data_ptr();
  g.logits_stride = logits.stride(0); g.history_steps = steps;
  g.eos_token_id = a[7] == Py_None ? -1 : int_arg(a[7]);
  g.pad_token_id = int_arg(a[8]);
  g.length_penalty = length_penalty;
  g.dtype = dtype; g.B = int32_size(B, "the batch"); g.num_beams = (int32_t)K; g.vocab = (int32_t)V;
  g.early_stopping = bool_arg(a[10]);
  const c10::cuda::CUDAGuard guard(dev);
  check_status(t5b_beam_search_step(&g, stream_of(dev)), "beam_search_step");
  return tuple_of(out);
  END_HANDLE_TH_ERRORS
}

// beam_sequences(tokens, parents, scores, finished_scores, finished_steps, finished_beams, done, num_return, eos, pad,
//                length_penalty) -> (sequences, scores)
PyObject* py_beam_sequences(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 11);
  at::AutoGradMode no_grad(false);
  const Tensor tokens = tensor_arg(a[0]), parents = tensor_arg(a[1]), scores = tensor_arg(a[2]);
  TORCH_CHECK_TYPE(tokens.defined() && scores.defined(), "tokens and scores must be tensors");
  require_cuda(tokens);
  TORCH_CHECK_VALUE(tokens.dim() == 3 && tokens.size(0) >= 1, "tokens must be (steps, batch, num_beams) with a step at least, got ", tokens.sizes());
  const int64_t T = tokens.size(0), B = tokens.size(1), K = tokens.size(2);
  TORCH_CHECK_VALUE(K >= 1 && K <= kMaxBeams, "between 1 and ", kMaxBeams, " beams, got ", K);
  const at::Device dev = tokens.device();
  check_plain(tokens, at::kInt, {T, B, K}, dev, "tokens");
  check_plain(parents, at::kInt, {T, B, K}, dev, "parents");
  const std::array<Tensor, 3> pool = {tensor_arg(a[3]), tensor_arg(a[4]), tensor_arg(a[5])};
  const Tensor done = tensor_arg(a[6]);
  check_plain(scores, at::kFloat, {B, K}, dev, "scores");
  check_plain(pool[0], at::kFloat, {B, K}, dev, "finished_scores");
  check_plain(pool[1], at::kInt, {B, K}, dev, "finished_steps");
  check_plain(pool[2], at::kInt, {B, K}, dev, "finished_beams");
  check_plain(done, at::kBool, {B}, dev, "done");
  const int64_t R = int_arg(a[7]);
  TORCH_CHECK_VALUE(R >= 1 && R <= K, "num_return_sequences must be between 1 and num_beams = ", K, ", got ", R);
  const double length_penalty = float_arg(a[10]);
  TORCH_CHECK_VALUE(std::isfinite(length_penalty), "length_penalty must be finite");
  const Tensor out = empty_like_dense({B, R, T}, at::kLong, dev), out_scores = empty_like_dense({B, R}, at::kFloat, dev);
  t5b_beam_sequences_args g;
  g.tokens = (const int32_t*)tokens.data_ptr(); g.parents = (const int32_t*)parents.data_ptr();
  g.scores = (const float*)scores.data_ptr(); g.finished_scores = (const float*)pool[0].data_ptr();
  g.finished_steps = (const int32_t*)pool[1].data_ptr(); g.finished_beams = (const int32_t*)pool[2].data_ptr();
  g.done = (const uint8_t*)done.data_ptr();
  g.sequences = (int64_t*)out.data_ptr(); g.sequence_scores = (float*)out_scores.data_ptr();
  g.eos_token_id = a[8] == Py_None ? -1 : int_arg(a[8]); g.pad_token_id = int_arg(a[9]);
  g.length_penalty = length_penalty;
  g.steps = int32_size(T, "the number of steps"); g.B = int32_size(B, "the batch"); g.num_beams = (int32_t)K; g.num_return = (int32_t)R;
  const c10::cuda::CUDAGuard guard(dev);
  check_status(t5b_beam_search_sequences(&g, stream_of(dev)), "beam_search_sequences");
  return wrap2(out, out_scores);
  END_HANDLE_TH_ERRORS
}

// A group of equal tensors whose rows are reordered together: dims (outer,) rows, heads, then `tail` contiguous dims.
struct Rows { int64_t outer = 1, outer_stride = 0, row_stride = 0, head_stride = 0; };
Rows rows_of(const std::vector<Tensor>& ts, int64_t dims, int64_t R, at::Device dev, const char* name, bool grad) {
  Rows r;
  const Tensor& t0 = ts[0];
  TORCH_CHECK_VALUE(t0.defined() && (t0.dim() == dims || t0.dim() == dims + 1), name, " must have ", dims, " or ", dims + 1, " dimensions");
  const int64_t d = t0.dim() - dims, es = t0.element_size();
  TORCH_CHECK_VALUE(t0.size(d) == R, name, " must have batch * num_beams = ", R, " rows, got ", t0.size(d));
  TORCH_CHECK_VALUE(t0.numel() == 0 || ((t0.size(-1) == 1 || t0.stride(-1) == 1) &&
                                        (dims == 3 || t0.size(-2) == 1 || t0.stride(-2) == t0.size(-1))),
                    name, ": a head's tokens must lie one behind the other");
  if (d == 1) { r.outer = t0.size(0); r.outer_stride = t0.stride(0) * es; }
  r.row_stride = t0.stride(d) * es; r.head_stride = t0.stride(d + 1) * es;
  for (const Tensor& t : ts) {
    TORCH_CHECK_VALUE(t.defined() && t.sizes() == t0.sizes() && t.strides() == t0.strides() && t.scalar_type() == t0.scalar_type(),
                      name, " must be alike in shape, strides and type");
    check_on(t, dev, name);
    check_written(t, name, grad);
  }
  std::vector<uintptr_t> at;
  for (const Tensor& t : ts) at.push_back((uintptr_t)t.data_ptr());
  TORCH_CHECK_VALUE(!any_share_bytes(t0, at.data(), at.size()), name, ": the same tensor twice, or two that overlap");
  return r;
}

// reorder_caches(caches, parents, seqlens, scales)
PyObject* py_reorder_caches(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 4);
  const bool grad = at::GradMode::is_enabled();
  at::AutoGradMode no_grad(false);
  const std::vector<Tensor> caches = tensors_of(a[0], "caches must be a sequence of tensors");
  const std::vector<Tensor> scales = tensors_of(a[3], "scales must be a sequence of tensors");
  const Tensor parents = tensor_arg(a[1]);
  TORCH_CHECK_TYPE(parents.defined(), "parents must be a tensor");
  require_cuda(parents);
  TORCH_CHECK_VALUE(parents.dim() == 2, "parents must be (batch, num_beams), got ", parents.sizes());
  const int64_t B = parents.size(0), K = parents.size(1), R = B * K;
  TORCH_CHECK_VALUE(K >= 1 && K <= kMaxBeams, "between 1 and ", kMaxBeams, " beams, got ", K);
  const at::Device dev = parents.device();
  check_plain(parents, at::kInt, {B, K}, dev, "parents");
  const Tensor seqlens = lengths_arg(a[2], R, dev, "seqlens");
  if (caches.empty()) {
    TORCH_CHECK_VALUE(scales.empty(), "scales belong to caches");
    Py_RETURN_NONE;
  }
  const Rows c = rows_of(caches, 4, R, dev, "caches", grad);
  const int64_t H = caches[0].size(-3), cap = caches[0].size(-2);
  Rows s;
  if (!scales.empty()) {
    s = rows_of(scales, 3, R, dev, "scales", grad);
    TORCH_CHECK_TYPE(scales[0].scalar_type() == at::kFloat, "scales must be float32");
    TORCH_CHECK_VALUE(scales.size() == caches.size() && scales[0].dim() + 1 == caches[0].dim() && s.outer == c.outer &&
                          scales[0].size(-2) == H && scales[0].size(-1) == (cap + T5B_CACHE_BLOCK - 1) / T5B_CACHE_BLOCK,
                      "scales of shape ", scales[0].sizes(), " do not belong to caches of shape ", caches[0].sizes());
  }
  if (caches[0].numel() == 0) Py_RETURN_NONE;
  for (const Tensor& t : caches) count_change(t);
  for (const Tensor& t : scales) count_change(t);
  t5b_cache_reorder_args g;
  g.parents = (const int32_t*)parents.data_ptr(); g.seqlens = (const int32_t*)ptr(seqlens);
  g.cache_stride_outer = c.outer_stride; g.cache_stride_row = c.row_stride; g.cache_stride_head = c.head_stride;
  g.scale_stride_outer = s.outer_stride; g.scale_stride_row = s.row_stride; g.scale_stride_head = s.head_stride;
  g.outer = int32_size(c.outer, "caches"); g.B = int32_size(B, "the batch"); g.num_beams = (int32_t)K; g.H = int32_size(H, "the heads");
  g.capacity = int32_size(cap, "the capacity");
  g.token_bytes = int32_size(caches[0].size(-1) * caches[0].element_size(), "a token");
  const c10::cuda::CUDAGuard guard(dev);
  for (size_t i = 0; i < caches.size(); i += T5B_REORDER_MAX_TENSORS) {
    const size_t count = std::min<size_t>(T5B_REORDER_MAX_TENSORS, caches.size() - i);
    g.n_caches = (int32_t)count; g.n_scales = scales.empty() ? 0 : (int32_t)count;
    for (size_t j = 0; j < count; ++j) {
      g.caches[j] = caches[i + j].data_ptr();
      if (!scales.empty()) g.scales[j] = scales[i + j].data_ptr();
    }
    check_status(t5b_beam_cache_reorder(&g, stream_of(dev)), "reorder_beam_cache");
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// an 8-bit cache (B, H, capacity, D) and its scales (B, H, capacity / 64)
void check_cache(const Tensor& cache, const Tensor& scale, int64_t B, int64_t H, int64_t D, at::Device dev, const char* name) {
  TORCH_CHECK_TYPE(cache.defined() && cache.scalar_type() == at::kFloat8_e4m3fn, name, " must be a float8_e4m3fn tensor");
  TORCH_CHECK_VALUE(cache.dim() == 4 && cache.size(0) == B && cache.size(1) == H && cache.size(3) == D, name, " must be (", B, ", ", H,
                    ", capacity, ", D, "), got ", cache.sizes());
  const int64_t cap = cache.size(2);
  TORCH_CHECK_VALUE(cap % T5B_CACHE_BLOCK == 0, name, ": the capacity must be a multiple of ", T5B_CACHE_BLOCK, ", got ", cap);
  TORCH_CHECK_TYPE(scale.defined() && scale.scalar_type() == at::kFloat, "the scales of ", name, " must be float32");
  TORCH_CHECK_VALUE(scale.sizes() == at::IntArrayRef({B, H, cap / T5B_CACHE_BLOCK}), "the scales of ", name, " must be of shape (", B, ", ", H, ", ",
                    cap / T5B_CACHE_BLOCK, "), got ", scale.sizes());
  check_on(cache, dev, name); check_on(scale, dev, name);
  TORCH_CHECK_VALUE(cache.numel() == 0 || (cache.stride(3) == 1 && cache.stride(2) == D), name, ": a head's tokens must lie one behind the other");
  TORCH_CHECK_VALUE(scale.numel() == 0 || scale.size(2) == 1 || scale.stride(2) == 1, "the scales of ", name, " must be contiguous in their last dimension");
}

// cache_quantize(k, v, k_cache, k_scale, v_cache, v_scale, start, seqlens)
PyObject* py_cache_quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 8);
  const bool grad = at::GradMode::is_enabled();
  at::AutoGradMode no_grad(false);
  Tensor k = tensor_arg(a[0]), v = tensor_arg(a[1]);
  const Tensor kc = tensor_arg(a[2]), ks = tensor_arg(a[3]), vc = tensor_arg(a[4]), vs = tensor_arg(a[5]);
  TORCH_CHECK_TYPE(k.defined() && v.defined(), "k and v must be tensors");
  require_cuda(k); require_cuda(v);
  TORCH_CHECK_TYPE(k.scalar_type() == v.scalar_type(), "k and v must share a dtype");
  const int dtype = dtype_code(k.scalar_type());
  TORCH_CHECK_VALUE(k.dim() == 4 && v.sizes() == k.sizes(), "k and v must be (B, H, M, D) of one shape");
  const int64_t B = k.size(0), H = k.size(1), M = k.size(2), D = k.size(3);
  TORCH_CHECK_VALUE(D == 16 || D == 32 || D == 64 || D == 128, "head dim must be 16, 32, 64 or 128");
  const at::Device dev = k.device();
  check_on(v, dev, "v");
  check_cache(kc, ks, B, H, D, dev, "k_cache"); check_cache(vc, vs, B, H, D, dev, "v_cache");
  for (const Tensor* t : {&kc, &vc, &ks, &vs}) check_written(*t, "the cache", grad);
  TORCH_CHECK_VALUE(kc.sizes() == vc.sizes() && kc.strides() == vc.strides() && ks.strides() == vs.strides(), "k_cache and v_cache must be alike in shape and strides");
  uintptr_t caches[2] = {(uintptr_t)kc.data_ptr(), (uintptr_t)vc.data_ptr()}, scales[2] = {(uintptr_t)ks.data_ptr(), (uintptr_t)vs.data_ptr()};
  TORCH_CHECK_VALUE(!any_share_bytes(kc, caches, 2) && !any_share_bytes(ks, scales, 2), "keys and values need caches of their own");
  const int64_t cap = kc.size(2);
  t5b_cache_quantize_args g;
  g.start_ptr = nullptr; g.start = 0;
  Tensor start;
  if (THPVariable_Check(a[6])) {
    start = tensor_arg(a[6]);
    TORCH_CHECK_TYPE(start.scalar_type() == at::kLong && start.numel() == 1, "start must be a whole number or one int64 on the device");
    check_on(start, dev, "start");
    g.start_ptr = (const int64_t*)start.data_ptr();
  } else {
    g.start = int_arg(a[6]);
    TORCH_CHECK_VALUE(g.start >= 0 && g.start <= cap && M <= cap - g.start, "tokens ", g.start, " to ", g.start + M, " do not fit in a cache of ", cap);
  }
  const Tensor seqlens = lengths_arg(a[7], B, dev, "seqlens");
  for (const Tensor* t : {&kc, &vc, &ks, &vs}) count_change(*t);
  k = unit_stride_last(k); v = unit_stride_last(v);
  g.k = k.data_ptr(); g.v = v.data_ptr(); g.k_cache = kc.data_ptr(); g.v_cache = vc.data_ptr();
  g.k_scale = (float*)ks.data_ptr(); g.v_scale = (float*)vs.data_ptr();
  g.seqlens = (const int32_t*)ptr(seqlens);
  g.k_stride_b = k.stride(0); g.k_stride_h = k.stride(1); g.k_stride_m = k.stride(2);
  g.v_stride_b = v.stride(0); g.v_stride_h = v.stride(1); g.v_stride_m = v.stride(2);
  g.cache_stride_b = kc.stride(0); g.cache_stride_h = kc.stride(1); g.scale_stride_b = ks.stride(0); g.scale_stride_h = ks.stride(1);
  g.dtype = dtype; g.B = int32_size(B, "the batch"); g.H = int32_size(H, "the heads"); g.M = int32_size(M, "the number of tokens");
  g.D = (int32_t)D; g.capacity = int32_size(cap, "the capacity");
  const c10::cuda::CUDAGuard guard(dev);
  check_status(t5b_cache_quantize(&g, stream_of(dev)), "quantize_into_cache");
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// decode_quantized(q, k, k_scale, v, v_scale, bias, causal, sm_scale, nb, md, kv_len, seqlens_k, q_pos_offset)
PyObject* py_decode_quantized(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 13);
  at::AutoGradMode no_grad(false);
  Tensor q = tensor_arg(a[0]), bias = tensor_arg(a[5]);
  const Tensor k = tensor_arg(a[1]), ks = tensor_arg(a[2]), v = tensor_arg(a[3]), vs = tensor_arg(a[4]);
  TORCH_CHECK_TYPE(q.defined(), "q must be a tensor");
  require_cuda(q);
  TORCH_CHECK_TYPE(is_half_type(q.scalar_type()), "queries of an 8-bit cache are float16 or bfloat16, got ", c10::toString(q.scalar_type()));
  TORCH_CHECK_VALUE(q.dim() == 4, "q must be (B, H, M, D)");
  const int64_t B = q.size(0), H = q.size(1), M = q.size(2), D = q.size(3);
  TORCH_CHECK_VALUE(D == 16 || D == 32 || D == 64 || D == 128, "head dim must be 16, 32, 64 or 128");
  const at::Device dev = q.device();
  check_cache(k, ks, B, H, D, dev, "k"); check_cache(v, vs, B, H, D, dev, "v");
  const int64_t cap = k.size(2);
  TORCH_CHECK_VALUE(v.size(2) == cap, "k and v must have one capacity");
  const int64_t N = opt_int(a[10]).value_or(cap);
  TORCH_CHECK_VALUE(N >= 0 && N <= cap, "kv_len exceeds the cache capacity");
  const Tensor seqlens = lengths_arg(a[11], B, dev, "seqlens_k");
  t5b_decode_quantized_args g;
  g.num_buckets = int32_option(int_arg(a[8]), "NUM_BUCKETS"); g.max_distance = int32_option(int_arg(a[9]), "MAX_DISTANCE");
  g.table = nullptr; g.table_dtype = T5B_F32; g.table_stride0 = 0;
  if (bias.defined()) {
    check_on(bias, dev, "the bias table");
    TORCH_CHECK_VALUE(bias.dim() == 2 && bias.size(1) == H && bias.size(0) >= g.num_buckets, "bias table must be [NUM_BUCKETS, ", H, "], got ", bias.sizes());
    if (bias.stride(1) != 1) bias = bias.contiguous();
    g.table = bias.data_ptr(); g.table_dtype = dtype_code(bias.scalar_type()); g.table_stride0 = bias.stride(0);
  }
  q = unit_stride_last(q);
  // q as a view of token-major rows: the result in the same order, so that merging the heads is free
  const bool by_tokens = M > 1 && q.stride(1) == D && q.stride(2) >= H * D;
  const Tensor out = by_tokens ? empty_strided({B, H, M, D}, {M * H * D, D, H * D, 1}, q.scalar_type(), dev)
                               : empty_like_dense({B, H, M, D}, q.scalar_type(), dev);
  g.q = q.data_ptr(); g.k = k.data_ptr(); g.v = v.data_ptr(); g.k_scale = (const float*)ks.data_ptr(); g.v_scale = (const float*)vs.data_ptr();
  g.out = out.data_ptr(); g.seqlens_k = (const int32_t*)ptr(seqlens);
  g.q_stride_b = q.stride(0); g.q_stride_h = q.stride(1); g.q_stride_m = q.stride(2);
  g.k_stride_b = k.stride(0); g.k_stride_h = k.stride(1); g.v_stride_b = v.stride(0); g.v_stride_h = v.stride(1);
  g.k_scale_stride_b = ks.stride(0); g.k_scale_stride_h = ks.stride(1); g.v_scale_stride_b = vs.stride(0); g.v_scale_stride_h = vs.stride(1);
  g.o_stride_b = out.stride(0); g.o_stride_h = out.stride(1); g.o_stride_m = out.stride(2);
  g.dtype = dtype_code(q.scalar_type());
  g.B = int32_size(B, "the batch"); g.H = int32_size(H, "the heads"); g.M = int32_size(M, "the rows"); g.N = int32_size(N, "the capacity");
  g.D = (int32_t)D; g.causal = bool_arg(a[6]);
  const int64_t offset = opt_int(a[12]).value_or(-1);
  g.q_pos_offset = int32_option(offset, "q_pos_offset");
  g.sm_scale = (float)(a[7] == Py_None ? 1.0 / std::sqrt((double)D) : float_arg(a[7]));
  const c10::cuda::CUDAGuard guard(dev);
  check_status(t5b_decode_quantized_fwd(&g, stream_of(dev)), "flash_decoding_quantized_with_fusing_bias");
  return wrap(out);
  END_HANDLE_TH_ERRORS
}

}  // namespace

PyMethodDef generation_methods[] = {
    T5B_METHOD("beam_step", py_beam_step), T5B_METHOD("beam_sequences", py_beam_sequences),
    T5B_METHOD("reorder_caches", py_reorder_caches), T5B_METHOD("cache_quantize", py_cache_quantize),
    T5B_METHOD("decode_quantized", py_decode_quantized), {nullptr, nullptr, 0, nullptr}};

}  // namespace t5b_host
