// torch.ops.d2sd.* — torch operators over the C ABI of libd2sd.so
// (include/d2sd.h), for the calls the reference's verify path makes:
//
//   single_prefill_with_kv_cache  flashinfer.single_prefill_with_kv_cache
//                                 (generation/verification.py:145, 159;
//                                  model/cascade_graph.py:54; model/dflash.py:112, 127)
//   merge_state_in_place          flashinfer.merge_state_in_place
//                                 (generation/verification.py:163;
//                                  model/cascade_graph.py:58; model/dflash.py:131)
//   local_attention_merge         the per-row local attention + merge loop that
//                                 CascadeGraphRunner captures (model/cascade_graph.py:52-60)
//   cascade_run / cascade_run_no_alloc
//                                 one cascade verify call of a d2sd_cascade_plan
//                                 (generation/verification.py:127-176 over a token tree)
//   rotary_embedding, cache_write, cache_append, cache_read(_out), chunk_attention(_out)
//                                 the paged-cache operators: d2sd_rotary_embedding,
//                                 d2sd_cache_write / _append / _read, d2sd_chunk_run
//
// Each operator checks its tensors, then calls the C entry point on the
// current HIP stream of the tensors' device; there is no other code path.
// Meta kernels give shapes for tracing (torch.compile / fake tensors).  The
// dispatch key named CUDA is where torch registers its GPU (here HIP) device.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPCachingAllocator.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>
#include <torch/library.h>

#include <cmath>
#include <cstring>
#include <initializer_list>

#include "d2sd.h"

namespace {

d2sd_stream_t current_stream() { return (d2sd_stream_t)c10::hip::getCurrentHIPStream().stream(); }

void check(int rc, const char* what) { TORCH_CHECK(rc == D2SD_OK, what, " failed: ", d2sd_last_error()); }

void need_device(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), "d2sd: ", name, " must be a ROCm device tensor");
}

void need_rows(const at::Tensor& t, const char* name, at::ScalarType dt) {
  need_device(t, name);
  TORCH_CHECK(t.scalar_type() == dt, "d2sd: ", name, " must be ", dt, ", got ", t.scalar_type());
  TORCH_CHECK(t.dim() == 3 && t.stride(2) == 1, "d2sd: ", name, " must be 3-D with a contiguous last dimension");
}

const void* ptr_or_null(const c10::optional<at::Tensor>& t) { return t.has_value() ? t->data_ptr() : nullptr; }

// ---- single_prefill_with_kv_cache ----
std::tuple<at::Tensor, at::Tensor> single_prefill(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                                  bool causal, c10::string_view kv_layout,
                                                  c10::optional<double> sm_scale, bool lse_base2) {
  need_rows(q, "q", at::kBFloat16);
  need_rows(k, "k", at::kBFloat16);
  need_rows(v, "v", at::kBFloat16);
  TORCH_CHECK(k.sizes() == v.sizes() && k.strides() == v.strides(), "d2sd: k and v must share shape and strides");
  const bool hnd = kv_layout == "HND";
  TORCH_CHECK(hnd || kv_layout == "NHD", "d2sd: kv_layout must be 'NHD' or 'HND'");
  const int64_t qo_len = q.size(0), hq = q.size(1), d = q.size(2);
  const int64_t kv_len = hnd ? k.size(1) : k.size(0), hkv = hnd ? k.size(0) : k.size(1);
  TORCH_CHECK(k.size(2) == d, "d2sd: q and k head_dim differ");
  const int64_t s_n = hnd ? k.stride(1) : k.stride(0), s_h = hnd ? k.stride(0) : k.stride(1);
  const float scale = (float)(sm_scale.has_value() ? *sm_scale : 1.0 / std::sqrt((double)d));
  const c10::DeviceGuard guard(q.device());
  at::Tensor out = at::empty(q.sizes(), q.options());
  at::Tensor lse = at::empty({qo_len, hq}, q.options().dtype(at::kFloat));
  const size_t ws = d2sd_single_prefill_workspace_size((int)qo_len, (int)kv_len, (int)hq, (int)hkv, (int)d, -1);
  at::Tensor work = at::empty({(int64_t)std::max<size_t>(ws, 1)}, q.options().dtype(at::kByte));
  check(d2sd_single_prefill_with_kv_cache(q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), v.data_ptr(), s_n,
                                          s_h, out.data_ptr(), out.stride(0), out.stride(1), lse.data_ptr<float>(),
                                          (int)qo_len, (int)kv_len, (int)hq, (int)hkv, (int)d, causal ? 1 : 0, -1,
                                          scale, lse_base2 ? 1 : 0, work.data_ptr(), (size_t)work.numel(),
                                          current_stream()),
        "d2sd.single_prefill_with_kv_cache");
  return {out, lse};
}

std::tuple<at::Tensor, at::Tensor> single_prefill_meta(const at::Tensor& q, const at::Tensor&, const at::Tensor&, bool,
                                                       c10::string_view, c10::optional<double>, bool) {
  return {at::empty_like(q), at::empty({q.size(0), q.size(1)}, q.options().dtype(at::kFloat))};
}

// ---- merge_state_in_place ----
void merge_state_in_place(at::Tensor& v, at::Tensor& s, const at::Tensor& v_other, const at::Tensor& s_other,
                          bool lse_base2) {
  need_rows(v, "v", at::kBFloat16);
  need_rows(v_other, "v_other", at::kBFloat16);
  need_device(s, "s");
  need_device(s_other, "s_other");
  TORCH_CHECK(v.sizes() == v_other.sizes(), "d2sd: v and v_other shapes differ");
  TORCH_CHECK(s.scalar_type() == at::kFloat && s_other.scalar_type() == at::kFloat, "d2sd: s, s_other must be float32");
  TORCH_CHECK(s.dim() == 2 && s.size(0) == v.size(0) && s.size(1) == v.size(1) && s_other.sizes() == s.sizes(),
              "d2sd: s / s_other must be [n, heads]");
  TORCH_CHECK(s.stride(1) == 1 && s_other.stride(1) == 1, "d2sd: s / s_other need a contiguous head dimension");
  const c10::DeviceGuard guard(v.device());
  check(d2sd_merge_state_in_place(v.data_ptr(), v.stride(0), v.stride(1), s.data_ptr<float>(), s.stride(0),
                                  v_other.data_ptr(), v_other.stride(0), v_other.stride(1), s_other.data_ptr<float>(),
                                  s_other.stride(0), (int)v.size(0), (int)v.size(1), (int)v.size(2),
                                  lse_base2 ? 1 : 0, current_stream()),
        "d2sd.merge_state_in_place");
}

void merge_state_meta(at::Tensor&, at::Tensor&, const at::Tensor&, const at::Tensor&, bool) {}

// ---- local_attention_merge ----
void local_attention_merge(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, at::Tensor& out,
                           at::Tensor& lse, bool causal, double sm_scale, const c10::optional<at::Tensor>& sinks,
                           bool lse_base2) {
  for (auto* t : {&q, &k, &v, (const at::Tensor*)&out}) {
    need_device(*t, "q/k/v/out");
    TORCH_CHECK(t->scalar_type() == at::kBFloat16 && t->dim() == 4 && t->stride(3) == 1,
                "d2sd: q/k/v/out must be bf16 [bsz, Lb, heads, D] with a contiguous head_dim");
  }
  TORCH_CHECK(out.sizes() == q.sizes() && k.sizes() == v.sizes() && k.strides() == v.strides(),
              "d2sd: out must match q, v must match k");
  TORCH_CHECK(lse.scalar_type() == at::kFloat && lse.dim() == 3 && lse.size(0) == q.size(0) &&
                  lse.size(1) == q.size(1) && lse.size(2) == q.size(2) && lse.stride(2) == 1,
              "d2sd: lse must be float32 [bsz, Lb, Hq] with contiguous heads");
  if (sinks.has_value())
    TORCH_CHECK(sinks->scalar_type() == at::kFloat && sinks->numel() == q.size(2) && sinks->is_contiguous(),
                "d2sd: sinks must be a contiguous float32 [Hq]");
  const c10::DeviceGuard guard(q.device());
  check(d2sd_local_attention_merge(q.data_ptr(), q.stride(0), q.stride(1), q.stride(2), k.data_ptr(), v.data_ptr(),
                                   k.stride(0), k.stride(1), k.stride(2), out.data_ptr(), out.stride(0), out.stride(1),
                                   out.stride(2), lse.data_ptr<float>(), lse.stride(0), lse.stride(1), (int)q.size(0),
                                   (int)q.size(1), (int)q.size(2), (int)k.size(2), (int)q.size(3), causal ? 1 : 0,
                                   (float)sm_scale, sinks.has_value() ? sinks->data_ptr<float>() : nullptr,
                                   lse_base2 ? 1 : 0, current_stream()),
        "d2sd.local_attention_merge");
}

void local_attention_merge_meta(const at::Tensor&, const at::Tensor&, const at::Tensor&, at::Tensor&, at::Tensor&,
                                bool, double, const c10::optional<at::Tensor>&, bool) {}

// ---- cascade_run ----
// info: the d2sd_cascade_plan_info bytes plan() produced (CPU uint8 tensor);
// prefix: the prefix strides / extent in elements, as run() passes them.
void cascade(bool no_alloc, const at::Tensor& info, const at::Tensor& plan, const at::Tensor& workspace,
             const at::Tensor& q, const at::Tensor& k_suffix, const at::Tensor& v_suffix,
             const c10::optional<at::Tensor>& k_prefix, const c10::optional<at::Tensor>& v_prefix,
             at::IntArrayRef prefix, const c10::optional<at::Tensor>& page_table,
             const c10::optional<at::Tensor>& tree_mask, int64_t mask_mode, int64_t mask_words,
             const c10::optional<at::Tensor>& prefix_len, const c10::optional<at::Tensor>& k_scale,
             const c10::optional<at::Tensor>& v_scale, const c10::optional<at::Tensor>& sinks, double sm_scale,
             bool lse_base2, at::Tensor& out, at::Tensor& lse, const c10::optional<at::Tensor>& k_prefix2,
             const c10::optional<at::Tensor>& v_prefix2, at::IntArrayRef prefix2,
             const c10::optional<at::Tensor>& k2_scale, const c10::optional<at::Tensor>& v2_scale) {
  TORCH_CHECK(info.device().is_cpu() && info.scalar_type() == at::kByte && info.is_contiguous() &&
                  (size_t)info.numel() == sizeof(d2sd_cascade_plan_info),
              "d2sd: info must hold the bytes of a d2sd_cascade_plan_info");
  TORCH_CHECK(prefix.size() == 4, "d2sd: prefix = (stride_tok, stride_head, stride_page, extent)");
  need_rows(q, "q", at::kBFloat16);
  need_rows(k_suffix, "k_suffix", at::kBFloat16);
  need_rows(v_suffix, "v_suffix", at::kBFloat16);
  need_rows(out, "out", at::kBFloat16);
  need_device(plan, "plan");
  need_device(lse, "lse");
  TORCH_CHECK(lse.scalar_type() == at::kFloat && lse.dim() == 2 && lse.stride(1) == 1,
              "d2sd: lse must be float32 [total_q, Hq] with contiguous heads");
  TORCH_CHECK(plan.scalar_type() == at::kInt && plan.is_contiguous(), "d2sd: plan must be a contiguous int32 tensor");
  d2sd_cascade_plan_info pi;
  std::memcpy(&pi, info.data_ptr(), sizeof(pi));
  TORCH_CHECK(plan.numel() >= pi.plan_ints, "d2sd: plan holds fewer entries than info.plan_ints");
  d2sd_cascade_run_args a;
  std::memset(&a, 0, sizeof(a));
  a.plan = plan.data_ptr<int32_t>();
  a.q = q.data_ptr();
  a.q_stride_n = q.stride(0);
  a.q_stride_h = q.stride(1);
  a.k_suffix = k_suffix.data_ptr();
  a.v_suffix = v_suffix.data_ptr();
  a.suffix_stride_n = k_suffix.stride(0);
  a.suffix_stride_h = k_suffix.stride(1);
  a.mask_mode = (int)mask_mode;
  a.mask_words = (int)mask_words;
  a.tree_mask = (const uint64_t*)ptr_or_null(tree_mask);
  a.k_prefix = ptr_or_null(k_prefix);
  a.v_prefix = ptr_or_null(v_prefix);
  a.prefix_stride_tok = prefix[0];
  a.prefix_stride_head = prefix[1];
  a.prefix_stride_page = prefix[2];
  a.prefix_extent = prefix[3];
  a.page_size = pi.page_size;
  a.page_table = (const int32_t*)ptr_or_null(page_table);
  a.prefix_len = (const int32_t*)ptr_or_null(prefix_len);
  a.k_scale = (const float*)ptr_or_null(k_scale);
  a.v_scale = (const float*)ptr_or_null(v_scale);
  a.sinks = (const float*)ptr_or_null(sinks);
  a.out = out.data_ptr();
  a.o_stride_n = out.stride(0);
  a.o_stride_h = out.stride(1);
  a.lse = lse.data_ptr<float>();
  a.lse_stride_n = lse.stride(0);
  a.sm_scale = (float)sm_scale;
  a.lse_base2 = lse_base2 ? 1 : 0;
  if (k_prefix2.has_value()) {
    TORCH_CHECK(prefix2.size() == 3, "d2sd: prefix2 = (stride_tok, stride_head, extent)");
    a.k_prefix2 = k_prefix2->data_ptr();
    a.v_prefix2 = ptr_or_null(v_prefix2);
    a.prefix2_stride_tok = prefix2[0];
    a.prefix2_stride_head = prefix2[1];
    a.prefix2_extent = prefix2[2];
    a.k2_scale = (const float*)ptr_or_null(k2_scale);
    a.v2_scale = (const float*)ptr_or_null(v2_scale);
  }
  if (!no_alloc) {
    need_device(workspace, "workspace");
    a.workspace = workspace.data_ptr();
    a.workspace_bytes = (size_t)workspace.nbytes();
  }
  const c10::DeviceGuard guard(q.device());
  check(no_alloc ? d2sd_cascade_run_noalloc(&pi, &a, current_stream()) : d2sd_cascade_run(&pi, &a, current_stream()),
        no_alloc ? "d2sd.cascade_run_no_alloc" : "d2sd.cascade_run");
}

#define CASCADE_ARGS                                                                                                 \
  const at::Tensor &info, const at::Tensor &plan, const at::Tensor &workspace, const at::Tensor &q,                 \
      const at::Tensor &k_suffix, const at::Tensor &v_suffix, const c10::optional<at::Tensor>&k_prefix,              \
      const c10::optional<at::Tensor>&v_prefix, at::IntArrayRef prefix,                                              \
      const c10::optional<at::Tensor>&page_table, const c10::optional<at::Tensor>&tree_mask, int64_t mask_mode,    \
      int64_t mask_words, const c10::optional<at::Tensor>&prefix_len, const c10::optional<at::Tensor>&k_scale,     \
      const c10::optional<at::Tensor>&v_scale, const c10::optional<at::Tensor>&sinks, double sm_scale,             \
      bool lse_base2, at::Tensor &out, at::Tensor &lse, const c10::optional<at::Tensor>&k_prefix2,               \
      const c10::optional<at::Tensor>&v_prefix2, at::IntArrayRef prefix2, const c10::optional<at::Tensor>&k2_scale, \
      const c10::optional<at::Tensor>&v2_scale
#define CASCADE_PASS                                                                                       \
  info, plan, workspace, q, k_suffix, v_suffix, k_prefix, v_prefix, prefix, page_table, tree_mask, mask_mode, \
      mask_words, prefix_len, k_scale, v_scale, sinks, sm_scale, lse_base2, out, lse, k_prefix2, v_prefix2,   \
      prefix2, k2_scale, v2_scale

void cascade_run(CASCADE_ARGS) { cascade(false, CASCADE_PASS); }
void cascade_run_no_alloc(CASCADE_ARGS) { cascade(true, CASCADE_PASS); }
void cascade_meta(CASCADE_ARGS) {}

// ---- rotary_embedding ----
// Every check of the paged-cache operators stands here, so that a call costs
// its host little more than the launch (from Python 6 us with it; 15 with the
// checks and argument structs in Python).
void same_device(const at::Tensor& t, const at::Device& dev, const char* name) {
  TORCH_CHECK_VALUE(t.is_cuda() && t.device() == dev, "d2sd: ", name, " must be on the ROCm device of the others");
}

void need_type(const at::Tensor& t, at::ScalarType dt, const char* name) {
  TORCH_CHECK_TYPE(t.scalar_type() == dt, "d2sd: ", name, " must be ", dt, " (got ", t.scalar_type(), ")");
}

const at::Tensor* or_null(const c10::optional<at::Tensor>& t) { return t.has_value() ? &*t : nullptr; }

// Tensors that a batch, plan or cache holds for its caller: made on one stream and
// read by a call on another, they may be let go of while the call is under way, and
// their memory waits for it then.  home: the stream all of them were made on
// (nothing to do for calls on it), -1 for any.  Captured calls have them held by the
// graph.
void in_use(int64_t home, std::initializer_list<const at::Tensor*> held) {
  const c10::hip::HIPStream stream = c10::hip::getCurrentHIPStream();
  if (home == (int64_t)(intptr_t)stream.stream()) return;
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(stream.stream(), &status) != hipSuccess) (void)hipGetLastError();
  if (status != hipStreamCaptureStatusNone) return;
  for (const at::Tensor* t : held)
    if (t) c10::hip::HIPCachingAllocator::recordStream(t->storage().data_ptr(), stream);
}

void rotary_embedding(const c10::optional<at::Tensor>& q, const c10::optional<at::Tensor>& k, const at::Tensor& positions,
                      const at::Tensor& inv_freq, const c10::optional<at::Tensor>& q_out,
                      const c10::optional<at::Tensor>& k_out, bool interleaved, double scale, bool inverse) {
  TORCH_CHECK_VALUE(q.has_value() || k.has_value(), "d2sd: rotary_embedding needs q or k");
  const at::Tensor& any = q.has_value() ? *q : *k;
  const at::Device dev = any.device();
  TORCH_CHECK_VALUE(any.dim() == 3, "d2sd: q and k must be [tokens, heads, head_dim]");
  const int64_t n = any.size(0), d = any.size(2);
  d2sd_rotary_args a;
  std::memset(&a, 0, sizeof(a));
  auto take = [&](const c10::optional<at::Tensor>& t, const c10::optional<at::Tensor>& y, const char* name, const void*& in,
                  void*& out, int64_t& sn, int64_t& sh, int64_t& on, int64_t& oh, int& heads) {
    TORCH_CHECK_VALUE(t.has_value() == y.has_value(), "d2sd: ", name, " and its output go together");
    if (!t.has_value()) return;
    for (const at::Tensor* x : {&*t, &*y}) {
      need_type(*x, at::kBFloat16, name);
      TORCH_CHECK_VALUE(x->dim() == 3 && x->size(0) == n && x->size(2) == d && x->size(1) == t->size(1) &&
                            x->stride(2) == 1,
                        "d2sd: ", name, " must be [tokens, heads, head_dim] with a contiguous head_dim, like its output");
      same_device(*x, dev, name);
    }
    in = t->data_ptr();
    out = y->data_ptr();
    sn = t->stride(0), sh = t->stride(1), on = y->stride(0), oh = y->stride(1);
    heads = (int)t->size(1);
  };
  take(q, q_out, "q", a.q, a.q_out, a.q_stride_n, a.q_stride_h, a.qo_stride_n, a.qo_stride_h, a.num_qo_heads);
  take(k, k_out, "k", a.k, a.k_out, a.k_stride_n, a.k_stride_h, a.ko_stride_n, a.ko_stride_h, a.num_kv_heads);
  TORCH_CHECK_TYPE(positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong,
                   "d2sd: positions must be int32 or int64");
  TORCH_CHECK_VALUE(positions.dim() == 1 && positions.size(0) == n && positions.is_contiguous(),
                    "d2sd: positions must be a contiguous [tokens] tensor");
  need_type(inv_freq, at::kDouble, "inv_freq");
  TORCH_CHECK_VALUE(inv_freq.dim() == 1 && inv_freq.is_contiguous(), "d2sd: inv_freq must be contiguous and 1-D");
  same_device(positions, dev, "positions");
  same_device(inv_freq, dev, "inv_freq");
  TORCH_CHECK_VALUE(n <= INT32_MAX && d <= 256, "d2sd: too many tokens, or head_dim above 256");
  a.positions = positions.data_ptr();
  a.inv_freq = inv_freq.data_ptr<double>();
  a.scale = (float)scale;
  a.num_tokens = (int)n;
  a.head_dim = (int)d;
  a.num_pairs = (int)inv_freq.size(0);
  a.positions_64 = positions.scalar_type() == at::kLong;
  a.interleaved = interleaved;
  a.inverse = inverse;
  const c10::DeviceGuard guard(dev);
  check(d2sd_rotary_embedding(&a, current_stream()), "d2sd.rotary_embedding");
}

void rotary_meta(const c10::optional<at::Tensor>&, const c10::optional<at::Tensor>&, const at::Tensor&, const at::Tensor&,
                 const c10::optional<at::Tensor>&, const c10::optional<at::Tensor>&, bool, double, bool) {}

// ---- paged cache ----
// The pools' geometry from their tensors (checked when a PagedKVCache is made,
// again here as far as a kernel's bounds depend on it).
d2sd_paged_cache cache_of(const at::Tensor& k_pool, const at::Tensor& v_pool, const c10::optional<at::Tensor>& k_scale,
                          const c10::optional<at::Tensor>& v_scale, int64_t format, bool nhd) {
  TORCH_CHECK_VALUE(k_pool.is_cuda() && k_pool.dim() == 4 && k_pool.sizes() == v_pool.sizes() &&
                        k_pool.strides() == v_pool.strides() && k_pool.stride(3) == 1 &&
                        v_pool.device() == k_pool.device() && v_pool.scalar_type() == k_pool.scalar_type(),
                    "d2sd: k_pool and v_pool must be 4-D device tensors alike");
  TORCH_CHECK_TYPE((k_pool.scalar_type() == at::kBFloat16) == (format == D2SD_CACHE_BF16) && k_pool.element_size() <= 2,
                   "d2sd: the pools' type is not the format's");
  const int tok = nhd ? 1 : 2, head = nhd ? 2 : 1;
  d2sd_paged_cache c;
  std::memset(&c, 0, sizeof(c));
  c.k = k_pool.data_ptr();
  c.v = v_pool.data_ptr();
  c.stride_page = k_pool.stride(0);
  c.stride_head = k_pool.stride(head);
  c.stride_tok = k_pool.stride(tok);
  c.format = (int)format;
  c.num_pages = (int)k_pool.size(0);
  c.page_size = (int)k_pool.size(tok);
  c.num_kv_heads = (int)k_pool.size(head);
  c.head_dim = (int)k_pool.size(3) * (format == D2SD_CACHE_MXFP4 ? 2 : 1);
  if (format != D2SD_CACHE_BF16) {
    TORCH_CHECK_VALUE(k_scale.has_value() && v_scale.has_value(), "d2sd: a quantised cache needs k_scale and v_scale");
    same_device(*k_scale, k_pool.device(), "k_scale");
    same_device(*v_scale, k_pool.device(), "v_scale");
    TORCH_CHECK_VALUE(k_scale->sizes() == v_scale->sizes() && k_scale->strides() == v_scale->strides(),
                      "d2sd: k_scale and v_scale must be alike");
    if (format == D2SD_CACHE_FP8) {
      TORCH_CHECK_VALUE(k_scale->scalar_type() == at::kFloat && v_scale->scalar_type() == at::kFloat &&
                            k_scale->numel() == c.num_kv_heads && k_scale->is_contiguous(),
                        "d2sd: fp8 scales must be contiguous float32 [Hkv]");
    } else {
      TORCH_CHECK_VALUE(k_scale->scalar_type() == at::kByte && v_scale->scalar_type() == at::kByte && k_scale->dim() == 4 &&
                            k_scale->size(0) == k_pool.size(0) && k_scale->size(1) == k_pool.size(1) &&
                            k_scale->size(2) == k_pool.size(2) && k_scale->size(3) * 32 == c.head_dim &&
                            k_scale->stride(3) == 1,
                        "d2sd: block scales must be uint8 of the pools' shape with head_dim / 32 last");
      c.scale_stride_page = k_scale->stride(0);
      c.scale_stride_head = k_scale->stride(head);
      c.scale_stride_tok = k_scale->stride(tok);
    }
    c.k_scale = k_scale->data_ptr();
    c.v_scale = v_scale->data_ptr();
  }
  return c;
}

void cache_io(bool write, const at::Tensor& k, const at::Tensor& v, int64_t rows, const at::Tensor& items, int64_t num_items,
              const at::Tensor& kv_len, const at::Tensor& page_table, const at::Tensor& k_pool, const at::Tensor& v_pool,
              const c10::optional<at::Tensor>& k_scale, const c10::optional<at::Tensor>& v_scale, int64_t format, bool nhd,
              int64_t home, bool zero_missing = false) {
  d2sd_cache_io_args a;
  std::memset(&a, 0, sizeof(a));
  a.cache = cache_of(k_pool, v_pool, k_scale, v_scale, format, nhd);
  const at::Device dev = k_pool.device();
  for (const at::Tensor* t : {&k, &v}) {
    need_type(*t, at::kBFloat16, "k / v");
    TORCH_CHECK_VALUE(t->dim() == 3 && t->size(0) >= rows && t->size(1) == a.cache.num_kv_heads &&
                          t->size(2) == a.cache.head_dim && t->stride(2) == 1 && t->strides() == k.strides(),
                      "d2sd: k and v must be [>= ", rows, ", ", a.cache.num_kv_heads, ", ", a.cache.head_dim,
                      "] with a contiguous head_dim and equal strides");
    same_device(*t, dev, "k / v");
  }
  for (const at::Tensor* t : {&items, &kv_len, &page_table}) {
    TORCH_CHECK_VALUE(t->scalar_type() == at::kInt && t->is_contiguous(), "d2sd: a batch's tensors are contiguous int32");
    same_device(*t, dev, "the batch");
  }
  TORCH_CHECK_VALUE(items.numel() >= num_items * (write ? 4 : 8), "d2sd: too few items");
  a.items = items.data_ptr();
  a.kv_len = kv_len.data_ptr<int32_t>();
  a.page_table = page_table.data_ptr<int32_t>();
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.stride_n = k.stride(0);
  a.stride_h = k.stride(1);
  a.num_items = (int)num_items;
  a.zero_missing = zero_missing;
  const c10::DeviceGuard guard(dev);
  check(write ? d2sd_cache_write(&a, current_stream()) : d2sd_cache_read(&a, current_stream()),
        write ? "d2sd.cache_write" : "d2sd.cache_read");
  in_use(home, {&items, &kv_len, &page_table, &k_pool, &v_pool, or_null(k_scale), or_null(v_scale)});
}

#define CACHE_ARGS                                                                                             \
  const at::Tensor &kv_len, const at::Tensor &page_table, const at::Tensor &k_pool, const at::Tensor &v_pool, \
      const c10::optional<at::Tensor>&k_scale, const c10::optional<at::Tensor>&v_scale, int64_t format, bool nhd
#define CACHE_PASS kv_len, page_table, k_pool, v_pool, k_scale, v_scale, format, nhd

void cache_write(const at::Tensor& k, const at::Tensor& v, const at::Tensor& items, int64_t num_items, CACHE_ARGS,
                 int64_t home) {
  cache_io(true, k, v, num_items, items, num_items, CACHE_PASS, home);
}

void cache_read_out(at::Tensor& k, at::Tensor& v, int64_t rows, const at::Tensor& items, int64_t num_items, CACHE_ARGS,
                    int64_t home) {
  cache_io(false, k, v, rows, items, num_items, CACHE_PASS, home);
}

std::tuple<at::Tensor, at::Tensor> cache_read(int64_t rows, const at::Tensor& items, int64_t num_items, CACHE_ARGS,
                                              int64_t home) {
  const auto opt = k_pool.options().dtype(at::kBFloat16);
  const int64_t hkv = k_pool.size(nhd ? 2 : 1), d = k_pool.size(3) * (format == D2SD_CACHE_MXFP4 ? 2 : 1);
  at::Tensor k = at::empty({rows, hkv, d}, opt), v = at::empty({rows, hkv, d}, opt);
  cache_io(false, k, v, rows, items, num_items, CACHE_PASS, home, true);
  return {k, v};
}

// ---- cache_append ----
void cache_append(const c10::optional<at::Tensor>& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& items,
                  int64_t num_items, CACHE_ARGS, const at::Tensor& inv_freq, const c10::optional<at::Tensor>& positions,
                  const c10::optional<at::Tensor>& q_norm, const c10::optional<at::Tensor>& k_norm, double eps, double scale,
                  bool interleaved, const c10::optional<at::Tensor>& q_out, int64_t home) {
  d2sd_cache_append_args a;
  std::memset(&a, 0, sizeof(a));
  a.cache = cache_of(k_pool, v_pool, k_scale, v_scale, format, nhd);
  const at::Device dev = k_pool.device();
  const int64_t d = a.cache.head_dim;
  for (const at::Tensor* t : {&k, &v}) {
    need_type(*t, at::kBFloat16, "k / v");
    TORCH_CHECK_VALUE(t->dim() == 3 && t->size(0) >= num_items && t->size(1) == a.cache.num_kv_heads && t->size(2) == d &&
                          t->stride(2) == 1,
                      "d2sd: k and v must be [>= ", num_items, ", ", a.cache.num_kv_heads, ", ", d,
                      "] with a contiguous head_dim");
    same_device(*t, dev, "k / v");
  }
  TORCH_CHECK_VALUE(q.has_value() == q_out.has_value(), "d2sd: q and its output go together");
  if (q.has_value()) {
    for (const at::Tensor* t : {&*q, &*q_out}) {
      need_type(*t, at::kBFloat16, "q / q_out");
      TORCH_CHECK_VALUE(t->dim() == 3 && t->size(0) >= num_items && t->size(1) == q->size(1) && t->size(2) == d &&
                            t->size(0) == q->size(0) && t->stride(2) == 1,
                        "d2sd: q and q_out must be [>= ", num_items, ", Hq, ", d, "] alike with a contiguous head_dim");
      same_device(*t, dev, "q / q_out");
    }
    // (heads inside a token's, or tokens inside a head's)
    const int64_t T = q_out->size(0), H = q_out->size(1), st = q_out->stride(0), sh = q_out->stride(1);
    TORCH_CHECK_VALUE((T < 2 || st >= d) && (H < 2 || sh >= d) && (T < 2 || H < 2 || st >= (H - 1) * sh + d || sh >= (T - 1) * st + d),
                      "d2sd: the rows of q_out must lie apart");
    TORCH_CHECK_VALUE(q->size(1) <= INT32_MAX, "d2sd: too many heads");
    a.q = q->data_ptr();
    a.q_out = q_out->data_ptr();
    a.q_stride_n = q->stride(0), a.q_stride_h = q->stride(1);
    a.qo_stride_n = q_out->stride(0), a.qo_stride_h = q_out->stride(1);
    a.num_qo_heads = (int)q->size(1);
  }
  for (const at::Tensor* t : {&items, &kv_len, &page_table}) {
    TORCH_CHECK_VALUE(t->scalar_type() == at::kInt && t->is_contiguous(), "d2sd: a batch's tensors are contiguous int32");
    same_device(*t, dev, "the batch");
  }
  TORCH_CHECK_VALUE(items.numel() >= num_items * 4, "d2sd: too few items");
  need_type(inv_freq, at::kDouble, "inv_freq");
  TORCH_CHECK_VALUE(inv_freq.dim() == 1 && inv_freq.is_contiguous() && inv_freq.size(0) <= d / 2,
                    "d2sd: inv_freq must be contiguous and 1-D, at most head_dim / 2 entries");
  same_device(inv_freq, dev, "inv_freq");
  if (positions.has_value()) {
    TORCH_CHECK_TYPE(positions->scalar_type() == at::kInt || positions->scalar_type() == at::kLong,
                     "d2sd: positions must be int32 or int64");
    TORCH_CHECK_VALUE(positions->dim() == 1 && positions->size(0) >= num_items && positions->is_contiguous(),
                      "d2sd: positions must be a contiguous [>= ", num_items, "] tensor");
    same_device(*positions, dev, "positions");
    a.positions = positions->data_ptr();
    a.positions_64 = positions->scalar_type() == at::kLong;
  }
  auto weight = [&](const c10::optional<at::Tensor>& t, const char* name) -> const void* {
    if (!t.has_value()) return nullptr;
    need_type(*t, at::kBFloat16, name);
    TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == d && t->is_contiguous(), "d2sd: ", name, " must be a contiguous [", d,
                      "] tensor");
    same_device(*t, dev, name);
    return t->data_ptr();
  };
  a.q_norm = weight(q_norm, "q_norm");
  a.k_norm = weight(k_norm, "k_norm");
  a.items = (const d2sd_cache_token*)items.data_ptr();
  a.kv_len = kv_len.data_ptr<int32_t>();
  a.page_table = page_table.data_ptr<int32_t>();
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.k_stride_n = k.stride(0), a.k_stride_h = k.stride(1);
  a.v_stride_n = v.stride(0), a.v_stride_h = v.stride(1);
  a.inv_freq = inv_freq.data_ptr<double>();
  a.eps = (float)eps;
  a.scale = (float)scale;
  a.num_tokens = (int)num_items;
  a.num_pairs = (int)inv_freq.size(0);
  a.interleaved = interleaved;
  const c10::DeviceGuard guard(dev);
  check(d2sd_cache_append(&a, current_stream()), "d2sd.cache_append");
  in_use(home, {&items, &kv_len, &page_table, &k_pool, &v_pool, or_null(k_scale), or_null(v_scale)});
}

void cache_append_meta(const c10::optional<at::Tensor>&, const at::Tensor&, const at::Tensor&, const at::Tensor&, int64_t,
                       CACHE_ARGS, const at::Tensor&, const c10::optional<at::Tensor>&, const c10::optional<at::Tensor>&,
                       const c10::optional<at::Tensor>&, double, double, bool, const c10::optional<at::Tensor>&, int64_t) {}
void cache_write_meta(const at::Tensor&, const at::Tensor&, const at::Tensor&, int64_t, CACHE_ARGS, int64_t) {}
void cache_read_out_meta(at::Tensor&, at::Tensor&, int64_t, const at::Tensor&, int64_t, CACHE_ARGS, int64_t) {}
std::tuple<at::Tensor, at::Tensor> cache_read_meta(int64_t rows, const at::Tensor&, int64_t, CACHE_ARGS, int64_t) {
  const auto opt = k_pool.options().dtype(at::kBFloat16);
  const int64_t hkv = k_pool.size(nhd ? 2 : 1), d = k_pool.size(3) * (format == D2SD_CACHE_MXFP4 ? 2 : 1);
  return {at::empty({rows, hkv, d}, opt), at::empty({rows, hkv, d}, opt)};
}

// ---- chunk_attention ----
// info: the d2sd_chunk_plan_info bytes plan() produced (CPU uint8 tensor).
void chunk_attention_out(const at::Tensor& q, at::Tensor& out, at::Tensor& lse, const c10::optional<at::Tensor>& workspace,
                         const at::Tensor& info, const at::Tensor& plan, CACHE_ARGS, const c10::optional<at::Tensor>& sinks,
                         double sm_scale, bool lse_base2, int64_t home) {
  TORCH_CHECK(info.device().is_cpu() && info.scalar_type() == at::kByte && info.is_contiguous() &&
                  (size_t)info.numel() == sizeof(d2sd_chunk_plan_info),
              "d2sd: info must hold the bytes of a d2sd_chunk_plan_info");
  d2sd_chunk_plan_info pi;
  std::memcpy(&pi, info.data_ptr(), sizeof(pi));
  d2sd_chunk_run_args a;
  std::memset(&a, 0, sizeof(a));
  a.cache = cache_of(k_pool, v_pool, k_scale, v_scale, format, nhd);
  const at::Device dev = k_pool.device();
  for (const at::Tensor* t : {&q, (const at::Tensor*)&out}) {
    need_type(*t, at::kBFloat16, "q / out");
    TORCH_CHECK_VALUE(t->dim() == 3 && t->size(0) >= pi.total_q && t->size(1) == pi.num_qo_heads &&
                          t->size(2) == pi.head_dim && t->stride(2) == 1 && t->size(0) == q.size(0),
                      "d2sd: q and out must be [>= ", pi.total_q, ", ", pi.num_qo_heads, ", ", pi.head_dim,
                      "] with a contiguous head_dim");
    same_device(*t, dev, "q / out");
  }
  TORCH_CHECK_VALUE(lse.scalar_type() == at::kFloat && lse.dim() == 2 && lse.size(0) == q.size(0) &&
                        lse.size(1) == pi.num_qo_heads && lse.stride(1) == 1,
                    "d2sd: lse must be float32 [rows of q, Hq] with contiguous heads");
  same_device(lse, dev, "lse");
  for (const at::Tensor* t : {&plan, &kv_len, &page_table}) {
    TORCH_CHECK_VALUE(t->scalar_type() == at::kInt && t->is_contiguous(), "d2sd: plan and batch are contiguous int32");
    same_device(*t, dev, "plan / batch");
  }
  TORCH_CHECK_VALUE(plan.numel() >= pi.plan_ints && kv_len.numel() >= pi.num_reqs &&
                        page_table.numel() >= pi.num_page_entries,
                    "d2sd: plan, kv_len or page_table is shorter than planned");
  if (sinks.has_value()) {
    TORCH_CHECK_VALUE(sinks->scalar_type() == at::kFloat && sinks->numel() == pi.num_qo_heads && sinks->is_contiguous(),
                      "d2sd: sinks must be a contiguous float32 [Hq]");
    same_device(*sinks, dev, "sinks");
    a.sinks = sinks->data_ptr<float>();
  }
  const c10::DeviceGuard guard(dev);
  at::Tensor work;
  if (pi.workspace_bytes > 0) {
    if (workspace.has_value()) {
      TORCH_CHECK_VALUE(workspace->is_contiguous() && (size_t)workspace->nbytes() >= pi.workspace_bytes,
                        "d2sd: workspace must be ", pi.workspace_bytes, " contiguous bytes");
      same_device(*workspace, dev, "workspace");
      work = *workspace;
    } else {
      work = at::empty({(int64_t)pi.workspace_bytes}, q.options().dtype(at::kByte));
    }
    a.workspace = work.data_ptr();
    a.workspace_bytes = (size_t)work.nbytes();
  }
  a.plan = plan.data_ptr<int32_t>();
  a.kv_len = kv_len.data_ptr<int32_t>();
  a.page_table = page_table.data_ptr<int32_t>();
  a.q = q.data_ptr();
  a.q_stride_n = q.stride(0);
  a.q_stride_h = q.stride(1);
  a.out = out.data_ptr();
  a.o_stride_n = out.stride(0);
  a.o_stride_h = out.stride(1);
  a.lse = lse.data_ptr<float>();
  a.lse_stride_n = lse.stride(0);
  a.sm_scale = (float)sm_scale;
  a.lse_base2 = lse_base2;
  check(d2sd_chunk_run(&pi, &a, current_stream()), "d2sd.chunk_attention");
  in_use(home, {&plan, &kv_len, &page_table, or_null(sinks), &k_pool, &v_pool, or_null(k_scale), or_null(v_scale)});
}

std::tuple<at::Tensor, at::Tensor> chunk_attention(const at::Tensor& q, const c10::optional<at::Tensor>& workspace,
                                                   const at::Tensor& info, const at::Tensor& plan, CACHE_ARGS,
                                                   const c10::optional<at::Tensor>& sinks, double sm_scale,
                                                   bool lse_base2, int64_t home) {
  TORCH_CHECK_VALUE(q.dim() == 3, "d2sd: q must be [tokens, Hq, D]");
  at::Tensor out = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
  at::Tensor lse = at::empty({q.size(0), q.size(1)}, q.options().dtype(at::kFloat));
  chunk_attention_out(q, out, lse, workspace, info, plan, CACHE_PASS, sinks, sm_scale, lse_base2, home);
  d2sd_chunk_plan_info pi;
  std::memcpy(&pi, info.data_ptr(), sizeof(pi));
  if (q.size(0) > pi.total_q) {  // rows behind the last request: empty ones
    out.narrow(0, pi.total_q, q.size(0) - pi.total_q).zero_();
    lse.narrow(0, pi.total_q, q.size(0) - pi.total_q).fill_(-INFINITY);
  }
  return {out, lse};
}

void chunk_attention_out_meta(const at::Tensor&, at::Tensor&, at::Tensor&, const c10::optional<at::Tensor>&, const at::Tensor&,
                              const at::Tensor&, CACHE_ARGS, const c10::optional<at::Tensor>&, double, bool, int64_t) {}
std::tuple<at::Tensor, at::Tensor> chunk_attention_meta(const at::Tensor& q, const c10::optional<at::Tensor>&,
                                                        const at::Tensor&, const at::Tensor&, CACHE_ARGS,
                                                        const c10::optional<at::Tensor>&, double, bool,
                                                        int64_t) {
  return {at::empty(q.sizes(), q.options()), at::empty({q.size(0), q.size(1)}, q.options().dtype(at::kFloat))};
}

}  // namespace

TORCH_LIBRARY(d2sd, m) {
  m.def("single_prefill_with_kv_cache(Tensor q, Tensor k, Tensor v, bool causal=False, str kv_layout=\"NHD\", "
        "float? sm_scale=None, bool lse_base2=False) -> (Tensor, Tensor)");
  m.def("merge_state_in_place(Tensor(a!) v, Tensor(b!) s, Tensor v_other, Tensor s_other, bool lse_base2=False) -> ()");
  m.def("local_attention_merge(Tensor q, Tensor k, Tensor v, Tensor(a!) out, Tensor(b!) lse, bool causal, "
        "float sm_scale, Tensor? sinks=None, bool lse_base2=False) -> ()");
  const char* cascade_schema =
      "(Tensor info, Tensor plan, Tensor workspace, Tensor q, Tensor k_suffix, Tensor v_suffix, Tensor? k_prefix, "
      "Tensor? v_prefix, int[] prefix, Tensor? page_table, Tensor? tree_mask, int mask_mode, int mask_words, "
      "Tensor? prefix_len, Tensor? k_scale, Tensor? v_scale, Tensor? sinks, float sm_scale, bool lse_base2, "
      "Tensor(a!) out, Tensor(b!) lse, Tensor? k_prefix2=None, Tensor? v_prefix2=None, int[] prefix2=[], "
      "Tensor? k2_scale=None, Tensor? v2_scale=None) -> ()";
  m.def((std::string("cascade_run") + cascade_schema).c_str());
  m.def((std::string("cascade_run_no_alloc") + cascade_schema).c_str());
  m.def("rotary_embedding(Tensor? q, Tensor? k, Tensor positions, Tensor inv_freq, Tensor(a!)? q_out, "
        "Tensor(b!)? k_out, bool interleaved, float scale, bool inverse) -> ()");
  const std::string read = "Tensor kv_len, Tensor page_table, Tensor k_pool, Tensor v_pool, Tensor? k_scale, Tensor? v_scale, "
                           "int format, bool nhd";
  m.def("cache_write(Tensor k, Tensor v, Tensor items, int num_items, Tensor kv_len, Tensor page_table, "
        "Tensor(a!) k_pool, Tensor(b!) v_pool, Tensor(c!)? k_scale, Tensor(d!)? v_scale, int format, bool nhd, "
        "int home=-1) -> ()");
  m.def("cache_append(Tensor? q, Tensor k, Tensor v, Tensor items, int num_items, Tensor kv_len, Tensor page_table, "
        "Tensor(a!) k_pool, Tensor(b!) v_pool, Tensor(c!)? k_scale, Tensor(d!)? v_scale, int format, bool nhd, "
        "Tensor inv_freq, Tensor? positions, Tensor? q_norm, Tensor? k_norm, float eps, float scale, bool interleaved, "
        "Tensor(e!)? q_out, int home=-1) -> ()");
  m.def(("cache_read_out(Tensor(a!) k, Tensor(b!) v, int rows, Tensor items, int num_items, " + read + ", int home=-1) -> ()").c_str());
  m.def(("cache_read(int rows, Tensor items, int num_items, " + read + ", int home=-1) -> (Tensor, Tensor)").c_str());
  const std::string attn = "Tensor? workspace, Tensor info, Tensor plan, " + read +
                           ", Tensor? sinks, float sm_scale, bool lse_base2, int home=-1";
  m.def(("chunk_attention_out(Tensor q, Tensor(a!) out, Tensor(b!) lse, " + attn + ") -> ()").c_str());
  m.def(("chunk_attention(Tensor q, " + attn + ") -> (Tensor, Tensor)").c_str());
}

TORCH_LIBRARY_IMPL(d2sd, CUDA, m) {
  m.impl("single_prefill_with_kv_cache", &single_prefill);
  m.impl("merge_state_in_place", &merge_state_in_place);
  m.impl("local_attention_merge", &local_attention_merge);
  m.impl("cascade_run", &cascade_run);
  m.impl("cascade_run_no_alloc", &cascade_run_no_alloc);
  m.impl("rotary_embedding", &rotary_embedding);
  m.impl("cache_write", &cache_write);
  m.impl("cache_append", &cache_append);
  m.impl("cache_read_out", &cache_read_out);
  m.impl("cache_read", &cache_read);
  m.impl("chunk_attention_out", &chunk_attention_out);
  m.impl("chunk_attention", &chunk_attention);
}

// CPU tensors: refused by the operators' own checks
TORCH_LIBRARY_IMPL(d2sd, CPU, m) {
  m.impl("rotary_embedding", &rotary_embedding);
  m.impl("cache_write", &cache_write);
  m.impl("cache_append", &cache_append);
  m.impl("cache_read_out", &cache_read_out);
  m.impl("chunk_attention_out", &chunk_attention_out);
}

TORCH_LIBRARY_IMPL(d2sd, Meta, m) {
  m.impl("single_prefill_with_kv_cache", &single_prefill_meta);
  m.impl("merge_state_in_place", &merge_state_meta);
  m.impl("local_attention_merge", &local_attention_merge_meta);
  m.impl("cascade_run", &cascade_meta);
  m.impl("cascade_run_no_alloc", &cascade_meta);
  m.impl("rotary_embedding", &rotary_meta);
  m.impl("cache_write", &cache_write_meta);
  m.impl("cache_append", &cache_append_meta);
  m.impl("cache_read_out", &cache_read_out_meta);
  m.impl("cache_read", &cache_read_meta);
  m.impl("chunk_attention_out", &chunk_attention_out_meta);
  m.impl("chunk_attention", &chunk_attention_meta);
}
