// torch.ops.kvr.* operators of the target model's side of a speculation
// round, over libkvr.so's C ABI:
//
//   kvr::paged_append     new tokens' keys and values into their pages
//   kvr::paged_attention  attention of the new tokens over the pages
//   kvr::paged_evict      the kept tokens of every sequence into new pages
//   kvr::verify_draft     accepted drafted tokens and the next one
//
// Checks raise ValueError before anything is allocated or launched.  Outputs
// come from the caching allocator.  Scratch is cached per (operator, device,
// stream), and a call holds it until its last launch is in the stream: the
// operators run without Python's lock, and a sampled verification is two
// launches with its counters non-zero between them, so another thread's call
// must not come in between.  Launches on one stream follow each other, and a
// completed call leaves the counters at zero.  Inside a CUDA graph capture a
// call takes its scratch from the graph's own memory (a memset node zeroes
// the counters on each replay), so a graph never depends on a cached buffer.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include <cfloat>
#include <cmath>
#include <cstring>
#include <map>
#include <mutex>
#include <string>
#include <tuple>
#include <utility>
#include <vector>

#include "../../include/kvr.h"

namespace {

void raise_status(const char* fn, int st) {
  if (st == KVR_OK) return;
  const std::string text = kvr_status_string(st);
  if (st == KVR_ERR_INVALID_ARGUMENT || st == KVR_ERR_UNSUPPORTED || st == KVR_ERR_MISALIGNED)
    TORCH_CHECK_VALUE(false, fn, " failed: ", text, " (status ", st, ")");
  TORCH_CHECK(false, fn, " failed: ", text, " (status ", st, ")", st == KVR_ERR_CUDA ? ": " : "",
              st == KVR_ERR_CUDA ? kvr_last_error() : "");
}

// A stride the kernels multiply an index with; an axis of one element is
// never stepped along, and torch lets it have any stride.
int64_t step(const at::Tensor& t, int64_t dim) { return t.size(dim) > 1 ? t.stride(dim) : 0; }

bool rows16(const at::Tensor& t) {
  for (int64_t d = 0; d + 1 < t.dim(); ++d)
    if (step(t, d) % 8) return false;
  return (t.size(t.dim() - 1) <= 1 || t.stride(t.dim() - 1) == 1) &&
         reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
}

// Keys, values and queries may have any strides as long as the head's
// elements are contiguous and rows start on 16 bytes; others are copied.
at::Tensor rows(const at::Tensor& t) { return rows16(t) ? t : t.clone(at::MemoryFormat::Contiguous); }

// Whether elements share memory along an axis (an expanded tensor): threads
// would write to one place.
bool shares_memory(const at::Tensor& t) {
  for (int64_t d = 0; d < t.dim(); ++d)
    if (t.size(d) > 1 && t.stride(d) == 0) return true;
  return false;
}

enum class Op { attention, verify };
struct Scratch {
  std::mutex mu;   // held from taking the buffers to the call's last launch
  at::Tensor workspace, counters;
};
std::mutex g_mu;   // the map and the list below
std::map<std::tuple<Op, int, uintptr_t>, Scratch> g_scratch;
// Buffers outgrown by a later call; launches in flight may still hold them,
// and the growth is geometric, so they are kept.
std::vector<at::Tensor> g_outgrown;

// A call's scratch, for as long as this object lives.
class Lease {
 public:
  at::Tensor workspace, counters;

  Lease(Op op, const at::Device& dev, cudaStream_t stream, int64_t bytes, int64_t n_counters) {
    const auto u8 = at::TensorOptions().dtype(at::kByte).device(dev);
    const auto i32 = at::TensorOptions().dtype(at::kInt).device(dev);
    if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) {
      workspace = at::empty({std::max<int64_t>(bytes, 16)}, u8);
      counters = at::zeros({std::max<int64_t>(n_counters, 1)}, i32);
      return;
    }
    {
      std::lock_guard<std::mutex> lock(g_mu);
      cached_ = &g_scratch[{op, dev.index(), reinterpret_cast<uintptr_t>(stream)}];   // (nodes of a map stay put)
    }
    held_ = std::unique_lock<std::mutex>(cached_->mu);
    if (!cached_->workspace.defined() || cached_->workspace.numel() < bytes) {
      outgrow(cached_->workspace);
      cached_->workspace = at::empty({std::max<int64_t>(2 * bytes, 1 << 20)}, u8);
    }
    if (!cached_->counters.defined() || cached_->counters.numel() < n_counters) {
      outgrow(cached_->counters);
      cached_->counters = at::zeros({std::max<int64_t>(2 * n_counters, 4096)}, i32);
    }
    workspace = cached_->workspace;
    counters = cached_->counters;
  }

  // The status of the call's launches: after a failed one the counters may
  // not be zero, so the next call gets others.
  int launched(int st) {
    if (st != KVR_OK && cached_) outgrow(cached_->counters);
    return st;
  }

 private:
  static void outgrow(at::Tensor& t) {
    if (!t.defined()) return;
    std::lock_guard<std::mutex> lock(g_mu);
    g_outgrown.push_back(std::move(t));
    t = at::Tensor();
  }
  Scratch* cached_ = nullptr;
  std::unique_lock<std::mutex> held_;
};

bool is_half_type(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf; }

void check_pages(const at::Tensor& kp, const at::Tensor& vp, const at::Tensor& table, const at::Tensor& lengths,
                 const at::Device& dev) {
  TORCH_CHECK_VALUE(dev.is_cuda(), "kv_reduce_b200 operates on CUDA tensors only (no CPU fallback).");
  for (const at::Tensor* t : {&kp, &vp, &table, &lengths})
    TORCH_CHECK_VALUE(t->device() == dev, "All tensors must be on the same CUDA device.");
  TORCH_CHECK_VALUE(kp.dim() == 4 && kp.sizes() == vp.sizes(),
                    "key_pages and value_pages must be [num_pages, kv_heads, page_size, head_dim] of one shape.");
  TORCH_CHECK_VALUE(is_half_type(kp.scalar_type()) && vp.scalar_type() == kp.scalar_type(),
                    "key_pages and value_pages must be bf16 or fp16, both the same.");
  TORCH_CHECK_VALUE(kp.size(1) > 0 && kp.size(2) > 0, "key_pages must have at least one head and one row per page.");
  TORCH_CHECK_VALUE(rows16(kp) && rows16(vp),
                    "pages must have contiguous head elements and rows that start on 16 bytes.");
  TORCH_CHECK_VALUE(table.dim() == 2 && table.scalar_type() == at::kInt && (table.size(1) <= 1 || table.stride(1) == 1),
                    "block_table must be int32 [batch, pages] with contiguous rows.");
  TORCH_CHECK_VALUE(lengths.dim() == 1 && lengths.scalar_type() == at::kInt && lengths.size(0) == table.size(0) &&
                        (lengths.size(0) <= 1 || lengths.stride(0) == 1),
                    "lengths must be a contiguous int32 [batch] tensor.");
}

const int* counts_of(const std::optional<at::Tensor>& counts, const at::Tensor& lengths) {
  if (!counts.has_value() || !counts->defined()) return nullptr;
  TORCH_CHECK_VALUE(counts->device() == lengths.device() && counts->scalar_type() == at::kInt && counts->dim() == 1 &&
                        counts->size(0) == lengths.size(0) && (counts->size(0) <= 1 || counts->stride(0) == 1),
                    "new_counts must be a contiguous int32 [batch] tensor.");
  return counts->data_ptr<int>();
}

void paged_append(const at::Tensor& key, const at::Tensor& value, const at::Tensor& kp, const at::Tensor& vp,
                  const at::Tensor& table, const at::Tensor& lengths, const std::optional<at::Tensor>& new_counts) {
  check_pages(kp, vp, table, lengths, key.device());
  TORCH_CHECK_VALUE(value.device() == key.device(), "All tensors must be on the same CUDA device.");
  TORCH_CHECK_VALUE(key.dim() == 4 && key.sizes() == value.sizes() && key.size(0) == lengths.size(0) &&
                        key.size(1) == kp.size(1) && key.size(3) == kp.size(3),
                    "key and value must be [batch, kv_heads, new_tokens, head_dim] and match the pages.");
  TORCH_CHECK_VALUE(key.scalar_type() == kp.scalar_type() && value.scalar_type() == kp.scalar_type(),
                    "key and value must have the pages' dtype.");
  TORCH_CHECK_VALUE(key.size(3) % 8 == 0, "head_dim must be a multiple of 8.");
  TORCH_CHECK_VALUE(!shares_memory(kp) && !shares_memory(vp), "pages that are written must not be expanded tensors.");
  const int* counts = counts_of(new_counts, lengths);
  c10::cuda::CUDAGuard guard(key.device());
  if (key.numel() == 0) return;
  const at::Tensor k = rows(key), v = rows(value);
  kvr_paged_append_args a;
  std::memset(&a, 0, sizeof(a));
  a.key = k.data_ptr();
  a.key_b_stride = step(k, 0), a.key_h_stride = step(k, 1), a.key_t_stride = step(k, 2);
  a.value = v.data_ptr();
  a.value_b_stride = step(v, 0), a.value_h_stride = step(v, 1), a.value_t_stride = step(v, 2);
  a.key_pages = kp.data_ptr();
  a.key_page_stride = step(kp, 0), a.key_head_stride = step(kp, 1), a.key_row_stride = step(kp, 2);
  a.value_pages = vp.data_ptr();
  a.value_page_stride = step(vp, 0), a.value_head_stride = step(vp, 1), a.value_row_stride = step(vp, 2);
  a.block_table = table.data_ptr<int>();
  a.table_stride = step(table, 0);
  a.table_width = (int)table.size(1);
  a.num_pages = (int)kp.size(0);
  a.lengths = lengths.data_ptr<int>();
  a.batch = (int)k.size(0), a.kv_heads = (int)k.size(1), a.new_tokens = (int)k.size(2), a.head_dim = (int)k.size(3);
  a.page_size = (int)kp.size(2);
  a.new_counts = counts;
  raise_status("kvr_paged_append", kvr_paged_append(&a, c10::cuda::getCurrentCUDAStream().stream()));
}

std::tuple<at::Tensor, at::Tensor> paged_attention(const at::Tensor& query, const at::Tensor& kp, const at::Tensor& vp,
                                                   const at::Tensor& table, const at::Tensor& lengths,
                                                   std::optional<double> scale, int64_t window, int64_t sinks,
                                                   const std::optional<at::Tensor>& token_weights, bool with_lse,
                                                   const std::optional<at::Tensor>& new_counts) {
  const at::Device dev = query.device();
  check_pages(kp, vp, table, lengths, dev);
  TORCH_CHECK_VALUE(query.dim() == 4, "query must have shape [batch, query_heads, new_tokens, head_dim].");
  TORCH_CHECK_VALUE(query.scalar_type() == kp.scalar_type(), "query must have the pages' dtype.");
  TORCH_CHECK_VALUE(query.size(0) == lengths.size(0), "Query and cache batch dimensions must match.");
  TORCH_CHECK_VALUE(query.size(3) == kp.size(3), "Query and cache head dimensions must match.");
  TORCH_CHECK_VALUE(query.size(1) > 0 && query.size(1) % kp.size(1) == 0, "Query heads must be divisible by KV heads.");
  TORCH_CHECK_VALUE(query.size(2) > 0, "query must hold at least one new token.");
  TORCH_CHECK_VALUE(query.size(3) == 64 || query.size(3) == 128, "head_dim must be one of [64, 128].");
  TORCH_CHECK_VALUE(window >= 0 && sinks >= 0 && window <= INT32_MAX / 2 && sinks <= INT32_MAX / 2,
                    "window and sinks must not be negative.");
  TORCH_CHECK_VALUE(table.size(1) * kp.size(2) <= (1 << 30), "block_table addresses more than 2^30 tokens.");
  const int* counts = counts_of(new_counts, lengths);
  const bool weighted = token_weights.has_value() && token_weights->defined();
  if (weighted) {
    const at::Tensor& w = *token_weights;
    TORCH_CHECK_VALUE(w.device() == dev && w.scalar_type() == at::kFloat && w.dim() == 2 &&
                          w.size(0) == query.size(0) && w.size(1) >= table.size(1) * kp.size(2) &&
                          (w.size(1) <= 1 || w.stride(1) == 1),
                      "token_weights must be fp32 [batch, >= block_table.shape[1] * page_size] with contiguous rows.");
    TORCH_CHECK_VALUE(w.size(0) <= 1 || w.stride(0) >= table.size(1) * kp.size(2),
                      "token_weights are added to: their rows must not share memory.");
  }
  c10::cuda::CUDAGuard guard(dev);
  at::Tensor out = at::empty(query.sizes(), query.options().memory_format(at::MemoryFormat::Contiguous));
  const auto f32 = query.options().dtype(at::kFloat).memory_format(at::MemoryFormat::Contiguous);
  at::Tensor lse;
  if (with_lse) lse = at::empty({query.size(0), query.size(1), query.size(2)}, f32);
  if (query.numel() > 0) {
    const at::Tensor q = rows(query);
    kvr_paged_attention_args a;
    std::memset(&a, 0, sizeof(a));
    a.query = q.data_ptr();
    a.q_b_stride = step(q, 0), a.q_h_stride = step(q, 1), a.q_t_stride = step(q, 2);
    a.key_pages = kp.data_ptr();
    a.key_page_stride = step(kp, 0), a.key_head_stride = step(kp, 1), a.key_row_stride = step(kp, 2);
    a.value_pages = vp.data_ptr();
    a.value_page_stride = step(vp, 0), a.value_head_stride = step(vp, 1), a.value_row_stride = step(vp, 2);
    a.block_table = table.data_ptr<int>();
    a.table_stride = step(table, 0);
    a.table_width = (int)table.size(1);
    a.num_pages = (int)kp.size(0);
    a.lengths = lengths.data_ptr<int>();
    a.out = out.data_ptr();
    a.lse = with_lse ? lse.data_ptr<float>() : nullptr;
    a.token_weights = weighted ? token_weights->data_ptr<float>() : nullptr;
    a.weights_b_stride = weighted ? step(*token_weights, 0) : 0;
    a.dtype = q.scalar_type() == at::kHalf ? 1 : 0;
    a.batch = (int)q.size(0), a.q_heads = (int)q.size(1), a.new_tokens = (int)q.size(2), a.head_dim = (int)q.size(3);
    a.kv_heads = (int)kp.size(1), a.page_size = (int)kp.size(2);
    a.window = (int)window, a.sinks = (int)sinks;
    a.new_counts = counts;
    a.scale = scale.has_value() ? (float)*scale : (float)(1.0 / std::sqrt((double)q.size(3)));
    size_t ws = 0, counters = 0, scores = 0;
    raise_status("kvr_paged_attention_plan", kvr_paged_attention_plan(&a, &ws, &counters, &scores));
    cudaStream_t stream = c10::cuda::getCurrentCUDAStream().stream();
    Lease s(Op::attention, dev, stream, (int64_t)ws, (int64_t)counters);
    a.workspace = s.workspace.data_ptr();
    a.workspace_bytes = (size_t)s.workspace.numel();
    a.counters = s.counters.data_ptr<int>();
    at::Tensor x;
    if (scores > 0) {
      x = at::empty({(int64_t)scores}, at::TensorOptions().dtype(at::kByte).device(dev));
      a.scores = x.data_ptr();
      a.scores_bytes = scores;
    }
    raise_status("kvr_paged_attention", s.launched(kvr_paged_attention(&a, stream)));
  }
  if (!with_lse) lse = at::empty({0}, f32);
  return {out, lse};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> paged_evict(const at::Tensor& kp, const at::Tensor& vp,
                                                           const at::Tensor& table, const at::Tensor& lengths,
                                                           const at::Tensor& weights, const at::Tensor& new_table,
                                                           int64_t keep, int64_t recent, int64_t first) {
  const at::Device dev = kp.device();
  check_pages(kp, vp, table, lengths, dev);
  TORCH_CHECK_VALUE(weights.device() == dev && new_table.device() == dev, "All tensors must be on the same CUDA device.");
  const int64_t B = table.size(0), cap = table.size(1) * kp.size(2);
  TORCH_CHECK_VALUE(keep > 0 && keep <= INT32_MAX / 2 && recent >= 0 && first >= 0 && first + recent <= keep,
                    "keep must be positive and hold first + recent tokens.");
  TORCH_CHECK_VALUE(weights.scalar_type() == at::kFloat && weights.dim() == 2 && weights.size(0) == B &&
                        weights.size(1) >= cap && (weights.size(1) <= 1 || weights.stride(1) == 1),
                    "token_weights must be fp32 [batch, >= block_table.shape[1] * page_size] with contiguous rows.");
  TORCH_CHECK_VALUE(new_table.dim() == 2 && new_table.scalar_type() == at::kInt && new_table.size(0) == B &&
                        (new_table.size(1) <= 1 || new_table.stride(1) == 1),
                    "new_block_table must be int32 [batch, pages] with contiguous rows.");
  TORCH_CHECK_VALUE(new_table.size(1) * kp.size(2) >= std::min(keep, cap),
                    "new_block_table must hold pages for min(keep, block_table.shape[1] * page_size) tokens.");
  TORCH_CHECK_VALUE(cap <= 320000, "eviction takes block tables of up to 320000 tokens.");
  TORCH_CHECK_VALUE(kp.size(3) % 8 == 0, "head_dim must be a multiple of 8.");
  TORCH_CHECK_VALUE(!shares_memory(kp) && !shares_memory(vp), "pages that are written must not be expanded tensors.");
  c10::cuda::CUDAGuard guard(dev);
  const auto i32 = at::TensorOptions().dtype(at::kInt).device(dev);
  at::Tensor kept = at::empty({B, keep}, i32), new_lengths = at::empty({B}, i32);
  at::Tensor new_weights = at::empty({B, keep}, i32.dtype(at::kFloat));
  kvr_paged_evict_args a;
  std::memset(&a, 0, sizeof(a));
  a.key_pages = kp.data_ptr();
  a.key_page_stride = step(kp, 0), a.key_head_stride = step(kp, 1), a.key_row_stride = step(kp, 2);
  a.value_pages = vp.data_ptr();
  a.value_page_stride = step(vp, 0), a.value_head_stride = step(vp, 1), a.value_row_stride = step(vp, 2);
  a.block_table = table.data_ptr<int>(), a.table_stride = step(table, 0), a.table_width = (int)table.size(1);
  a.num_pages = (int)kp.size(0);
  a.new_block_table = new_table.data_ptr<int>(), a.new_table_stride = step(new_table, 0);
  a.new_table_width = (int)new_table.size(1);
  a.lengths = lengths.data_ptr<int>();
  a.token_weights = weights.data_ptr<float>(), a.weights_b_stride = step(weights, 0);
  a.kept = kept.data_ptr<int>(), a.new_lengths = new_lengths.data_ptr<int>(), a.new_weights = new_weights.data_ptr<float>();
  a.batch = (int)B, a.kv_heads = (int)kp.size(1), a.head_dim = (int)kp.size(3), a.page_size = (int)kp.size(2);
  a.keep = (int)keep, a.recent = (int)recent, a.first = (int)first;
  raise_status("kvr_paged_evict", kvr_paged_evict(&a, c10::cuda::getCurrentCUDAStream().stream()));
  return {kept, new_lengths, new_weights};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> verify_draft(const at::Tensor& target,
                                                            const std::optional<at::Tensor>& draft,
                                                            const at::Tensor& tokens,
                                                            const std::optional<at::Tensor>& uniforms,
                                                            const std::optional<at::Tensor>& noise,
                                                            double temperature,
                                                            const std::optional<at::Tensor>& draft_lengths) {
  const at::Device dev = target.device();
  TORCH_CHECK_VALUE(dev.is_cuda(), "kv_reduce_b200 operates on CUDA tensors only (no CPU fallback).");
  TORCH_CHECK_VALUE(target.dim() == 3 && target.size(1) > 0 && target.size(2) > 0,
                    "target_logits must be [batch, draft + 1, vocab].");
  const at::ScalarType type = target.scalar_type();
  TORCH_CHECK_VALUE(is_half_type(type) || type == at::kFloat, "logits must be bf16, fp16 or fp32.");
  const int64_t B = target.size(0), K = target.size(1) - 1, V = target.size(2);
  TORCH_CHECK_VALUE(V <= (1 << 30), "vocab must be at most 2^30.");
  TORCH_CHECK_VALUE(temperature >= 0 && std::isfinite(temperature), "temperature must be 0 or a positive finite number.");
  TORCH_CHECK_VALUE(tokens.device() == dev && tokens.dim() == 2 && tokens.size(0) == B && tokens.size(1) == K &&
                        (tokens.scalar_type() == at::kLong || tokens.scalar_type() == at::kInt),
                    "draft_tokens must be int64 or int32 [batch, draft] on the logits' device.");
  const bool greedy = temperature == 0;
  auto given = [](const std::optional<at::Tensor>& t) { return t.has_value() && t->defined(); };
  if (!greedy) {
    TORCH_CHECK_VALUE(given(draft) && given(uniforms) && given(noise),
                      "sampling (temperature > 0) needs draft_logits, uniforms and noise.");
    TORCH_CHECK_VALUE(draft->device() == dev && draft->scalar_type() == type && draft->dim() == 3 &&
                          draft->size(0) == B && draft->size(1) == K && draft->size(2) == V,
                      "draft_logits must be [batch, draft, vocab] of the target's dtype and device.");
    TORCH_CHECK_VALUE(uniforms->device() == dev && uniforms->scalar_type() == at::kFloat && uniforms->dim() == 2 &&
                          uniforms->size(0) == B && uniforms->size(1) == K,
                      "uniforms must be fp32 [batch, draft].");
    TORCH_CHECK_VALUE(noise->device() == dev && noise->scalar_type() == at::kFloat && noise->dim() == 2 &&
                          noise->size(0) == B && noise->size(1) == V,
                      "noise must be fp32 [batch, vocab].");
  }
  if (given(draft_lengths))
    TORCH_CHECK_VALUE(draft_lengths->device() == dev && draft_lengths->scalar_type() == at::kInt &&
                          draft_lengths->dim() == 1 && draft_lengths->size(0) == B &&
                          (B <= 1 || draft_lengths->stride(0) == 1),
                      "draft_lengths must be a contiguous int32 [batch] tensor.");
  c10::cuda::CUDAGuard guard(dev);
  const auto f32 = at::TensorOptions().dtype(at::kFloat).device(dev);
  at::Tensor out = at::empty({B, K + 1}, f32.dtype(at::kLong)), accepted = at::empty({B}, f32.dtype(at::kInt));
  at::Tensor prob = at::empty({B, K}, f32);
  if (B == 0) return {out, accepted, prob};
  // rows with contiguous elements, at any alignment; others are copied
  auto last_contiguous = [](const at::Tensor& t) {
    return t.size(t.dim() - 1) <= 1 || t.stride(t.dim() - 1) == 1 ? t : t.contiguous();
  };
  const at::Tensor t = last_contiguous(target), x = last_contiguous(tokens.to(at::kLong));
  at::Tensor d, u, e;
  kvr_verify_args a;
  std::memset(&a, 0, sizeof(a));
  a.target = t.data_ptr(), a.target_b_stride = step(t, 0), a.target_k_stride = step(t, 1);
  if (K > 0) a.tokens = x.data_ptr<int64_t>(), a.tokens_b_stride = step(x, 0);
  if (!greedy) {
    e = last_contiguous(*noise);
    a.noise = e.data_ptr<float>(), a.noise_b_stride = step(e, 0);
    if (K > 0) {
      d = last_contiguous(*draft), u = last_contiguous(*uniforms);
      a.draft = d.data_ptr(), a.draft_b_stride = step(d, 0), a.draft_k_stride = step(d, 1);
      a.uniforms = u.data_ptr<float>(), a.uniforms_b_stride = step(u, 0);
    }
  }
  if (given(draft_lengths)) a.draft_lengths = draft_lengths->data_ptr<int>();
  a.out_tokens = out.data_ptr<int64_t>(), a.accepted = accepted.data_ptr<int>();
  a.accept_prob = K > 0 ? prob.data_ptr<float>() : nullptr;
  a.dtype = type == at::kBFloat16 ? 0 : type == at::kHalf ? 1 : 2;
  a.batch = (int)B, a.draft_tokens = (int)K, a.vocab = (int)V;
  a.temperature = (float)temperature;
  TORCH_CHECK_VALUE(greedy || a.temperature >= FLT_MIN, "temperature is too small for fp32.");
  size_t zeroed = 0, ws = 0;
  raise_status("kvr_verify_plan", kvr_verify_plan(&a, &zeroed, &ws));
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream().stream();
  Lease s(Op::verify, dev, stream, (int64_t)ws, (int64_t)(zeroed + 3) / 4);
  a.zeroed = s.counters.data_ptr(), a.zeroed_bytes = (size_t)s.counters.numel() * 4;
  a.workspace = s.workspace.data_ptr(), a.workspace_bytes = (size_t)s.workspace.numel();
  raise_status("kvr_verify", s.launched(kvr_verify(&a, stream)));
  return {out, accepted, prob};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(kvr, m) {
  m.def("paged_append(Tensor key, Tensor value, Tensor(a!) key_pages, Tensor(b!) value_pages, Tensor block_table, "
        "Tensor lengths, Tensor? new_counts=None) -> ()");
  m.def("paged_attention(Tensor query, Tensor key_pages, Tensor value_pages, Tensor block_table, Tensor lengths, "
        "float? scale=None, int window=0, int sinks=0, Tensor(a!)? token_weights=None, bool return_lse=False, "
        "Tensor? new_counts=None) "
        "-> (Tensor, Tensor)");
  m.def("paged_evict(Tensor(a!) key_pages, Tensor(b!) value_pages, Tensor block_table, Tensor lengths, "
        "Tensor token_weights, Tensor new_block_table, int keep, int recent, int first) -> (Tensor, Tensor, Tensor)");
  m.def("verify_draft(Tensor target_logits, Tensor? draft_logits, Tensor draft_tokens, Tensor? uniforms, "
        "Tensor? noise, float temperature=1.0, Tensor? draft_lengths=None) -> (Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(kvr, CUDA, m) {
  m.impl("paged_append", &paged_append);
  m.impl("paged_attention", &paged_attention);
  m.impl("paged_evict", &paged_evict);
  m.impl("verify_draft", &verify_draft);
}

// Host tensors reach the same functions, whose first check raises ValueError.
TORCH_LIBRARY_IMPL(kvr, CPU, m) {
  m.impl("paged_append", &paged_append);
  m.impl("paged_attention", &paged_attention);
  m.impl("paged_evict", &paged_evict);
  m.impl("verify_draft", &verify_draft);
}
