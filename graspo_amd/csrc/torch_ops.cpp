// torch_ops.cpp -- thin PyTorch-ROCm binding of the C ABI (host-only C++).
//
// Registers torch.ops.graspo_tokpath.{sample, sample_route, sample_spread,
// logprob_entropy, token_logprob, token_logprob_backward, verdict_begin,
// verdict_end, logprob_backward, graspo_loss_*, lse_partial, lse_finalize,
// decode_update, to_bf16_exact, logprob_backward_split, time_next_launch,
// lm_head_logprob, lm_head_logprob_save, softmax_grad_bf16, linear_logprob,
// linear_logprob_backward, linear_loss, embedding, embedding_backward,
// token_embedding, grad_norm, clip_grads_, clip_grad_norm_, beam_candidates,
// beam_advance, beam_step, beam_finish, reorder_states_, expand_states,
// lora_add_state, lora_backward, lora_add}.  Each op validates
// its tensors (TORCH_CHECK surfaces as a Python RuntimeError), allocates the
// outputs on the logits' device, and enqueues the HIP kernels on the stream handle passed in from Python
// (torch.cuda.current_stream().cuda_stream), so work orders with the
// caller's other torch work exactly as the reference's ATen ops did.
#include <ATen/ATen.h>
#include <ATen/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/library.h>

#include <algorithm>
#include <limits>
#include <map>
#include <mutex>
#include <string>
#include <tuple>
#include <utility>
#include <vector>

#include "graspo_tokpath.h"

namespace {

int dtype_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat:
      return GTP_DTYPE_F32;
    case at::kBFloat16:
      return GTP_DTYPE_BF16;
    case at::kHalf:
      return GTP_DTYPE_F16;
    default:
      TORCH_CHECK(false, "graspo_tokpath: logits must be float32, bfloat16 or float16, got ",
                  t.scalar_type());
  }
  return -1;
}

void check_rc(int rc, const char* what) {
  TORCH_CHECK(rc == GTP_OK, "graspo_tokpath: ", what, " failed with code ", rc,
              rc == GTP_ERR_INVALID_ARGUMENT ? " (invalid argument)"
              : rc == GTP_ERR_UNSUPPORTED    ? " (unsupported shape)"
                                             : " (kernel launch error)");
}

void check_rows(const at::Tensor& logits, const char* name) {
  TORCH_CHECK(logits.is_cuda(), "graspo_tokpath: ", name, " must be a GPU tensor");
  TORCH_CHECK(logits.dim() == 2, "graspo_tokpath: ", name, " must be 2-D [rows, V], got ",
              logits.dim(), "-D");
  TORCH_CHECK(logits.size(1) == 0 || logits.stride(1) == 1, "graspo_tokpath: ", name,
              " rows must be contiguous (stride(-1) == 1)");
}

int64_t row_stride_of(const at::Tensor& logits) {
  return logits.size(0) > 1 ? logits.stride(0) : logits.size(1);
}

void check_same_device(const at::Tensor& a, const at::Tensor& b, const char* name) {
  TORCH_CHECK(b.device() == a.device(), "graspo_tokpath: ", name, " must be on ", a.device());
}

// Sampler workspace, one per (device, stream): zero-filled when allocated (the
// library keeps it reusable from call to call), grown when a call needs more.
// Calls on one stream are ordered, so they can share it.  One that has been
// outgrown is kept, for a captured graph may hold its address; a new one is
// at least twice as large, so all of them together stay below twice the last.
void* sampler_workspace(const at::Tensor& like, size_t bytes, int64_t stream) {
  if (bytes == 0) return nullptr;
  static std::mutex mu;
  static std::map<std::pair<int, int64_t>, std::vector<at::Tensor>> cache;
  std::lock_guard<std::mutex> lock(mu);
  std::vector<at::Tensor>& all = cache[{(int)like.get_device(), stream}];
  if (all.empty() || (size_t)all.back().numel() < bytes) {
    const size_t least = all.empty() ? 0 : 2 * (size_t)all.back().numel();
    const int64_t n = (int64_t)((std::max(bytes, least) + 4095) / 4096 * 4096);
    all.push_back(at::zeros({n}, like.options().dtype(at::kByte)));
  }
  return all.back().data_ptr();
}

// 16-byte aligned logits and row stride
bool rows_aligned(const at::Tensor& logits) {
  return (reinterpret_cast<uintptr_t>(logits.data_ptr()) & 15u) == 0 &&
         ((uint64_t)(row_stride_of(logits) * logits.element_size()) & 15u) == 0;
}

using SampleOut =
    std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor>;

SampleOut sample(const at::Tensor& logits, double temperature, int64_t top_k, double top_p,
                 double repetition_penalty, const c10::optional<at::Tensor>& history,
                 const c10::optional<at::Tensor>& allow_mask,
                 const c10::optional<at::Tensor>& uniforms,
                 const c10::optional<at::Tensor>& finished, int64_t pad_token_id, int64_t stream) {
  check_rows(logits, "logits");
  const int64_t B = logits.size(0), V = logits.size(1);
  TORCH_CHECK(V > 0, "graspo_tokpath.sample: empty vocabulary");
  TORCH_CHECK(V <= GTP_SAMPLER_MAX_V, "graspo_tokpath.sample: V = ", V, " exceeds ",
              GTP_SAMPLER_MAX_V);
  TORCH_CHECK(repetition_penalty > 0.0, "graspo_tokpath.sample: repetition_penalty must be > 0");
  TORCH_CHECK(top_k >= 0 && top_k <= INT32_MAX, "graspo_tokpath.sample: top_k must be >= 0");
  const int32_t* hist = nullptr;
  int64_t hist_len = 0, hist_stride = 0;
  if (history.has_value() && history->numel() > 0) {
    const auto& h = *history;
    check_same_device(logits, h, "history");
    TORCH_CHECK(h.scalar_type() == at::kInt && h.dim() == 2 && h.size(0) == B && h.stride(1) == 1,
                "graspo_tokpath.sample: history must be int32 [B, L] with contiguous rows");
    hist = h.data_ptr<int32_t>();
    hist_len = h.size(1);
    hist_stride = B > 1 ? h.stride(0) : hist_len;
  }
  const uint32_t* mask = nullptr;
  int64_t mask_stride = 0;
  if (allow_mask.has_value()) {
    const auto& m = *allow_mask;
    check_same_device(logits, m, "allow_mask");
    TORCH_CHECK((m.scalar_type() == at::kInt || m.scalar_type() == at::kUInt32) && m.dim() == 2 &&
                    m.size(0) == B && m.size(1) >= (V + 31) / 32 && m.stride(1) == 1,
                "graspo_tokpath.sample: allow_mask must be int32/uint32 [B, >= ceil(V/32)]");
    mask = static_cast<const uint32_t*>(m.data_ptr());
    mask_stride = B > 1 ? m.stride(0) : m.size(1);
  }
  const bool greedy = !(temperature > 0.0);
  const float* u = nullptr;
  if (uniforms.has_value()) {
    const auto& uu = *uniforms;
    check_same_device(logits, uu, "uniforms");
    TORCH_CHECK(uu.scalar_type() == at::kFloat && uu.dim() == 1 && uu.size(0) == B &&
                    uu.is_contiguous(),
                "graspo_tokpath.sample: uniforms must be float32 [B]");
    u = uu.data_ptr<float>();
  }
  TORCH_CHECK(greedy || u != nullptr, "graspo_tokpath.sample: uniforms are required when T > 0");
  const uint8_t* fin = nullptr;
  if (finished.has_value()) {
    const auto& f = *finished;
    check_same_device(logits, f, "finished");
    TORCH_CHECK((f.scalar_type() == at::kBool || f.scalar_type() == at::kByte) && f.dim() == 1 &&
                    f.size(0) == B && f.is_contiguous(),
                "graspo_tokpath.sample: finished must be bool/uint8 [B]");
    fin = static_cast<const uint8_t*>(f.data_ptr());
  }
  auto opt = logits.options();
  // Each output has a storage of its own (it can be saved, resized or handed
  // to another stream by itself).  Six of the seven come from the allocator
  // directly: a greedy call of one row, whose kernel takes 7 us, takes 12.1 us
  // with seven at::empty, 10.9 this way (9.4 as parts of one allocation).
  const at::Tensor ids = at::empty({B}, opt.dtype(at::kLong));
  c10::Allocator* const alloc = ids.storage().allocator();
  const c10::DeviceGuard guard(logits.device());
  auto output = [&](at::ScalarType type) {
    return at::Tensor(at::detail::empty_generic({B}, alloc, ids.key_set(), type, c10::nullopt));
  };
  const at::Tensor lp = output(at::kFloat), slp = output(at::kFloat), kept = output(at::kInt),
                   tv = output(at::kFloat), tid = output(at::kInt), st = output(at::kInt);
  gtp_sampler_params p;
  p.temperature = (float)temperature;
  p.top_k = (int32_t)top_k;
  p.top_p = (float)top_p;
  p.repetition_penalty = (float)repetition_penalty;
  const int dt = dtype_code(logits);
  const bool spread = gtp_sample_spread_wins(dt, B, V, rows_aligned(logits), hist_len,
                                             mask != nullptr, &p) != 0;
  at::Tensor own;  // the spread kernels' workspace carries nothing between calls
  const size_t ws_bytes = spread ? gtp_sample_spread_workspace_bytes(B, V, &p)
                                 : gtp_sample_workspace_bytes(dt, B, V, &p);
  if (spread) own = at::empty({(int64_t)ws_bytes}, opt.dtype(at::kByte));
  void* ws = spread ? own.data_ptr() : sampler_workspace(logits, ws_bytes, stream);
  const int rc = (spread ? gtp_sample_rows_spread : gtp_sample_rows)(
      logits.data_ptr(), dt, B, V, row_stride_of(logits), hist, hist_len,
      hist_stride, mask, mask_stride, u, &p, fin, pad_token_id, ids.data_ptr<int64_t>(),
      lp.data_ptr<float>(), slp.data_ptr<float>(), kept.data_ptr<int32_t>(), tv.data_ptr<float>(),
      tid.data_ptr<int32_t>(), st.data_ptr<int32_t>(), ws, ws_bytes,
      reinterpret_cast<void*>(stream));
  check_rc(rc, spread ? "gtp_sample_rows_spread" : "gtp_sample_rows");
  return {ids, lp, slp, kept, tv, tid, st};
}

// The kernel `sample` would run for these logits and parameters (with the
// workspace it would pass): (GTP_ROUTE_*, workgroups per row).
std::tuple<int64_t, int64_t> sample_route(const at::Tensor& logits, double temperature,
                                          int64_t top_k, double top_p, double repetition_penalty,
                                          int64_t hist_len, bool has_mask) {
  check_rows(logits, "logits");
  const int64_t B = logits.size(0), V = logits.size(1);
  TORCH_CHECK(B > 0 && V > 0 && V <= GTP_SAMPLER_MAX_V && top_k >= 0 && top_k <= INT32_MAX &&
                  hist_len >= 0,
              "graspo_tokpath.sample_route: bad shape or parameters");
  gtp_sampler_params p;
  p.temperature = (float)temperature;
  p.top_k = (int32_t)top_k;
  p.top_p = (float)top_p;
  p.repetition_penalty = (float)repetition_penalty;
  const int dt = dtype_code(logits);
  const size_t ws_bytes = gtp_sample_workspace_bytes(dt, B, V, &p);
  int32_t route = 0, slices = 0;
  check_rc(gtp_sample_route(dt, B, V, rows_aligned(logits) ? 1 : 0, hist_len, has_mask ? 1 : 0, &p, ws_bytes,
                            &route, &slices),
           "gtp_sample_route");
  return {route, slices};
}

// Whether `sample` runs the spread kernels for these logits and parameters
// (then not sample_route's).
bool sample_spread(const at::Tensor& logits, double temperature, int64_t top_k, double top_p,
                   double repetition_penalty, int64_t hist_len, bool has_mask) {
  check_rows(logits, "logits");
  gtp_sampler_params p;
  p.temperature = (float)temperature;
  p.top_k = (int32_t)top_k;
  p.top_p = (float)top_p;
  p.repetition_penalty = (float)repetition_penalty;
  return gtp_sample_spread_wins(dtype_code(logits), logits.size(0), logits.size(1),
                                rows_aligned(logits), hist_len, has_mask, &p) != 0;
}

const void* targets_ptr(const at::Tensor& logits, const at::Tensor& targets, int64_t N,
                        int* is64) {
  check_same_device(logits, targets, "targets");
  TORCH_CHECK((targets.scalar_type() == at::kInt || targets.scalar_type() == at::kLong) &&
                  targets.dim() == 1 && targets.size(0) == N && targets.is_contiguous(),
              "graspo_tokpath: targets must be int32/int64 [N] contiguous");
  *is64 = targets.scalar_type() == at::kLong;
  return targets.data_ptr();
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> logprob_entropy(const at::Tensor& logits,
                                                               const at::Tensor& targets,
                                                               int64_t stream) {
  check_rows(logits, "logits");
  const int64_t N = logits.size(0), V = logits.size(1);
  TORCH_CHECK(V > 0, "graspo_tokpath.logprob_entropy: empty vocabulary");
  int t64 = 0;
  const void* tp = targets_ptr(logits, targets, N, &t64);
  auto opt = logits.options();
  at::Tensor lp = at::empty({N}, opt.dtype(at::kFloat));
  at::Tensor H = at::empty({N}, opt.dtype(at::kFloat));
  at::Tensor st = at::empty({N}, opt.dtype(at::kInt));
  const int rc = gtp_logprob_entropy_rows(logits.data_ptr(), dtype_code(logits), N, V,
                                          row_stride_of(logits), tp, t64, lp.data_ptr<float>(),
                                          H.data_ptr<float>(), st.data_ptr<int32_t>(),
                                          reinterpret_cast<void*>(stream));
  check_rc(rc, "gtp_logprob_entropy_rows");
  return {lp, H, st};
}

// [S, V] or [B, S, V] logits with unit column stride and targets of their
// leading shape, each with its own strides.
gtp_token_rows token_rows(const at::Tensor& logits, const at::Tensor& targets,
                          const c10::optional<int64_t>& ignore_index) {
  TORCH_CHECK(logits.is_cuda(), "graspo_tokpath: logits must be a GPU tensor");
  const int64_t d = logits.dim();
  TORCH_CHECK((d == 2 || d == 3) && logits.size(d - 1) > 0 && (logits.size(d - 1) == 1 || logits.stride(d - 1) == 1),
              "graspo_tokpath: logits must be [S, V] or [B, S, V] with contiguous rows");
  check_same_device(logits, targets, "targets");
  TORCH_CHECK((targets.scalar_type() == at::kInt || targets.scalar_type() == at::kLong) &&
                  targets.dim() == d - 1 && targets.sizes() == logits.sizes().slice(0, d - 1),
              "graspo_tokpath: targets must be int32/int64 of the logits' leading shape");
  gtp_token_rows r;
  r.logits = logits.data_ptr();
  r.targets = targets.data_ptr();
  r.dtype = dtype_code(logits);
  r.targets_int64 = targets.scalar_type() == at::kLong;
  r.has_ignore = ignore_index.has_value();
  r.ignore_index = ignore_index.value_or(0);
  r.B = d == 3 ? logits.size(0) : 1;
  r.S = logits.size(d - 2);
  r.V = logits.size(d - 1);
  r.batch_stride = d == 3 ? logits.stride(0) : 0;
  r.row_stride = logits.stride(d - 2);
  r.target_batch_stride = d == 3 ? targets.stride(0) : 0;
  r.target_row_stride = targets.stride(d - 2);
  return r;
}

uint32_t* verdict_ptr(const at::Tensor& words) {
  return reinterpret_cast<uint32_t*>(words.data_ptr<int32_t>());
}

// Pinned words for a look at the targets, each of them pending.
at::Tensor verdict_words() {
  at::Tensor words = at::empty({GTP_VERDICT_WORDS},
                               at::TensorOptions().dtype(at::kInt).pinned_memory(true));
  for (int i = 0; i < GTP_VERDICT_WORDS; ++i) verdict_ptr(words)[i] = GTP_VERDICT_PENDING;
  return words;
}

// Waits for the words of a look that has been launched (or whose launch
// failed), before anything is raised: given back to the allocator while the
// kernel may still write them, they would answer for a later call.  Words
// whose wait fails are kept for good.
int verdict_wait(const at::Tensor& words, int* found, void* stream) {
  const int rc = gtp_verdict_wait(verdict_ptr(words), found, stream);
  if (rc != GTP_OK) new at::Tensor(words);
  return rc;
}

// (logprob, entropy or an empty tensor, mean loss, counted rows, whether a
// target lies outside [0, V)).  mean: also -sum(logprob) / count.  Waits for
// the look at the targets, which runs ahead of the rows, not for the rows.
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, bool> token_logprob(
    const at::Tensor& logits, const at::Tensor& targets, c10::optional<int64_t> ignore_index,
    bool entropy, bool mean, int64_t stream) {
  const gtp_token_rows r = token_rows(logits, targets, ignore_index);
  void* st = reinterpret_cast<void*>(stream);
  TORCH_CHECK(!gtp_stream_capturing(st),
              "graspo_tokpath.token_logprob: waits for the targets, so it cannot be captured");
  const int64_t N = r.B * r.S;
  const auto f32 = logits.options().dtype(at::kFloat);
  at::Tensor lp = at::empty(targets.sizes(), f32);
  at::Tensor H = at::empty({0}, f32), loss = H, count = H;
  if (entropy) H = at::empty(targets.sizes(), f32);
  if (mean) {
    loss = at::empty({}, f32);
    count = at::empty({}, f32.dtype(at::kLong));
  }
  const at::Tensor words = verdict_words();
  const size_t ws_bytes = gtp_token_logprob_workspace_bytes(r.dtype, N, r.V);
  at::Tensor ws;
  if (ws_bytes) ws = at::empty({(int64_t)ws_bytes}, logits.options().dtype(at::kByte));
  const int rc = gtp_token_logprob_rows(&r, lp.data_ptr<float>(),
                                        entropy ? H.data_ptr<float>() : nullptr, nullptr,
                                        verdict_ptr(words), ws_bytes ? ws.data_ptr() : nullptr,
                                        ws_bytes, st);
  // an argument error comes before any launch, a launch error after the look's
  if (rc != GTP_OK && rc != GTP_ERR_LAUNCH) check_rc(rc, "gtp_token_logprob_rows");
  const int mean_rc = mean ? gtp_token_mean_loss(&r, lp.data_ptr<float>(), loss.data_ptr<float>(),
                                                 count.data_ptr<int64_t>(), st)
                           : GTP_OK;
  int bad = 0;
  const int wait_rc = verdict_wait(words, &bad, st);
  check_rc(rc, "gtp_token_logprob_rows");
  check_rc(mean_rc, "gtp_token_mean_loss");
  check_rc(wait_rc, "gtp_verdict_wait");
  return {lp, H, loss, count, bad != 0};
}

// Queues the look at `targets` (against [0, V)) and at up to two device flags
// (a nonzero one: inexact), and returns the pinned words that it answers in.
at::Tensor verdict_begin(const at::Tensor& targets, int64_t V, const c10::optional<at::Tensor>& flag_a,
                         const c10::optional<at::Tensor>& flag_b, int64_t stream) {
  void* st = reinterpret_cast<void*>(stream);
  TORCH_CHECK(targets.is_cuda() && targets.dim() == 1 &&
                  (targets.scalar_type() == at::kInt || targets.scalar_type() == at::kLong),
              "graspo_tokpath.verdict_begin: targets must be an int32/int64 [N] GPU tensor");
  TORCH_CHECK(!gtp_stream_capturing(st),
              "graspo_tokpath.verdict_begin: the host waits for it, so it cannot be captured");
  const uint32_t* flags[2] = {nullptr, nullptr};
  int k = 0;
  for (const auto* f : {&flag_a, &flag_b}) {
    if (f->has_value()) {
      check_same_device(targets, **f, "flag");
      TORCH_CHECK((*f)->scalar_type() == at::kInt && (*f)->numel() == 1,
                  "graspo_tokpath.verdict_begin: flags must be int32 [1]");
      flags[k] = reinterpret_cast<const uint32_t*>((*f)->data_ptr<int32_t>());
    }
    ++k;
  }
  const at::Tensor words = verdict_words();
  const int rc = gtp_targets_verdict(targets.data_ptr(), targets.scalar_type() == at::kLong,
                                     targets.size(0), targets.stride(0), V, flags[0], flags[1],
                                     verdict_ptr(words), st);
  int found = 0;
  if (rc == GTP_ERR_LAUNCH) verdict_wait(words, &found, st);
  check_rc(rc, "gtp_targets_verdict");
  return words;
}

// Waits for verdict_begin's answer: 0, or 1 (a bad target) + 2 (a flag set).
int64_t verdict_end(const at::Tensor& words, int64_t stream) {
  TORCH_CHECK(words.device().is_cpu() && words.scalar_type() == at::kInt &&
                  words.numel() == GTP_VERDICT_WORDS && words.is_contiguous(),
              "graspo_tokpath.verdict_end: expected verdict_begin's words");
  int found = 0;
  check_rc(verdict_wait(words, &found, reinterpret_cast<void*>(stream)), "gtp_verdict_wait");
  return found;
}

// The gradient of token_logprob's logprobs by its logits, contiguous, of the
// logits' shape and dtype.  The first `targets.size(-1)` positions of each
// sequence have a target; mean_count: `grad` is the gradient of the mean.
at::Tensor token_logprob_backward(const at::Tensor& logits, const at::Tensor& targets,
                                  const at::Tensor& logprob, const at::Tensor& grad,
                                  const c10::optional<at::Tensor>& mean_count,
                                  c10::optional<int64_t> ignore_index, int64_t stream) {
  const int64_t d = logits.dim();
  TORCH_CHECK((d == 2 || d == 3) && targets.dim() == d - 1 &&
                  targets.size(d - 2) <= logits.size(d - 2),
              "graspo_tokpath.token_logprob_backward: bad shapes");
  const int64_t S = logits.size(d - 2), St = targets.size(d - 2);
  gtp_token_rows r = token_rows(logits.narrow(d - 2, 0, St), targets, ignore_index);
  r.logits = logits.data_ptr();
  r.S = S;  // positions St.. have no target: their gradient is zero
  const bool is_mean = mean_count.has_value();
  for (const at::Tensor* t : {&logprob, &grad}) {
    check_same_device(logits, *t, "logprob / grad");
    TORCH_CHECK(t->scalar_type() == at::kFloat && t->is_contiguous(),
                "graspo_tokpath.token_logprob_backward: logprob and grad must be contiguous float32");
  }
  TORCH_CHECK(logprob.numel() == targets.numel() &&
                  grad.numel() == (is_mean ? 1 : targets.numel()) &&
                  (!is_mean || (mean_count->scalar_type() == at::kLong && mean_count->numel() == 1)),
              "graspo_tokpath.token_logprob_backward: logprob, grad and mean_count must match the "
              "targets");
  if (is_mean) check_same_device(logits, *mean_count, "mean_count");
  at::Tensor out = at::empty(logits.sizes(), logits.options());
  check_rc(gtp_token_logprob_backward(&r, St, logprob.data_ptr<float>(), grad.data_ptr<float>(),
                                      is_mean ? mean_count->data_ptr<int64_t>() : nullptr,
                                      out.data_ptr(), S * r.V, r.V, reinterpret_cast<void*>(stream)),
           "gtp_token_logprob_backward");
  return out;
}

void lse_partial(const at::Tensor& logits, const c10::optional<at::Tensor>& targets,
                 int64_t col_offset, const at::Tensor& state, bool accumulate, int64_t stream) {
  check_rows(logits, "logits");
  const int64_t N = logits.size(0), Vc = logits.size(1);
  TORCH_CHECK(Vc > 0, "graspo_tokpath.lse_partial: empty chunk");
  check_same_device(logits, state, "state");
  TORCH_CHECK(state.scalar_type() == at::kFloat && state.dim() == 2 && state.size(0) == N &&
                  state.size(1) == 4 && state.is_contiguous(),
              "graspo_tokpath.lse_partial: state must be float32 [N, 4] contiguous");
  int t64 = 0;
  const void* tp = nullptr;
  if (targets.has_value()) tp = targets_ptr(logits, *targets, N, &t64);
  const int rc = gtp_lse_partial_rows(logits.data_ptr(), dtype_code(logits), N, Vc,
                                      row_stride_of(logits), col_offset, tp, t64,
                                      state.data_ptr<float>(), accumulate ? 1 : 0,
                                      reinterpret_cast<void*>(stream));
  check_rc(rc, "gtp_lse_partial_rows");
}

std::tuple<at::Tensor, at::Tensor> lse_finalize(const at::Tensor& state, int64_t stream) {
  TORCH_CHECK(state.is_cuda() && state.scalar_type() == at::kFloat && state.dim() == 2 &&
                  state.size(1) == 4 && state.is_contiguous(),
              "graspo_tokpath.lse_finalize: state must be a float32 [N, 4] GPU tensor");
  const int64_t N = state.size(0);
  at::Tensor lp = at::empty({N}, state.options());
  at::Tensor H = at::empty({N}, state.options());
  const int rc = gtp_lse_finalize_rows(state.data_ptr<float>(), N, lp.data_ptr<float>(),
                                       H.data_ptr<float>(), reinterpret_cast<void*>(stream));
  check_rc(rc, "gtp_lse_finalize_rows");
  return {lp, H};
}

at::Tensor logprob_backward(const at::Tensor& logits, const at::Tensor& targets,
                            const at::Tensor& grad_logprob, const at::Tensor& lse,
                            int64_t col_offset, const c10::optional<at::Tensor>& out,
                            int64_t stream) {
  check_rows(logits, "logits");
  const int64_t N = logits.size(0), V = logits.size(1);
  TORCH_CHECK(V > 0, "graspo_tokpath.logprob_backward: empty vocabulary");
  int t64 = 0;
  const void* tp = targets_ptr(logits, targets, N, &t64);
  for (const at::Tensor* t : {&grad_logprob, &lse}) {
    check_same_device(logits, *t, "grad_logprob / lse");
    TORCH_CHECK(t->scalar_type() == at::kFloat && t->dim() == 1 && t->size(0) == N &&
                    t->is_contiguous(),
                "graspo_tokpath.logprob_backward: grad_logprob and lse must be float32 [N] "
                "contiguous");
  }
  at::Tensor grad;
  if (out.has_value()) {
    grad = *out;
    check_same_device(logits, grad, "out");
    TORCH_CHECK(grad.scalar_type() == logits.scalar_type() && grad.dim() == 2 &&
                    grad.size(0) == N && grad.size(1) == V && (V == 1 || grad.stride(1) == 1) &&
                    grad.stride(0) >= V,
                "graspo_tokpath.logprob_backward: out must be [N, V] of the logits' dtype "
                "with unit column stride");
  } else {
    grad = at::empty({N, V}, logits.options());
  }
  const int64_t gstride = N > 1 ? grad.stride(0) : V;
  const int rc = gtp_logprob_backward_rows(
      logits.data_ptr(), dtype_code(logits), N, V, row_stride_of(logits), col_offset, tp, t64,
      grad_logprob.data_ptr<float>(), lse.data_ptr<float>(), grad.data_ptr(), gstride,
      reinterpret_cast<void*>(stream));
  check_rc(rc, "gtp_logprob_backward_rows");
  return grad;
}

void check_loss_input(const at::Tensor& t, const at::Tensor& ref, const char* name) {
  check_same_device(ref, t, name);
  TORCH_CHECK(t.scalar_type() == at::kFloat && t.is_contiguous() && t.sizes() == ref.sizes(),
              "graspo_tokpath.graspo_loss: ", name, " must be float32, contiguous, of the shape "
              "of log_probs");
}

// fp32 weights or bool / uint8 0-1 bytes, of the shape of log_probs
const void* loss_mask(const c10::optional<at::Tensor>& mask, const at::Tensor& logp, int* u8) {
  *u8 = 0;
  if (!mask.has_value()) return nullptr;
  const at::Tensor& m = *mask;
  check_same_device(logp, m, "action_mask");
  TORCH_CHECK((m.scalar_type() == at::kFloat || m.scalar_type() == at::kBool ||
               m.scalar_type() == at::kByte) &&
                  m.is_contiguous() && m.sizes() == logp.sizes(),
              "graspo_tokpath.graspo_loss: action_mask must be float32, bool or uint8, "
              "contiguous, of the shape of log_probs");
  *u8 = m.scalar_type() != at::kFloat;
  return m.data_ptr();
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> graspo_loss_forward(
    const at::Tensor& logp, const at::Tensor& old_logp, const at::Tensor& adv,
    const c10::optional<at::Tensor>& mask, double clip_lo, double clip_hi, int64_t stream) {
  TORCH_CHECK(logp.is_cuda() && logp.dim() == 2 && logp.size(0) > 0 && logp.size(1) > 0,
              "graspo_tokpath.graspo_loss: log_probs must be a non-empty [B, T] GPU tensor");
  check_loss_input(logp, logp, "log_probs");
  check_loss_input(old_logp, logp, "old_log_probs");
  check_loss_input(adv, logp, "advantages");
  int mu8 = 0;
  const void* mp = loss_mask(mask, logp, &mu8);
  const int64_t B = logp.size(0), T = logp.size(1);
  at::Tensor loss = at::empty({}, logp.options());
  at::Tensor per_seq = at::empty({B}, logp.options());
  at::Tensor inv_den = at::empty({B}, logp.options());
  const int rc = gtp_graspo_loss_forward(
      logp.data_ptr<float>(), old_logp.data_ptr<float>(), adv.data_ptr<float>(), mp, mu8, B, T,
      (float)clip_lo, (float)clip_hi, loss.data_ptr<float>(), per_seq.data_ptr<float>(),
      inv_den.data_ptr<float>(), reinterpret_cast<void*>(stream));
  check_rc(rc, "gtp_graspo_loss_forward");
  return {loss, per_seq, inv_den};
}

at::Tensor graspo_loss_backward(const at::Tensor& logp, const at::Tensor& old_logp,
                                const at::Tensor& adv, const c10::optional<at::Tensor>& mask,
                                const at::Tensor& inv_denom, const at::Tensor& grad_loss,
                                double clip_lo, double clip_hi, int64_t stream) {
  check_loss_input(old_logp, logp, "old_log_probs");
  check_loss_input(adv, logp, "advantages");
  int mu8 = 0;
  const void* mp = loss_mask(mask, logp, &mu8);
  const int64_t B = logp.size(0), T = logp.size(1);
  TORCH_CHECK(inv_denom.scalar_type() == at::kFloat && inv_denom.numel() == B &&
                  grad_loss.scalar_type() == at::kFloat && grad_loss.numel() == 1,
              "graspo_tokpath.graspo_loss_backward: bad inv_denom / grad_loss");
  at::Tensor grad = at::empty_like(logp);
  const int rc = gtp_graspo_loss_backward(
      logp.data_ptr<float>(), old_logp.data_ptr<float>(), adv.data_ptr<float>(), mp, mu8,
      inv_denom.data_ptr<float>(), grad_loss.data_ptr<float>(), B, T, (float)clip_lo,
      (float)clip_hi, grad.data_ptr<float>(), reinterpret_cast<void*>(stream));
  check_rc(rc, "gtp_graspo_loss_backward");
  return grad;
}

// one [B] byte flag tensor (bool or uint8) or a [B, >col] column target
uint8_t* byte_arg(const at::Tensor& t, const at::Tensor& ids, const char* name) {
  check_same_device(ids, t, name);
  TORCH_CHECK(t.scalar_type() == at::kBool || t.scalar_type() == at::kByte,
              "graspo_tokpath.decode_update: ", name, " must be bool or uint8");
  return static_cast<uint8_t*>(t.data_ptr());
}

void decode_update(const at::Tensor& ids, const c10::optional<at::Tensor>& status,
                   const at::Tensor& finished, int64_t eos_token_id, int64_t pad_token_id,
                   const c10::optional<at::Tensor>& seq, const c10::optional<at::Tensor>& attn,
                   int64_t col, const at::Tensor& flags, int64_t stream) {
  TORCH_CHECK(ids.is_cuda(), "graspo_tokpath.decode_update: ids must be a GPU tensor");
  TORCH_CHECK(ids.scalar_type() == at::kLong && ids.dim() == 1 && ids.is_contiguous(),
              "graspo_tokpath.decode_update: ids must be int64 [B]");
  const int64_t B = ids.size(0);
  TORCH_CHECK(finished.dim() == 1 && finished.size(0) == B && finished.is_contiguous(),
              "graspo_tokpath.decode_update: finished must be [B], contiguous");
  uint8_t* fin = byte_arg(finished, ids, "finished");
  const int32_t* st = nullptr;
  if (status.has_value()) {
    check_same_device(ids, *status, "status");
    TORCH_CHECK(status->scalar_type() == at::kInt && status->numel() == B && status->is_contiguous(),
                "graspo_tokpath.decode_update: status must be int32 [B]");
    st = status->data_ptr<int32_t>();
  }
  int64_t* sp = nullptr;
  int64_t s_stride = 0;
  if (seq.has_value()) {
    const auto& s = *seq;
    check_same_device(ids, s, "sequences");
    TORCH_CHECK(s.scalar_type() == at::kLong && s.dim() == 2 && s.size(0) == B &&
                    s.size(1) > col && (B <= 1 || s.stride(1) == 1),
                "graspo_tokpath.decode_update: sequences must be int64 [B, > col] with "
                "contiguous rows");
    sp = s.data_ptr<int64_t>();
    s_stride = B > 1 ? s.stride(0) : s.size(1);
  }
  uint8_t* ap = nullptr;
  int64_t a_stride = 0;
  if (attn.has_value()) {
    const auto& a = *attn;
    ap = byte_arg(a, ids, "attention_mask");
    TORCH_CHECK(a.dim() == 2 && a.size(0) == B && a.size(1) > col && (B <= 1 || a.stride(1) == 1),
                "graspo_tokpath.decode_update: attention_mask must be [B, > col] with contiguous "
                "rows");
    a_stride = B > 1 ? a.stride(0) : a.size(1);
  }
  check_same_device(ids, flags, "flags");
  TORCH_CHECK(flags.scalar_type() == at::kInt && flags.numel() >= 2 && flags.is_contiguous(),
              "graspo_tokpath.decode_update: flags must be int32 [2]");
  const int rc = gtp_decode_update_rows(ids.data_ptr<int64_t>(), st, B, eos_token_id,
                                        pad_token_id, fin, sp, s_stride, ap, a_stride, col,
                                        flags.data_ptr<int32_t>(), reinterpret_cast<void*>(stream));
  check_rc(rc, "gtp_decode_update_rows");
}

// (hi, lo) bf16 parts of the logprob gradient of fp32 logits [N, V]
std::tuple<at::Tensor, at::Tensor> logprob_backward_split(const at::Tensor& logits,
                                                          const at::Tensor& targets,
                                                          const at::Tensor& grad_logprob,
                                                          const at::Tensor& lse,
                                                          int64_t col_offset, int64_t stream) {
  check_rows(logits, "logits");
  TORCH_CHECK(logits.scalar_type() == at::kFloat,
              "graspo_tokpath.logprob_backward_split: logits must be float32");
  const int64_t N = logits.size(0), V = logits.size(1);
  check_same_device(logits, targets, "targets");
  check_same_device(logits, grad_logprob, "grad_logprob");
  check_same_device(logits, lse, "lse");
  TORCH_CHECK((targets.scalar_type() == at::kInt || targets.scalar_type() == at::kLong) &&
                  targets.numel() == N && targets.is_contiguous(),
              "graspo_tokpath.logprob_backward_split: targets must be int32/int64 [N]");
  TORCH_CHECK(grad_logprob.scalar_type() == at::kFloat && grad_logprob.numel() == N &&
                  grad_logprob.is_contiguous() && lse.scalar_type() == at::kFloat &&
                  lse.numel() == N && lse.is_contiguous(),
              "graspo_tokpath.logprob_backward_split: grad_logprob and lse must be float32 [N]");
  at::Tensor hi = at::empty({N, V}, logits.options().dtype(at::kBFloat16));
  at::Tensor lo = at::empty({N, V}, logits.options().dtype(at::kBFloat16));
  const int rc = gtp_logprob_backward_split_rows(
      logits.data_ptr<float>(), N, V, row_stride_of(logits), col_offset, targets.data_ptr(),
      targets.scalar_type() == at::kLong ? 1 : 0, grad_logprob.data_ptr<float>(),
      lse.data_ptr<float>(), static_cast<uint16_t*>(hi.data_ptr()),
      static_cast<uint16_t*>(lo.data_ptr()), V, reinterpret_cast<void*>(stream));
  check_rc(rc, "gtp_logprob_backward_split_rows");
  return {hi, lo};
}

// bf16 copy of a contiguous fp32 tensor, and whether any value was not a bf16
// value (a device flag the caller reads)
std::tuple<at::Tensor, at::Tensor> to_bf16_exact(const at::Tensor& src, int64_t stream) {
  TORCH_CHECK(src.is_cuda(), "graspo_tokpath.to_bf16_exact: src must be a GPU tensor");
  TORCH_CHECK(src.scalar_type() == at::kFloat && src.is_contiguous(),
              "graspo_tokpath.to_bf16_exact: src must be a contiguous float32 tensor");
  at::Tensor dst = at::empty(src.sizes(), src.options().dtype(at::kBFloat16));
  at::Tensor flag = at::zeros({1}, src.options().dtype(at::kInt));
  const int rc = gtp_f32_to_bf16_exact(src.data_ptr<float>(), src.numel(),
                                       static_cast<uint16_t*>(dst.data_ptr()),
                                       reinterpret_cast<uint32_t*>(flag.data_ptr<int32_t>()),
                                       reinterpret_cast<void*>(stream));
  check_rc(rc, "gtp_f32_to_bf16_exact");
  return {dst, flag};
}

}  // namespace

void time_next_launch(int64_t start_event, int64_t stop_event) {
  TORCH_CHECK(start_event != 0 && stop_event != 0,
              "graspo_tokpath.time_next_launch: both events must exist (record them once first)");
  check_rc(gtp_time_next_launch(reinterpret_cast<void*>(start_event),
                                reinterpret_cast<void*>(stop_event)),
           "gtp_time_next_launch");
}

// logprob / entropy / lse of h W^T rows without the [N, V] logits: bf16
// hidden [N, K] and weight [V, K] (rows contiguous, 16-byte aligned, K a
// multiple of 128), targets int32/int64 [N].
std::tuple<at::Tensor, at::Tensor, at::Tensor> lm_head_logprob(const at::Tensor& hidden,
                                                               const at::Tensor& weight,
                                                               const at::Tensor& targets,
                                                               int64_t stream) {
  for (const at::Tensor* t : {&hidden, &weight}) {
    TORCH_CHECK(t->is_cuda(), "graspo_tokpath.lm_head_logprob: hidden / weight must be GPU tensors");
    TORCH_CHECK(t->scalar_type() == at::kBFloat16 && t->dim() == 2 && t->stride(1) == 1,
                "graspo_tokpath.lm_head_logprob: hidden / weight must be bfloat16 2-D with "
                "contiguous rows");
  }
  check_same_device(hidden, weight, "weight");
  const int64_t N = hidden.size(0), K = hidden.size(1), V = weight.size(0);
  TORCH_CHECK(weight.size(1) == K, "graspo_tokpath.lm_head_logprob: hidden is [N, ", K,
              "] but weight is [V, ", weight.size(1), "]");
  int t64 = 0;
  const void* tp = targets_ptr(hidden, targets, N, &t64);
  at::Tensor lp = at::empty({N}, hidden.options().dtype(at::kFloat));
  at::Tensor H = at::empty({N}, lp.options());
  at::Tensor lse = at::empty({N}, lp.options());
  const size_t ws_bytes = gtp_lm_head_workspace_bytes(N, V);
  at::Tensor ws = at::empty({(int64_t)ws_bytes}, hidden.options().dtype(at::kByte));
  const int64_t ldh = N > 1 ? hidden.stride(0) : K, ldw = V > 1 ? weight.stride(0) : K;
  const int rc = gtp_lm_head_logprob_rows(
      reinterpret_cast<const uint16_t*>(hidden.data_ptr()), N, K, ldh,
      reinterpret_cast<const uint16_t*>(weight.data_ptr()), V, ldw, tp, t64, lp.data_ptr<float>(),
      H.data_ptr<float>(), lse.data_ptr<float>(), nullptr, ws.data_ptr(), ws_bytes,
      reinterpret_cast<void*>(stream));
  check_rc(rc, "gtp_lm_head_logprob_rows");
  return {lp, H, lse};
}

// Row length of the backward's [V, N] and [N, V] arrays: a multiple of 8
// elements, so that their rows take 16-byte accesses whatever the counts.
// 535 tokens of 151936 logits: the softmax pass 317 us on rows of 535, 133 on
// rows of 536.
int64_t padded(int64_t n) { return (n + 7) / 8 * 8; }

// lm_head_logprob that also keeps the fp32 logits, vocabulary-major [V, N],
// and returns the per-row status, for the backward.
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> lm_head_logprob_save(
    const at::Tensor& hidden, const at::Tensor& weight, const at::Tensor& targets,
    int64_t stream) {
  for (const at::Tensor* t : {&hidden, &weight}) {
    TORCH_CHECK(t->is_cuda(),
                "graspo_tokpath.lm_head_logprob_save: hidden / weight must be GPU tensors");
    TORCH_CHECK(t->scalar_type() == at::kBFloat16 && t->dim() == 2 && t->stride(1) == 1,
                "graspo_tokpath.lm_head_logprob_save: hidden / weight must be bfloat16 2-D "
                "with contiguous rows");
  }
  check_same_device(hidden, weight, "weight");
  const int64_t N = hidden.size(0), K = hidden.size(1), V = weight.size(0);
  TORCH_CHECK(weight.size(1) == K, "graspo_tokpath.lm_head_logprob_save: hidden is [N, ", K,
              "] but weight is [V, ", weight.size(1), "]");
  int t64 = 0;
  const void* tp = targets_ptr(hidden, targets, N, &t64);
  at::Tensor lp = at::empty({N}, hidden.options().dtype(at::kFloat));
  at::Tensor lse = at::empty({N}, lp.options());
  at::Tensor status = at::empty({N}, lp.options().dtype(at::kInt));
  at::Tensor logits_t = at::empty({V, padded(N)}, lp.options()).narrow(1, 0, N);
  const size_t ws_bytes = gtp_lm_head_workspace_bytes(N, V);
  at::Tensor ws = at::empty({(int64_t)ws_bytes}, hidden.options().dtype(at::kByte));
  const int64_t ldh = N > 1 ? hidden.stride(0) : K, ldw = V > 1 ? weight.stride(0) : K;
  const int rc = gtp_lm_head_logprob_save_rows(
      reinterpret_cast<const uint16_t*>(hidden.data_ptr()), N, K, ldh,
      reinterpret_cast<const uint16_t*>(weight.data_ptr()), V, ldw, tp, t64, lp.data_ptr<float>(),
      nullptr, lse.data_ptr<float>(), status.data_ptr<int32_t>(), logits_t.data_ptr<float>(),
      padded(N), ws.data_ptr(), ws_bytes, reinterpret_cast<void*>(stream));
  check_rc(rc, "gtp_lm_head_logprob_save_rows");
  return {lp, lse, logits_t, status};
}

// bf16(-g * softmax) of vocabulary-major fp32 logits [V, N] (row stride
// free, unit column stride), g and lse fp32 [N]; returns ([V, N] bf16 or an
// empty tensor, [N, V] bf16 or an empty tensor) as `layouts` asks (1:
// vocabulary-major, 2: token-major, 3: both)
std::tuple<at::Tensor, at::Tensor> softmax_grad_bf16(const at::Tensor& logits_t,
                                                     const at::Tensor& grad_logprob,
                                                     const at::Tensor& lse, int64_t layouts,
                                                     int64_t stream) {
  TORCH_CHECK(logits_t.is_cuda() && logits_t.scalar_type() == at::kFloat && logits_t.dim() == 2 &&
                  (logits_t.size(1) <= 1 || logits_t.stride(1) == 1),
              "graspo_tokpath.softmax_grad_bf16: logits_t must be a float32 [V, N] GPU tensor "
              "with unit column stride");
  const int64_t V = logits_t.size(0), N = logits_t.size(1);
  check_same_device(logits_t, grad_logprob, "grad_logprob");
  check_same_device(logits_t, lse, "lse");
  TORCH_CHECK(grad_logprob.scalar_type() == at::kFloat && grad_logprob.numel() == N &&
                  grad_logprob.is_contiguous() && lse.scalar_type() == at::kFloat &&
                  lse.numel() == N && lse.is_contiguous(),
              "graspo_tokpath.softmax_grad_bf16: grad_logprob and lse must be float32 [N]");
  TORCH_CHECK(layouts >= 1 && layouts <= 3, "graspo_tokpath.softmax_grad_bf16: layouts must be 1, 2 or 3");
  const auto bf = logits_t.options().dtype(at::kBFloat16);
  at::Tensor out_t = (layouts & 1) ? at::empty({V, padded(N)}, bf).narrow(1, 0, N) : at::empty({0}, bf);
  at::Tensor out_n = (layouts & 2) ? at::empty({N, padded(V)}, bf).narrow(1, 0, V) : at::empty({0}, bf);
  if (V == 0 || N == 0) return {out_t, out_n};
  const int64_t ld = V > 1 ? logits_t.stride(0) : N;
  const int rc = gtp_softmax_grad_bf16_cols(
      logits_t.data_ptr<float>(), V, N, ld, grad_logprob.data_ptr<float>(),
      lse.data_ptr<float>(), (layouts & 1) ? static_cast<uint16_t*>(out_t.data_ptr()) : nullptr,
      padded(N), (layouts & 2) ? static_cast<uint16_t*>(out_n.data_ptr()) : nullptr, padded(V),
      reinterpret_cast<void*>(stream));
  check_rc(rc, "gtp_softmax_grad_bf16_cols");
  return {out_t, out_n};
}

// ------------------------------------------------- the hidden-state losses

// The weight with rows that the kernels read in place: unit column stride,
// 16-byte aligned rows, whole 16-byte chunks.  Another one is copied into
// such rows (zeros behind the last column).
at::Tensor linear_weight(const at::Tensor& weight) {
  const int64_t V = weight.size(0), K = weight.size(1);
  const int64_t ld = V > 1 ? weight.stride(0) : K;
  if ((K <= 1 || weight.stride(1) == 1) && K % 8 == 0 && ld >= K && ld % 8 == 0 && ld < (1 << 22) &&
      (reinterpret_cast<uintptr_t>(weight.data_ptr()) & 15u) == 0)
    return weight;
  const int64_t K8 = (K + 7) / 8 * 8;
  at::Tensor rows = at::empty({V, K8}, weight.options());
  if (K8 > K) rows.narrow(1, K, K8 - K).zero_();
  rows.narrow(1, 0, K).copy_(weight);
  return rows;
}

// hidden [B, S, K] (unit column stride), weight [V, K] (linear_weight's) and
// targets [B, T <= S]
gtp_linear_rows linear_rows(const at::Tensor& hidden, const at::Tensor& weight, int64_t K,
                            const at::Tensor& targets, const c10::optional<int64_t>& ignore_index) {
  gtp_linear_rows r;
  r.hidden = hidden.data_ptr();
  r.weight = weight.data_ptr();
  r.targets = targets.data_ptr();
  r.dtype = dtype_code(hidden);
  r.targets_int64 = targets.scalar_type() == at::kLong;
  r.has_ignore = ignore_index.has_value();
  r.ignore_index = ignore_index.value_or(0);
  r.B = hidden.size(0);
  r.S = hidden.size(1);
  r.T = targets.size(1);
  r.K = K;
  r.V = weight.size(0);
  r.hidden_batch_stride = hidden.stride(0);
  r.hidden_row_stride = hidden.stride(1);
  r.weight_stride = r.V > 1 ? weight.stride(0) : weight.size(1);
  r.target_batch_stride = targets.stride(0);
  r.target_row_stride = targets.stride(1);
  return r;
}

void check_linear(const at::Tensor& hidden, const at::Tensor& weight, const at::Tensor& targets,
                  const char* what) {
  TORCH_CHECK(hidden.is_cuda() && hidden.dim() == 3 && weight.dim() == 2 && targets.dim() == 2,
              "graspo_tokpath.", what, ": expected hidden [B, S, K], weight [V, K] and targets "
              "[B, T] on a GPU");
  check_same_device(hidden, weight, "weight");
  check_same_device(hidden, targets, "targets");
  TORCH_CHECK((hidden.scalar_type() == at::kBFloat16 || hidden.scalar_type() == at::kHalf) &&
                  weight.scalar_type() == hidden.scalar_type(),
              "graspo_tokpath.", what, ": hidden and weight must both be bfloat16 or both float16, "
              "got ", hidden.scalar_type(), " and ", weight.scalar_type());
  TORCH_CHECK(targets.scalar_type() == at::kInt || targets.scalar_type() == at::kLong,
              "graspo_tokpath.", what, ": targets must be int32 or int64");
  TORCH_CHECK(hidden.size(2) > 0 && weight.size(0) > 0 && weight.size(1) == hidden.size(2),
              "graspo_tokpath.", what, ": hidden is [B, S, ", hidden.size(2), "] but weight is [",
              weight.size(0), ", ", weight.size(1), "]");
  TORCH_CHECK(targets.size(0) == hidden.size(0) && targets.size(1) <= hidden.size(1),
              "graspo_tokpath.", what, ": targets must be [B, T] with T <= S");
}

at::Tensor unit_columns(const at::Tensor& t) {
  return t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous();
}

// (logprob [B, T], lse [B, T], mean loss and count or empty tensors, whether a
// target lies outside [0, V)).  Waits for the look at the targets, which runs
// ahead of the products; a captured call does not (a bad target's logprob, and
// the mean with it, is NaN).
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, bool> linear_logprob(
    const at::Tensor& hidden_, const at::Tensor& weight_, const at::Tensor& targets,
    c10::optional<int64_t> ignore_index, bool mean, int64_t stream) {
  check_linear(hidden_, weight_, targets, "linear_logprob");
  const c10::DeviceGuard guard(hidden_.device());
  const at::Tensor hidden = unit_columns(hidden_), weight = linear_weight(weight_);
  const gtp_linear_rows r = linear_rows(hidden, weight, hidden.size(2), targets, ignore_index);
  void* st = reinterpret_cast<void*>(stream);
  const auto f32 = hidden.options().dtype(at::kFloat);
  at::Tensor lp = at::empty(targets.sizes(), f32), lse = at::empty(targets.sizes(), f32);
  at::Tensor loss = at::empty({0}, f32), count = at::empty({0}, f32.dtype(at::kLong));
  if (mean) {
    loss = at::empty({}, f32);
    count = at::empty({}, f32.dtype(at::kLong));
  }
  const size_t ws_bytes = gtp_linear_logprob_workspace_bytes(&r);
  at::Tensor ws = at::empty({(int64_t)std::max<size_t>(ws_bytes, 256)},
                            hidden.options().dtype(at::kByte));
  at::Tensor words;
  if (!gtp_stream_capturing(st)) words = verdict_words();
  const int rc = gtp_linear_logprob_rows(
      &r, lp.data_ptr<float>(), lse.data_ptr<float>(), mean ? loss.data_ptr<float>() : nullptr,
      mean ? count.data_ptr<int64_t>() : nullptr, words.defined() ? verdict_ptr(words) : nullptr,
      ws.data_ptr(), (size_t)ws.numel(), st);
  // an argument error comes before any launch, a launch error after the look's
  if (rc != GTP_OK && rc != GTP_ERR_LAUNCH) check_rc(rc, "gtp_linear_logprob_rows");
  int bad = 0, wait_rc = GTP_OK;
  if (words.defined()) wait_rc = verdict_wait(words, &bad, st);
  check_rc(rc, "gtp_linear_logprob_rows");
  check_rc(wait_rc, "gtp_verdict_wait");
  return {lp, lse, loss, count, bad != 0};
}

// The gradients of sum(grad * logprob) (mean_count: of grad times the mean)
// by hidden and weight, of their shapes and type, contiguous; an empty tensor
// for one that is not asked for.
std::tuple<at::Tensor, at::Tensor> linear_logprob_backward(
    const at::Tensor& hidden_, const at::Tensor& weight_, const at::Tensor& targets,
    const at::Tensor& lse, const at::Tensor& grad, const c10::optional<at::Tensor>& mean_count,
    c10::optional<int64_t> ignore_index, bool need_hidden, bool need_weight, int64_t stream) {
  check_linear(hidden_, weight_, targets, "linear_logprob_backward");
  const bool is_mean = mean_count.has_value();
  for (const at::Tensor* t : {&lse, &grad}) {
    check_same_device(hidden_, *t, "lse / grad");
    TORCH_CHECK(t->scalar_type() == at::kFloat && t->is_contiguous(),
                "graspo_tokpath.linear_logprob_backward: lse and grad must be contiguous float32");
  }
  TORCH_CHECK(lse.numel() == targets.numel() && grad.numel() == (is_mean ? 1 : targets.numel()) &&
                  (!is_mean || (mean_count->scalar_type() == at::kLong && mean_count->numel() == 1)),
              "graspo_tokpath.linear_logprob_backward: lse, grad and mean_count must match the "
              "targets");
  if (is_mean) check_same_device(hidden_, *mean_count, "mean_count");
  const c10::DeviceGuard guard(hidden_.device());
  at::Tensor gh = need_hidden ? at::empty(hidden_.sizes(), hidden_.options())
                              : at::empty({0}, hidden_.options());
  at::Tensor gw = need_weight ? at::empty(weight_.sizes(), weight_.options())
                              : at::empty({0}, weight_.options());
  if (targets.numel() == 0) return {gh.zero_(), gw.zero_()};
  if (!need_hidden && !need_weight) return {gh, gw};
  const at::Tensor hidden = unit_columns(hidden_), weight = linear_weight(weight_);
  const gtp_linear_rows r = linear_rows(hidden, weight, hidden.size(2), targets, ignore_index);
  const size_t ws_bytes = gtp_linear_logprob_backward_workspace_bytes(&r);
  at::Tensor ws = at::empty({(int64_t)std::max<size_t>(ws_bytes, 256)},
                            hidden.options().dtype(at::kByte));
  check_rc(gtp_linear_logprob_backward(
               &r, lse.data_ptr<float>(), grad.data_ptr<float>(),
               is_mean ? mean_count->data_ptr<int64_t>() : nullptr,
               need_hidden ? gh.data_ptr() : nullptr, need_weight ? gw.data_ptr() : nullptr,
               ws.data_ptr(), (size_t)ws.numel(), reinterpret_cast<void*>(stream)),
           "gtp_linear_logprob_backward");
  return {gh, gw};
}

// A gradient that raises where it is differentiated itself.
at::Tensor once_only(at::Tensor grad, const at::Tensor& from, const char* what) {
  if (!grad.defined() || !at::GradMode::is_enabled() || !from.requires_grad()) return grad;
  grad.requires_grad_();
  return (*std::make_shared<torch::autograd::DelayedError>(
      std::string(what) + " is differentiable once only", 1))({grad})[0];
}

// The nodes have no forward-mode derivative: an operand with a tangent is
// refused, which a call that needs no backward would drop without a word.
void check_no_tangent(const at::Tensor& t, const char* what) {
  TORCH_CHECK(!c10::AutogradState::get_tls_state().get_fw_grad_mode() || !t._fw_grad(0).defined(),
              what, ": forward-mode derivatives are not supported");
}

// In a graph capture: the accumulator of a leaf's gradient runs on the stream
// that it was made on, so while an eager graph of the leaf lives that was made
// on the default stream, which cannot join a capture, a captured backward ends
// the process.  (Another stream joins it.)
void check_leaf(const at::Tensor& leaf, const char* what, int64_t stream) {
  if (!leaf.requires_grad() || !leaf.is_leaf() ||
      !gtp_stream_capturing(reinterpret_cast<void*>(stream)))
    return;
  const auto node = torch::autograd::impl::try_get_grad_accumulator(leaf);
  if (!node) return;
  const auto made_on = node->stream();
  const c10::impl::VirtualGuardImpl streams(leaf.device().type());
  TORCH_CHECK(!made_on.has_value() || *made_on != streams.getDefaultStream(leaf.device()), what,
              ": an eager graph of the same parameter is alive on the default stream; a backward "
              "cannot be captured beside it (drop the graph first)");
}

// linear_logprob() as a node of the C++ engine (8 tokens of 512, 32000 of the
// vocabulary, forward and backward: 135 us with a Python function, 95 so).
struct LinearLoss : torch::autograd::Function<LinearLoss> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& hidden,
                            const at::Tensor& weight, const at::Tensor& targets,
                            c10::optional<int64_t> ignore_index, bool mean,
                            const std::string& what, int64_t stream) {
    auto [lp, lse, loss, count, bad] =
        linear_logprob(hidden, weight, targets, ignore_index, mean, stream);
    TORCH_CHECK(!bad, what, ": a target is outside [0, vocab_size)");
    // a copy of the targets (8 bytes each): a loader may refill its labels
    // before the backward
    ctx->save_for_backward({hidden, weight, targets.clone(), lse, mean ? count : at::Tensor()});
    ctx->saved_data["has_ignore"] = ignore_index.has_value();
    ctx->saved_data["ignore_index"] = ignore_index.value_or(0);
    ctx->saved_data["stream"] = stream;
    return mean ? loss : lp;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const char* what = "a token loss from hidden states";
    check_no_tangent(grads[0], what);
    const auto saved = ctx->get_saved_variables();
    c10::optional<int64_t> ignore_index;
    if (ctx->saved_data["has_ignore"].toBool()) ignore_index = ctx->saved_data["ignore_index"].toInt();
    c10::optional<at::Tensor> count;
    if (saved[4].defined()) count = saved[4];
    const bool need_hidden = ctx->needs_input_grad(0), need_weight = ctx->needs_input_grad(1);
    // (the engine runs a node on its forward's stream)
    auto [gh, gw] = linear_logprob_backward(
        saved[0].detach(), saved[1].detach(), saved[2], saved[3],
        grads[0].detach().to(at::kFloat).contiguous(), count, ignore_index, need_hidden,
        need_weight, ctx->saved_data["stream"].toInt());
    return {need_hidden ? once_only(gh, grads[0], what) : at::Tensor(),
            need_weight ? once_only(gw, grads[0], what) : at::Tensor(),
            at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

// The logprobs, or their mean loss, of `what`, differentiable in both operands.
at::Tensor linear_loss(const at::Tensor& hidden, const at::Tensor& weight,
                       const at::Tensor& targets, c10::optional<int64_t> ignore_index, bool mean,
                       std::string what, int64_t stream) {
  for (const at::Tensor* t : {&hidden, &weight}) check_no_tangent(*t, what.c_str());
  if (at::GradMode::is_enabled() && (hidden.requires_grad() || weight.requires_grad())) {
    for (const at::Tensor* t : {&hidden, &weight}) check_leaf(*t, what.c_str(), stream);
    return LinearLoss::apply(hidden, weight, targets, ignore_index, mean, what, stream);
  }
  auto [lp, lse, loss, count, bad] =
      linear_logprob(hidden, weight, targets, ignore_index, mean, stream);
  TORCH_CHECK(!bad, what, ": a target is outside [0, vocab_size)");
  return mean ? loss : lp;
}

// ------------------------------------------------- embedding

at::Tensor flat_ids(const at::Tensor& ids, const at::Tensor& like, const char* what) {
  check_same_device(like, ids, "ids");
  TORCH_CHECK(ids.scalar_type() == at::kInt || ids.scalar_type() == at::kLong, "graspo_tokpath.",
              what, ": ids must be int32 or int64");
  return ids.reshape({-1});
}

// (out [*ids.shape, H], whether an id lies outside [0, V): its row is NaN, the
// tokens' order).  check: waits for a look at the ids, which runs ahead of the
// rows (not in a captured call).  ordered: sorts the tokens but padding_idx's
// beside the rows, for the backward; else the order is empty.
std::tuple<at::Tensor, bool, at::Tensor> embedding(const at::Tensor& ids_, const at::Tensor& weight,
                                                   double scale, bool check, bool ordered,
                                                   int64_t padding_idx, int64_t stream) {
  TORCH_CHECK(weight.is_cuda() && weight.dim() == 2 && weight.size(0) > 0 && weight.size(1) > 0,
              "graspo_tokpath.embedding: weight must be a non-empty [V, H] GPU tensor");
  const at::Tensor ids = flat_ids(ids_, weight, "embedding");
  const c10::DeviceGuard guard(weight.device());
  const int64_t N = ids.size(0), V = weight.size(0), H = weight.size(1);
  // (rows that overlap, as an expanded one's do, are copied too)
  const bool in_place = (H == 1 || weight.stride(1) == 1) && (V == 1 || weight.stride(0) >= H);
  const at::Tensor w = in_place ? weight : weight.contiguous();
  void* st = reinterpret_cast<void*>(stream);
  auto shape = ids_.sizes().vec();
  shape.push_back(H);
  // (what may raise comes before the look's launch: see verdict_wait)
  const int dt = dtype_code(w);
  at::Tensor out = at::empty(shape, weight.options());
  const size_t order_bytes = ordered ? gtp_embedding_order_bytes(N, V) : 0;
  at::Tensor order = at::empty({(int64_t)order_bytes / 4}, weight.options().dtype(at::kInt));
  const int ids64 = ids.scalar_type() == at::kLong;
  const int64_t ids_stride = N > 1 ? ids.stride(0) : 1;
  at::Tensor words;
  if (check && N > 0 && !gtp_stream_capturing(st)) {
    words = verdict_words();
    const int rc = gtp_targets_verdict(ids.data_ptr(), ids64, N, ids_stride, V, nullptr, nullptr,
                                       verdict_ptr(words), st);
    int found = 0;
    if (rc == GTP_ERR_LAUNCH) verdict_wait(words, &found, st);
    check_rc(rc, "gtp_targets_verdict");
  }
  const int64_t ld = V > 1 ? w.stride(0) : H;
  const int rc =
      ordered ? gtp_embedding_rows_ordered(ids.data_ptr(), ids64, N, ids_stride, w.data_ptr(),
                                           dt, V, H, ld, (float)scale, out.data_ptr(),
                                           padding_idx, order.data_ptr(), order_bytes, st)
              : gtp_embedding_rows(ids.data_ptr(), ids64, N, ids_stride, w.data_ptr(),
                                   dt, V, H, ld, (float)scale, out.data_ptr(), st);
  int bad = 0, wait_rc = GTP_OK;
  if (words.defined()) wait_rc = verdict_wait(words, &bad, st);
  check_rc(rc, "gtp_embedding_rows");
  check_rc(wait_rc, "gtp_verdict_wait");
  return {out, (bad & 1) != 0, order};
}

// A tensor written through its pointer counts as written: a graph that saved
// it raises then.  (One made in inference mode has no counter.)
void count_write(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// The gradient of the table from that of embedding()'s rows; out: added to.
// order: embedding()'s, in the ids' place.
at::Tensor embedding_backward(const c10::optional<at::Tensor>& ids_, const at::Tensor& grad_,
                              int64_t V, double scale, int64_t padding_idx,
                              const c10::optional<at::Tensor>& out,
                              const c10::optional<at::Tensor>& order, int64_t stream) {
  TORCH_CHECK(grad_.is_cuda() && grad_.dim() >= 1 && grad_.size(-1) > 0 && V > 0,
              "graspo_tokpath.embedding_backward: grad must be a [..., H] GPU tensor and V > 0");
  const int64_t H = grad_.size(-1);
  const int64_t N = grad_.numel() / H;
  at::Tensor ids;
  if (order.has_value()) {
    check_same_device(grad_, *order, "order");
    TORCH_CHECK(order->scalar_type() == at::kInt && order->is_contiguous() &&
                    (size_t)order->numel() * 4 == gtp_embedding_order_bytes(N, V),
                "graspo_tokpath.embedding_backward: the order is not one of ", N, " tokens of ", V,
                " rows");
  } else {
    TORCH_CHECK(ids_.has_value(), "graspo_tokpath.embedding_backward: neither ids nor an order");
    ids = flat_ids(*ids_, grad_, "embedding_backward");
    TORCH_CHECK(ids.size(0) == N,
                "graspo_tokpath.embedding_backward: grad must be [*ids.shape, H]");
  }
  const c10::DeviceGuard guard(grad_.device());
  at::Tensor grad = grad_.reshape({N, H});
  if (H > 1 && grad.stride(1) != 1) grad = grad.contiguous();
  at::Tensor to;
  if (out.has_value()) {
    to = *out;
    check_same_device(grad, to, "out");
    TORCH_CHECK(to.scalar_type() == grad.scalar_type() && to.dim() == 2 && to.size(0) == V &&
                    to.size(1) == H && to.is_contiguous(),
                "graspo_tokpath.embedding_backward: out must be a contiguous [V, H] of the "
                "gradient's dtype");
  } else {
    to = at::empty({V, H}, grad.options());
  }
  const int dt = dtype_code(grad);
  const size_t ws_bytes = order.has_value()
                              ? gtp_embedding_backward_ordered_workspace_bytes(dt, N, H)
                              : gtp_embedding_backward_workspace_bytes(dt, N, V, H);
  at::Tensor ws = at::empty({(int64_t)std::max<size_t>(ws_bytes, 256)},
                            grad.options().dtype(at::kByte));
  const int64_t ld = N > 1 ? grad.stride(0) : H;
  void* st = reinterpret_cast<void*>(stream);
  const int rc =
      order.has_value()
          ? gtp_embedding_backward_ordered(order->data_ptr(), (size_t)order->numel() * 4, N,
                                           grad.data_ptr(), dt, ld, V, H, (float)scale,
                                           out.has_value(), to.data_ptr(), ws.data_ptr(),
                                           (size_t)ws.numel(), st)
          : gtp_embedding_backward(ids.data_ptr(), ids.scalar_type() == at::kLong, N,
                                   N > 1 ? ids.stride(0) : 1, grad.data_ptr(), dt, ld, V, H,
                                   (float)scale, padding_idx, out.has_value(), to.data_ptr(),
                                   ws.data_ptr(), (size_t)ws.numel(), st);
  check_rc(rc, "gtp_embedding_backward");
  if (out.has_value()) count_write(to);
  return to;
}

// embedding() with its gradient.  A C++ node: for few tokens Python's part of
// a forward and a backward is most of what they take (999 tokens of a 206 MB
// table: 102 us with a Python function, 66 so).
struct TokenEmbedding : torch::autograd::Function<TokenEmbedding> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& ids,
                            const at::Tensor& weight, double scale, int64_t padding_idx, bool check,
                            int64_t stream) {
    auto [out, bad, order] = embedding(ids, weight, scale, check, true, padding_idx, stream);
    TORCH_CHECK(!bad, "token_embedding: an id is outside [0, vocab_size)");
    // the tokens' order is kept, not the ids: a loader may refill its batch
    // before the backward
    ctx->save_for_backward({order});
    ctx->saved_data["vocab"] = weight.size(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["stream"] = stream;
    return out;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const at::Tensor& grad = grads[0];
    check_no_tangent(grad, "token_embedding");
    // (the engine runs a node on its forward's stream)
    at::Tensor out = embedding_backward(
        c10::nullopt, grad.detach(), ctx->saved_data["vocab"].toInt(),
        ctx->saved_data["scale"].toDouble(), -1, c10::nullopt, ctx->get_saved_variables()[0],
        ctx->saved_data["stream"].toInt());
    out = once_only(out, grad, "token_embedding");
    return {at::Tensor(), out, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

at::Tensor token_embedding(const at::Tensor& ids, const at::Tensor& weight, double scale,
                           int64_t padding_idx, bool check, int64_t stream) {
  check_no_tangent(weight, "token_embedding");
  if (at::GradMode::is_enabled() && weight.requires_grad()) {
    check_leaf(weight, "token_embedding", stream);
    return TokenEmbedding::apply(ids, weight, scale, padding_idx, check, stream);
  }
  auto [out, bad, order] = embedding(ids, weight, scale, check, false, padding_idx, stream);
  TORCH_CHECK(!bad, "token_embedding: an id is outside [0, vocab_size)");
  return out;
}

// ------------------------------------------------- gradient norm and clipping

// Tensors as address, size and type; one whose elements do not fill its
// memory without gaps goes through a contiguous copy.
struct GradList {
  std::vector<void*> p;
  std::vector<int64_t> n;
  std::vector<int32_t> dtype;
  std::vector<std::pair<at::Tensor, at::Tensor>> copies;  // (tensor, its copy)
  explicit GradList(at::TensorList tensors, const char* what) {
    TORCH_CHECK(!tensors.empty(), "graspo_tokpath.", what, ": no tensor");
    p.reserve(tensors.size());
    n.reserve(tensors.size());
    dtype.reserve(tensors.size());
    for (const at::Tensor& t : tensors) {
      TORCH_CHECK_VALUE(!t.is_sparse(), "graspo_tokpath.", what,
                        ": sparse gradients are not supported");
      TORCH_CHECK(t.is_cuda(), "graspo_tokpath.", what, ": tensors must be on a GPU");
      check_same_device(tensors[0], t, "every tensor");
      const at::ScalarType s = t.scalar_type();
      TORCH_CHECK(s == at::kFloat || s == at::kBFloat16 || s == at::kHalf, "graspo_tokpath.", what,
                  ": tensors must be float32, bfloat16 or float16, got ", s);
      const bool whole = t.is_contiguous() || t.is_non_overlapping_and_dense();
      if (!whole) copies.emplace_back(t, t.contiguous());
      p.push_back((whole ? t : copies.back().second).data_ptr());
      n.push_back(t.numel());
      dtype.push_back(s == at::kFloat ? GTP_DTYPE_F32
                                      : s == at::kBFloat16 ? GTP_DTYPE_BF16 : GTP_DTYPE_F16);
    }
  }
  int64_t size() const { return (int64_t)p.size(); }
};

// Whether a and b, whose spans in memory overlap, are known to share no byte:
// columns of one buffer, say.  At some stride P of theirs, the dims that step
// by multiples of P aside, each fills less than P bytes, and modulo P these do
// not meet.
bool apart(const at::Tensor& a, const at::Tensor& b) {
  const int64_t sa = a.element_size(), sb = b.element_size();
  auto extent = [](const at::Tensor& t, int64_t es, int64_t P) {
    int64_t bytes = es;
    for (int64_t d = 0; d < t.dim(); ++d)
      if (t.stride(d) * es % P != 0) bytes += (t.size(d) - 1) * t.stride(d) * es;
    return bytes;
  };
  auto apart_at = [&](int64_t P) {
    const int64_t ea = extent(a, sa, P), eb = extent(b, sb, P);
    int64_t off = (reinterpret_cast<intptr_t>(b.data_ptr()) - reinterpret_cast<intptr_t>(a.data_ptr())) % P;
    if (off < 0) off += P;
    return ea <= off && off + eb <= P;
  };
  for (int64_t d = 0; d < a.dim(); ++d)
    if (a.size(d) > 1 && apart_at(a.stride(d) * sa)) return true;
  for (int64_t d = 0; d < b.dim(); ++d)
    if (b.size(d) > 1 && apart_at(b.stride(d) * sb)) return true;
  return false;
}

// In-place products of overlapping tensors would race (and scale twice).
void check_apart(at::TensorList tensors, const char* what = "clip_grads_") {
  struct Span {
    uintptr_t from, to;
    const at::Tensor* t;
    bool operator<(const Span& o) const { return from < o.from; }
  };
  std::vector<Span> at;
  at.reserve(tensors.size());
  bool sorted = true;
  for (const at::Tensor& t : tensors) {
    if (t.numel() == 0) continue;
    int64_t span = t.numel();
    if (!t.is_contiguous()) {
      span = 1;
      for (int64_t d = 0; d < t.dim(); ++d) {
        TORCH_CHECK(t.size(d) <= 1 || t.stride(d) != 0,
                    "graspo_tokpath.", what, ": a tensor overlaps itself");
        span += (t.size(d) - 1) * t.stride(d);
      }
    }
    const uintptr_t a = reinterpret_cast<uintptr_t>(t.data_ptr());
    sorted = sorted && (at.empty() || at.back().from <= a);
    at.push_back({a, a + span * t.element_size(), &t});
  }
  if (!sorted) std::sort(at.begin(), at.end());
  uintptr_t reach = 0;
  for (size_t i = 0; i < at.size(); ++i) {
    for (size_t j = 0; at[i].from < reach && j < i; ++j)
      TORCH_CHECK(at[j].to <= at[i].from || apart(*at[j].t, *at[i].t),
                  "graspo_tokpath.", what, ": tensors overlap in memory (the same one twice?)");
    reach = std::max(reach, at[i].to);
  }
}

at::Tensor norm_of(const GradList& l, const at::Tensor& like, double norm_type, void* st) {
  const int kind = norm_type == 1.0 ? 1 : norm_type == 2.0 ? 2 : 3;
  TORCH_CHECK(kind < 3 || norm_type == std::numeric_limits<double>::infinity(),
              "graspo_tokpath.grad_norm: norm_type must be 1, 2 or inf, got ", norm_type);
  at::Tensor out = at::empty({}, like.options().dtype(at::kFloat));
  const size_t ws_bytes = gtp_grad_norm_workspace_bytes(l.p.data(), l.n.data(), l.dtype.data(), l.size());
  at::Tensor ws = at::empty({(int64_t)std::max<size_t>(ws_bytes, 256)},
                            like.options().dtype(at::kByte));
  check_rc(gtp_grad_norm(l.p.data(), l.n.data(), l.dtype.data(), l.size(), kind,
                         out.data_ptr<float>(), ws.data_ptr(), (size_t)ws.numel(), st),
           "gtp_grad_norm");
  return out;
}

void clip_by(at::TensorList tensors, GradList& l, const at::Tensor& norm, double max_norm, void* st) {
  check_rc(gtp_clip_grads(l.p.data(), l.n.data(), l.dtype.data(), l.size(), norm.data_ptr<float>(),
                          (float)max_norm, st),
           "gtp_clip_grads");
  for (const at::Tensor& t : tensors) count_write(t);
  const at::NoGradGuard untracked;  // (gradients may be of a graph)
  for (auto& c : l.copies) c.first.copy_(c.second);
}

at::Tensor grad_norm(at::TensorList tensors, double norm_type, int64_t stream) {
  const GradList l(tensors, "grad_norm");
  const c10::DeviceGuard guard(tensors[0].device());
  return norm_of(l, tensors[0], norm_type, reinterpret_cast<void*>(stream));
}

void clip_grads_(at::TensorList tensors, const at::Tensor& norm, double max_norm, int64_t stream) {
  GradList l(tensors, "clip_grads_");
  check_apart(tensors);
  check_same_device(tensors[0], norm, "norm");
  TORCH_CHECK(norm.scalar_type() == at::kFloat && norm.numel() == 1,
              "graspo_tokpath.clip_grads_: norm must be one float32");
  const c10::DeviceGuard guard(tensors[0].device());
  clip_by(tensors, l, norm, max_norm, reinterpret_cast<void*>(stream));
}

// Both, from one look at the list.
at::Tensor clip_grad_norm_(at::TensorList tensors, double max_norm, double norm_type,
                           int64_t stream) {
  GradList l(tensors, "clip_grad_norm_");
  check_apart(tensors);
  const c10::DeviceGuard guard(tensors[0].device());
  void* st = reinterpret_cast<void*>(stream);
  const at::Tensor norm = norm_of(l, tensors[0], norm_type, st);
  clip_by(tensors, l, norm, max_norm, st);
  return norm;
}

// ------------------------------------------------- beam search

// Contiguous outputs, each with a storage of its own, as sample's: the first by
// at::empty, the others from its allocator directly.  (A beam step of one request
// takes 15.8 us, and 13.9 with parts of one allocation, of which none could be
// saved, resized or dropped by itself.)  The current device is the first's.
struct Outputs {
  const at::TensorOptions options;
  c10::Allocator* alloc = nullptr;
  c10::DispatchKeySet keys;
  explicit Outputs(const at::Tensor& like) : options(like.options()) {}
  at::Tensor take(at::IntArrayRef sizes, at::ScalarType dt) {
    if (alloc) return at::Tensor(at::detail::empty_generic(sizes, alloc, keys, dt, c10::nullopt));
    const at::Tensor t = at::empty(sizes, options.dtype(dt));
    alloc = t.storage().allocator();
    keys = t.key_set();
    return t;
  }
};

// logits [G * K, V] or [G, K, V], any strides but of the columns; scores [G, K]
gtp_beam_rows beam_rows(const at::Tensor& logits, const at::Tensor& scores, int64_t candidates,
                        const c10::optional<at::Tensor>& allow_mask,
                        const c10::optional<at::Tensor>& done, const char* what) {
  TORCH_CHECK(logits.is_cuda(), "graspo_tokpath.", what, ": logits must be a GPU tensor");
  check_same_device(logits, scores, "scores");
  TORCH_CHECK(scores.scalar_type() == at::kFloat && scores.dim() == 2 && scores.is_contiguous() &&
                  scores.size(1) > 0,
              "graspo_tokpath.", what, ": scores must be contiguous float32 [groups, beams]");
  const int64_t G = scores.size(0), K = scores.size(1), V = logits.size(-1);
  TORCH_CHECK((logits.dim() == 2 && logits.size(0) == G * K) ||
                  (logits.dim() == 3 && logits.size(0) == G && logits.size(1) == K),
              "graspo_tokpath.", what, ": logits must be [groups * beams, V] or [groups, beams, V]");
  TORCH_CHECK(V > 0 && (V == 1 || logits.stride(-1) == 1), "graspo_tokpath.", what,
              ": logits rows must be contiguous and not empty");
  TORCH_CHECK(K <= 32 && candidates >= 1 && candidates <= 64, "graspo_tokpath.", what,
              ": at most 32 beams and 64 candidates, got ", K, " and ", candidates);
  gtp_beam_rows r{};
  r.logits = logits.data_ptr();
  r.scores = scores.data_ptr<float>();
  r.groups = G;
  r.vocab = V;
  const bool two = logits.dim() == 2;
  r.beam_stride = two ? logits.stride(0) : logits.stride(1);
  r.group_stride = two ? K * logits.stride(0) : logits.stride(0);
  r.dtype = dtype_code(logits);
  r.beams = (int32_t)K;
  r.candidates = (int32_t)candidates;
  if (allow_mask.has_value()) {
    const auto& m = *allow_mask;
    check_same_device(logits, m, "allow_mask");
    TORCH_CHECK((m.scalar_type() == at::kInt || m.scalar_type() == at::kUInt32) && m.dim() == 2 &&
                    m.size(0) == G * K && m.size(1) >= (V + 31) / 32 &&
                    (m.size(1) == 1 || m.stride(1) == 1),
                "graspo_tokpath.", what,
                ": allow_mask must be int32/uint32 [groups * beams, >= ceil(V/32)]");
    // (rows that share a mask are copied)
    TORCH_CHECK(m.size(0) <= 1 || m.stride(0) >= (V + 31) / 32, "graspo_tokpath.", what,
                ": allow_mask rows overlap");
    r.allow_mask = static_cast<const uint32_t*>(m.data_ptr());
    r.mask_stride = G * K > 1 ? m.stride(0) : m.size(1);
  }
  if (done.has_value()) {
    check_same_device(logits, *done, "done");
    TORCH_CHECK(done->scalar_type() == at::kBool && done->dim() == 1 && done->size(0) == G &&
                    done->is_contiguous(),
                "graspo_tokpath.", what, ": done must be contiguous bool [groups]");
    r.done = static_cast<const uint8_t*>(done->data_ptr());
  }
  return r;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> beam_candidates(
    const at::Tensor& logits, const at::Tensor& scores, int64_t candidates,
    const c10::optional<at::Tensor>& allow_mask, const c10::optional<at::Tensor>& done,
    int64_t stream) {
  const gtp_beam_rows r = beam_rows(logits, scores, candidates, allow_mask, done, "beam_candidates");
  const c10::DeviceGuard guard(logits.device());
  const auto i32 = scores.options().dtype(at::kInt);
  at::Tensor out = at::empty({r.groups, candidates}, scores.options());
  at::Tensor beams = at::empty({r.groups, candidates}, i32);
  at::Tensor tokens = at::empty({r.groups, candidates}, i32.dtype(at::kLong));
  at::Tensor status = at::empty({r.groups * r.beams}, i32);
  at::Tensor ws = at::empty({(int64_t)gtp_beam_workspace_bytes(&r)}, i32.dtype(at::kByte));
  check_rc(gtp_beam_candidates(&r, out.data_ptr<float>(), beams.data_ptr<int32_t>(),
                               tokens.data_ptr<int64_t>(), status.data_ptr<int32_t>(),
                               ws.data_ptr(), (size_t)ws.numel(), reinterpret_cast<void*>(stream)),
           "gtp_beam_candidates");
  return {out, beams, tokens, status};
}

using BeamOut = std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor,
                           at::Tensor>;

// A step's state, with new tensors for what it becomes.
struct BeamStep {
  gtp_beam_state s{};
  BeamOut out;
  at::Tensor status;
  BeamStep(const at::Tensor& scores, const at::Tensor& pool_scores, const at::Tensor& pool_rows,
           const at::Tensor& pool_steps, const at::Tensor& done, int64_t eos, int64_t pad,
           double length, int64_t step, bool early, const c10::optional<at::Tensor>& tokens_out,
           const c10::optional<at::Tensor>& parents_out, const char* what) {
    const int64_t G = scores.size(0), K = scores.size(1);
    auto check = [&](const at::Tensor& t, at::ScalarType dt, const char* name) {
      check_same_device(scores, t, name);
      TORCH_CHECK(t.scalar_type() == dt && t.dim() == 2 && t.size(0) == G && t.size(1) == K &&
                      t.is_contiguous(),
                  "graspo_tokpath.", what, ": ", name, " must be contiguous ", dt,
                  " [groups, beams]");
    };
    check(pool_scores, at::kFloat, "pool_scores");
    check(pool_rows, at::kInt, "pool_rows");
    check(pool_steps, at::kInt, "pool_steps");
    check_same_device(scores, done, "done");
    TORCH_CHECK(done.scalar_type() == at::kBool && done.dim() == 1 && done.size(0) == G &&
                    done.is_contiguous(),
                "graspo_tokpath.", what, ": done must be contiguous bool [groups]");
    TORCH_CHECK(step >= 0 && step < INT32_MAX, "graspo_tokpath.", what, ": step must be >= 0");
    TORCH_CHECK(length > 0.0 && length <= std::numeric_limits<double>::max(), "graspo_tokpath.",
                what, ": (step + 1)^length_penalty must be positive and finite");
    const int64_t n = G * K;
    Outputs own(scores);
    auto to = [&](const c10::optional<at::Tensor>& t, at::ScalarType dt, const char* name) {
      if (!t.has_value()) return own.take({n}, dt);
      check_same_device(scores, *t, name);
      TORCH_CHECK(t->scalar_type() == dt && t->dim() == 1 && t->size(0) == G * K &&
                      t->is_contiguous(),
                  "graspo_tokpath.", what, ": ", name, " must be contiguous ", dt,
                  " [groups * beams]");
      return *t;
    };
    at::Tensor tokens = to(tokens_out, at::kLong, "tokens_out");
    at::Tensor parents = to(parents_out, at::kInt, "parents_out");
    at::Tensor n_scores = own.take({G, K}, at::kFloat);
    at::Tensor n_pool = own.take({G, K}, at::kFloat);
    at::Tensor n_rows = own.take({G, K}, at::kInt);
    at::Tensor n_steps = own.take({G, K}, at::kInt);
    at::Tensor n_done = own.take({G}, at::kBool);
    status = own.take({n}, at::kInt);
    s.scores = scores.data_ptr<float>();
    s.pool_scores = pool_scores.data_ptr<float>();
    s.pool_rows = pool_rows.data_ptr<int32_t>();
    s.pool_steps = pool_steps.data_ptr<int32_t>();
    s.done = static_cast<const uint8_t*>(done.data_ptr());
    s.out_tokens = tokens.data_ptr<int64_t>();
    s.out_parents = parents.data_ptr<int32_t>();
    s.out_scores = n_scores.data_ptr<float>();
    s.out_pool_scores = n_pool.data_ptr<float>();
    s.out_pool_rows = n_rows.data_ptr<int32_t>();
    s.out_pool_steps = n_steps.data_ptr<int32_t>();
    s.out_done = static_cast<uint8_t*>(n_done.data_ptr());
    s.eos_token_id = eos;
    s.pad_token_id = pad;
    s.length = length;
    s.step = (int32_t)step;
    s.early_stopping = early;
    out = {tokens, parents, n_scores, n_pool, n_rows, n_steps, n_done};
  }
  // tensors of the caller's that were written
  void written(const c10::optional<at::Tensor>& tokens_out,
               const c10::optional<at::Tensor>& parents_out) const {
    for (const auto* t : {&tokens_out, &parents_out})
      if (t->has_value() && !(*t)->is_inference()) (*t)->unsafeGetTensorImpl()->bump_version();
  }
};

BeamOut beam_advance(const at::Tensor& c_scores, const at::Tensor& c_beams,
                     const at::Tensor& c_tokens, const at::Tensor& scores,
                     const at::Tensor& pool_scores, const at::Tensor& pool_rows,
                     const at::Tensor& pool_steps, const at::Tensor& done, int64_t eos, int64_t pad,
                     double length, int64_t step, bool early,
                     const c10::optional<at::Tensor>& tokens_out,
                     const c10::optional<at::Tensor>& parents_out, int64_t stream) {
  TORCH_CHECK(scores.is_cuda() && scores.scalar_type() == at::kFloat && scores.dim() == 2 &&
                  scores.is_contiguous() && scores.size(1) > 0 && scores.size(1) <= 32,
              "graspo_tokpath.beam_advance: scores must be a contiguous float32 GPU tensor "
              "[groups, beams], at most 32 beams");
  const int64_t G = scores.size(0), n = c_scores.dim() == 2 ? c_scores.size(1) : 0;
  TORCH_CHECK(n >= 1 && n <= 64, "graspo_tokpath.beam_advance: 1 to 64 candidates, got ", n);
  auto check = [&](const at::Tensor& t, at::ScalarType dt, const char* name) {
    check_same_device(scores, t, name);
    TORCH_CHECK(t.scalar_type() == dt && t.dim() == 2 && t.size(0) == G && t.size(1) == n &&
                    t.is_contiguous(),
                "graspo_tokpath.beam_advance: ", name, " must be contiguous ", dt,
                " [groups, candidates]");
  };
  check(c_scores, at::kFloat, "candidates' scores");
  check(c_beams, at::kInt, "candidates' beams");
  check(c_tokens, at::kLong, "candidates' tokens");
  const c10::DeviceGuard guard(scores.device());
  BeamStep b(scores, pool_scores, pool_rows, pool_steps, done, eos, pad, length, step, early,
             tokens_out, parents_out, "beam_advance");
  check_rc(gtp_beam_advance(c_scores.data_ptr<float>(), c_beams.data_ptr<int32_t>(),
                            c_tokens.data_ptr<int64_t>(), G, (int32_t)scores.size(1), (int32_t)n,
                            &b.s, reinterpret_cast<void*>(stream)),
           "gtp_beam_advance");
  b.written(tokens_out, parents_out);
  return b.out;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor,
           at::Tensor>
beam_step(const at::Tensor& logits, const at::Tensor& scores, const at::Tensor& pool_scores,
          const at::Tensor& pool_rows, const at::Tensor& pool_steps, const at::Tensor& done,
          int64_t candidates, int64_t eos, int64_t pad, double length, int64_t step, bool early,
          const c10::optional<at::Tensor>& allow_mask, const c10::optional<at::Tensor>& tokens_out,
          const c10::optional<at::Tensor>& parents_out, int64_t stream) {
  const gtp_beam_rows r = beam_rows(logits, scores, candidates, allow_mask, done, "beam_step");
  const c10::DeviceGuard guard(logits.device());
  BeamStep b(scores, pool_scores, pool_rows, pool_steps, done, eos, pad, length, step, early,
             tokens_out, parents_out, "beam_step");
  at::Tensor ws = at::empty({(int64_t)gtp_beam_workspace_bytes(&r)}, scores.options().dtype(at::kByte));
  check_rc(gtp_beam_step(&r, &b.s, b.status.data_ptr<int32_t>(), ws.data_ptr(), (size_t)ws.numel(),
                         reinterpret_cast<void*>(stream)),
           "gtp_beam_step");
  b.written(tokens_out, parents_out);
  return std::tuple_cat(b.out, std::make_tuple(b.status));
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> beam_finish(
    const at::Tensor& scores, const at::Tensor& pool_scores, const at::Tensor& pool_rows,
    const at::Tensor& pool_steps, const at::Tensor& done, const at::Tensor& tokens,
    const at::Tensor& parents, double length, int64_t eos, int64_t pad, int64_t give,
    int64_t stream) {
  TORCH_CHECK(scores.is_cuda() && scores.dim() == 2 && scores.size(1) > 0 && scores.size(1) <= 32,
              "graspo_tokpath.beam_finish: scores must be a GPU tensor [groups, beams], at most 32 "
              "beams");
  const int64_t G = scores.size(0), K = scores.size(1);
  auto check = [&](const at::Tensor& t, at::ScalarType dt, at::IntArrayRef shape, const char* name) {
    check_same_device(scores, t, name);
    TORCH_CHECK(t.scalar_type() == dt && t.sizes() == shape && t.is_contiguous(),
                "graspo_tokpath.beam_finish: ", name, " must be contiguous ", dt, " ", shape);
  };
  const int64_t T = tokens.dim() == 2 ? tokens.size(0) : -1;
  check(scores, at::kFloat, {G, K}, "scores");
  check(pool_scores, at::kFloat, {G, K}, "pool_scores");
  check(pool_rows, at::kInt, {G, K}, "pool_rows");
  check(pool_steps, at::kInt, {G, K}, "pool_steps");
  check(done, at::kBool, {G}, "done");
  check(tokens, at::kLong, {T, G * K}, "tokens");
  check(parents, at::kInt, {T, G * K}, "parents");
  TORCH_CHECK(give >= 1 && give <= K && T < INT32_MAX,
              "graspo_tokpath.beam_finish: 1 to ", K, " hypotheses of a group, got ", give);
  TORCH_CHECK(length > 0.0, "graspo_tokpath.beam_finish: the length must be positive");
  const c10::DeviceGuard guard(scores.device());
  at::Tensor out = at::empty({G, give}, scores.options());
  at::Tensor lengths = at::empty({G, give}, pool_rows.options());
  at::Tensor seq = at::empty({G, give, T}, tokens.options());
  check_rc(gtp_beam_finish(scores.data_ptr<float>(), pool_scores.data_ptr<float>(),
                           pool_rows.data_ptr<int32_t>(), pool_steps.data_ptr<int32_t>(),
                           static_cast<const uint8_t*>(done.data_ptr()), tokens.data_ptr<int64_t>(),
                           parents.data_ptr<int32_t>(), G, (int32_t)K, (int32_t)T, length, eos, pad,
                           (int32_t)give, out.data_ptr<float>(), lengths.data_ptr<int32_t>(),
                           seq.data_ptr<int64_t>(), T, reinterpret_cast<void*>(stream)),
           "gtp_beam_finish");
  return {out, lengths, seq};
}

// ------------------------------------------------- states of the beams

// A state's rows as runs of bytes.  in_memory_order: dimensions by stride, as
// suits a copy onto itself; else in the tensor's own order.
gtp_state_shape state_shape(const at::Tensor& t, bool in_memory_order, const char* what) {
  const int64_t es = t.element_size();
  std::vector<std::pair<int64_t, int64_t>> dims;  // (stride, size), innermost first
  for (int64_t d = t.dim() - 1; d >= 1; --d)
    if (t.size(d) != 1) dims.emplace_back(t.stride(d) * es, t.size(d));
  if (in_memory_order) {
    std::stable_sort(dims.begin(), dims.end(),
                     [](const auto& a, const auto& b) { return a.first < b.first; });
    // (each dimension steps over all that lies within it, the rows' own too)
    std::vector<std::pair<int64_t, int64_t>> all = dims;
    if (t.size(0) > 1) all.emplace_back(t.stride(0) * es, t.size(0));
    std::sort(all.begin(), all.end());
    int64_t span = es;
    for (const auto& d : all) {
      TORCH_CHECK(d.first >= span || t.numel() == 0, "graspo_tokpath.", what,
                  ": a state overlaps itself");
      span += (d.second - 1) * d.first;
    }
  }
  gtp_state_shape s;
  s.run_bytes = t.numel() == 0 ? 0 : es;
  s.row_stride = t.size(0) > 1 ? t.stride(0) * es : 0;
  for (int d = 0; d < GTP_STATE_DIMS; ++d) {
    s.sizes[d] = 1;
    s.strides[d] = 0;
  }
  int at = -1;  // the last dimension of runs
  for (const auto& d : dims) {
    if (at < 0 && d.first == s.run_bytes) {
      s.run_bytes *= d.second;
    } else if (at >= 0 && d.first == s.strides[at] * s.sizes[at]) {
      s.sizes[at] *= d.second;
    } else {
      ++at;
      TORCH_CHECK(at < GTP_STATE_DIMS, "graspo_tokpath.", what,
                  ": a state of more strided dimensions than are supported");
      s.sizes[at] = d.second;
      s.strides[at] = d.first;
    }
  }
  return s;
}

// of every state; neighbours alike are looked at once
std::vector<gtp_state_shape> state_shapes(at::TensorList states, bool in_memory_order,
                                          const char* what) {
  std::vector<gtp_state_shape> shapes;
  shapes.reserve(states.size());
  for (size_t i = 0; i < states.size(); ++i) {
    const at::Tensor& t = states[i];
    if (i > 0 && t.sizes() == states[i - 1].sizes() && t.strides() == states[i - 1].strides() &&
        t.element_size() == states[i - 1].element_size())
      shapes.push_back(shapes.back());
    else
      shapes.push_back(state_shape(t, in_memory_order, what));
  }
  return shapes;
}

bool same_shape(const gtp_state_shape& a, const gtp_state_shape& b) {
  bool same = a.run_bytes == b.run_bytes && a.row_stride == b.row_stride;
  for (int d = 0; d < GTP_STATE_DIMS; ++d)
    same = same && a.sizes[d] == b.sizes[d] && a.strides[d] == b.strides[d];
  return same;
}

void check_states(at::TensorList states, int64_t rows, const char* what) {
  for (const at::Tensor& t : states) {
    TORCH_CHECK(t.is_cuda() && t.layout() == at::kStrided && !t.is_conj() && !t.is_neg(),
                "graspo_tokpath.", what, ": states must be dense GPU tensors");
    check_same_device(states[0], t, "every state");
    TORCH_CHECK(t.dim() >= 1 && (rows < 0 || t.size(0) == rows), "graspo_tokpath.", what,
                ": a state's first dimension must count the rows (", rows, "), got ", t.sizes());
  }
}

void reorder_states_(at::TensorList states, const at::Tensor& parents, int64_t beams, bool check,
                     int64_t stream) {
  if (states.empty()) return;
  TORCH_CHECK(beams >= 1 && beams <= 64, "graspo_tokpath.reorder_states_: 1 to 64 beams, got ",
              beams);
  TORCH_CHECK(parents.scalar_type() == at::kInt && parents.dim() == 1 && parents.is_contiguous() &&
                  parents.size(0) % beams == 0,
              "graspo_tokpath.reorder_states_: parents must be contiguous int32 [groups * beams]");
  const int64_t R = parents.size(0);
  check_states(states, R, "reorder_states_");
  check_same_device(states[0], parents, "parents");
  for (const at::Tensor& t : states)
    TORCH_CHECK(!t.requires_grad() || !at::GradMode::is_enabled(),
                "graspo_tokpath.reorder_states_: a state that requires a gradient");
  const c10::DeviceGuard guard(states[0].device());
  const std::vector<gtp_state_shape> shapes = state_shapes(states, true, "reorder_states_");
  // (one behind the other, as a cache's layers mostly are, they are apart)
  uintptr_t reach = 0;
  for (const at::Tensor& t : states) {
    const uintptr_t from = reinterpret_cast<uintptr_t>(t.data_ptr());
    if (from < reach) {
      check_apart(states, "reorder_states_");
      break;
    }
    int64_t last = 0;
    for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
    if (t.numel() > 0) reach = from + (last + 1) * t.element_size();
  }
  void* st = reinterpret_cast<void*>(stream);
  at::Tensor bad;
  check = check && R > 0 && !gtp_stream_capturing(st);
  if (check) bad = at::zeros({1}, parents.options());
  std::vector<void*> p;
  p.reserve(states.size());
  for (const at::Tensor& t : states) p.push_back(t.data_ptr());
  // neighbours of one shape in a call; of several shapes all are looked at before
  // any is moved
  const auto alike = [&](auto call) {
    for (size_t i = 0, j = 0; i < p.size(); i = j) {
      while (j < p.size() && same_shape(shapes[i], shapes[j])) ++j;
      check_rc(call(&p[i], (int64_t)(j - i), &shapes[i]), "gtp_reorder_states");
    }
  };
  const int64_t groups = R / beams;
  alike([&](void** q, int64_t n, const gtp_state_shape* s) {
    return n == (int64_t)p.size() ? GTP_OK
                                  : gtp_reorder_states_check(q, n, s, groups, (int32_t)beams);
  });
  alike([&](void** q, int64_t n, const gtp_state_shape* s) {
    return gtp_reorder_states(q, n, s, parents.data_ptr<int32_t>(), groups, (int32_t)beams,
                              check ? bad.data_ptr<int32_t>() : nullptr, st);
  });
  for (const at::Tensor& t : states)
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  TORCH_CHECK(!check || bad.item<int32_t>() == 0,
              "graspo_tokpath.reorder_states_: a parent lies outside its row's group (such rows "
              "stay as they were)");
}

std::vector<at::Tensor> expand_states(at::TensorList states, int64_t beams, int64_t stream) {
  TORCH_CHECK(beams >= 1 && beams <= 64, "graspo_tokpath.expand_states: 1 to 64 beams, got ", beams);
  std::vector<at::Tensor> outs;
  if (states.empty()) return outs;
  check_states(states, states[0].dim() >= 1 ? states[0].size(0) : -1, "expand_states");
  for (const at::Tensor& t : states)
    TORCH_CHECK(!t.requires_grad() || !at::GradMode::is_enabled(),
                "graspo_tokpath.expand_states: a state that requires a gradient");
  const c10::DeviceGuard guard(states[0].device());
  const std::vector<gtp_state_shape> shapes = state_shapes(states, false, "expand_states");
  outs.reserve(states.size());
  Outputs own(states[0]);
  std::vector<int64_t> size;
  for (const at::Tensor& t : states) {
    size.assign(t.sizes().begin(), t.sizes().end());
    size[0] *= beams;
    outs.push_back(own.take(size, t.scalar_type()));
  }
  std::vector<const void*> from;
  std::vector<void*> to;
  for (size_t i = 0; i < states.size();) {
    from.clear();
    to.clear();
    size_t j = i;
    for (; j < states.size() && same_shape(shapes[i], shapes[j]); ++j) {
      from.push_back(states[j].data_ptr());
      to.push_back(outs[j].data_ptr());
    }
    check_rc(gtp_expand_states(from.data(), to.data(), (int64_t)from.size(), &shapes[i],
                               states[i].size(0), (int32_t)beams, reinterpret_cast<void*>(stream)),
             "gtp_expand_states");
    i = j;
  }
  return outs;
}

// ------------------------------------------------- low-rank adapters

// [..., n] as rows with unit column stride: their distance, or a copy
at::Tensor as_rows(const at::Tensor& t, int64_t n, int64_t& stride) {
  if (t.is_contiguous()) {
    stride = n;
    return t;
  }
  at::Tensor rows = t.reshape({-1, n});
  if ((n > 1 && rows.stride(1) != 1) || (rows.size(0) > 1 && rows.stride(0) < 0)) rows = rows.contiguous();
  stride = rows.size(0) > 1 ? rows.stride(0) : n;
  return rows;
}

// x [..., K], a [E, r, K], b [E, N, r]; requests of as many rows each (none:
// all rows have adapter 0 of 1)
gtp_lora lora_of(const at::Tensor& x, const at::Tensor& a, const at::Tensor& b,
                 c10::optional<int64_t> requests, const char* what) {
  TORCH_CHECK(x.is_cuda() && x.dim() >= 1 && x.size(-1) > 0, "graspo_tokpath.", what,
              ": x must be a [..., K] GPU tensor");
  const int64_t K = x.size(-1);
  for (const auto* t : {&a, &b}) {
    check_same_device(x, *t, "the adapters");
    TORCH_CHECK(t->scalar_type() == x.scalar_type() && t->dim() == 3 && t->is_contiguous(),
                "graspo_tokpath.", what, ": adapters must be contiguous [E, r, K] and [E, N, r] of "
                "x's dtype");
  }
  const int64_t E = a.size(0), r = a.size(1), N = b.size(1);
  TORCH_CHECK(a.size(2) == K && b.size(0) == E && b.size(2) == r && E > 0 && r > 0 && N > 0,
              "graspo_tokpath.", what, ": adapters ", a.sizes(), " and ", b.sizes(),
              " do not go with x ", x.sizes());
  TORCH_CHECK(r <= 256 && E <= 1024, "graspo_tokpath.", what,
              ": at most 1024 adapters of rank 256, got ", E, " of ", r);
  gtp_lora q{};
  q.a = a.data_ptr();
  q.b = b.data_ptr();
  q.in = K;
  q.out = N;
  q.rank = (int32_t)r;
  q.adapters = (int32_t)E;
  q.dtype = dtype_code(x);
  const int64_t rows = x.numel() / K;
  if (requests.has_value()) {
    TORCH_CHECK(*requests > 0 ? rows % *requests == 0 : rows == 0, "graspo_tokpath.", what, ": ",
                rows, " rows are not those of ", *requests, " requests");
    q.ids = &q;  // (there; the forward says where)
    q.requests = *requests;
    q.rows = q.requests > 0 ? rows / q.requests : 0;
  } else {
    TORCH_CHECK(E == 1, "graspo_tokpath.", what, ": ", E, " adapters and no adapter_ids");
    q.requests = 1;
    q.rows = rows;
  }
  return q;
}

// (base + s x a^T b^T, what the backward takes of it)
std::tuple<at::Tensor, at::Tensor> lora_add_state(const at::Tensor& base, const at::Tensor& x,
                                                  const at::Tensor& a, const at::Tensor& b,
                                                  const c10::optional<at::Tensor>& ids,
                                                  const c10::optional<at::Tensor>& scales,
                                                  double scale, bool check, int64_t stream) {
  c10::optional<int64_t> requests;
  if (ids.has_value()) {
    check_same_device(x, *ids, "adapter_ids");
    TORCH_CHECK((ids->scalar_type() == at::kInt || ids->scalar_type() == at::kLong) &&
                    ids->dim() == 1 && ids->is_contiguous(),
                "graspo_tokpath.lora_add: adapter_ids must be contiguous int32 or int64 [requests]");
    requests = ids->size(0);
  }
  gtp_lora q = lora_of(x, a, b, requests, "lora_add");
  if (ids.has_value()) {
    q.ids = ids->data_ptr();
    q.ids_int64 = ids->scalar_type() == at::kLong;
  }
  q.scale = (float)scale;
  if (scales.has_value()) {
    check_same_device(x, *scales, "scaling");
    TORCH_CHECK(scales->scalar_type() == at::kFloat && scales->dim() == 1 &&
                    scales->size(0) == q.adapters && scales->is_contiguous(),
                "graspo_tokpath.lora_add: scaling must be contiguous float32 [E]");
    q.scales = scales->data_ptr<float>();
  }
  check_same_device(x, base, "base");
  TORCH_CHECK(base.scalar_type() == x.scalar_type() && base.dim() == x.dim() &&
                  base.sizes().slice(0, base.dim() - 1) == x.sizes().slice(0, x.dim() - 1) &&
                  base.size(-1) == q.out,
              "graspo_tokpath.lora_add: base must be [..., N] beside x [..., K], of its dtype; got ",
              base.sizes(), " and ", x.sizes());
  const c10::DeviceGuard guard(x.device());
  const at::Tensor xr = as_rows(x, q.in, q.x_stride), br = as_rows(base, q.out, q.base_stride);
  at::Tensor out = at::empty(base.sizes(), base.options());
  q.x = xr.data_ptr();
  q.base = br.data_ptr();
  q.y = out.data_ptr();
  at::Tensor state = at::empty({(int64_t)gtp_lora_state_bytes(&q)}, x.options().dtype(at::kByte));
  void* st = reinterpret_cast<void*>(stream);
  at::Tensor words, shifted;
  check = check && ids.has_value() && q.requests * q.rows > 0 && !gtp_stream_capturing(st);
  if (check) {
    // (-1, no adapter, is one of the good ones)
    shifted = at::add(*ids, 1);
    words = verdict_words();
    const int rc = gtp_targets_verdict(shifted.data_ptr(), q.ids_int64, q.requests, 1,
                                       q.adapters + 1, nullptr, nullptr, verdict_ptr(words), st);
    int found = 0;
    if (rc == GTP_ERR_LAUNCH) verdict_wait(words, &found, st);
    check_rc(rc, "gtp_targets_verdict");
  }
  const int rc = gtp_lora_add(&q, state.data_ptr(), (size_t)state.numel(), st);
  int bad = 0, wait_rc = GTP_OK;
  if (check) wait_rc = verdict_wait(words, &bad, st);
  check_rc(rc, "gtp_lora_add");
  check_rc(wait_rc, "gtp_verdict_wait");
  TORCH_CHECK(!(bad & 1), "lora_add: an adapter id is outside [-1, ", q.adapters, ")");
  return {out, state};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> lora_backward(
    const at::Tensor& grad, const at::Tensor& x, const at::Tensor& a, const at::Tensor& b,
    const at::Tensor& state, c10::optional<int64_t> requests, bool need_x, bool need_a, bool need_b,
    int64_t stream) {
  gtp_lora q = lora_of(x, a, b, requests, "lora_backward");
  if (requests.has_value()) q.ids = state.data_ptr();
  check_same_device(x, grad, "grad");
  check_same_device(x, state, "state");
  TORCH_CHECK(grad.scalar_type() == x.scalar_type() && grad.dim() >= 1 && grad.size(-1) == q.out &&
                  grad.numel() == q.requests * q.rows * q.out,
              "graspo_tokpath.lora_backward: grad must be the output's shape and dtype");
  TORCH_CHECK(state.scalar_type() == at::kByte && state.is_contiguous() &&
                  (size_t)state.numel() == gtp_lora_state_bytes(&q),
              "graspo_tokpath.lora_backward: the state is not one of these sizes");
  const c10::DeviceGuard guard(x.device());
  const at::Tensor xr = as_rows(x, q.in, q.x_stride);
  q.x = xr.data_ptr();
  gtp_lora_grads d{};
  const at::Tensor gr = as_rows(grad, q.out, d.grad_stride);
  d.grad = gr.data_ptr();
  at::Tensor gx, ga, gb;
  const bool none = q.requests * q.rows == 0;
  if (need_x) gx = at::empty(x.sizes(), x.options());
  if (need_a) ga = none ? at::zeros(a.sizes(), a.options()) : at::empty(a.sizes(), a.options());
  if (need_b) gb = none ? at::zeros(b.sizes(), b.options()) : at::empty(b.sizes(), b.options());
  if (none || !(need_x || need_a || need_b)) return {gx, ga, gb};
  d.grad_x = need_x ? gx.data_ptr() : nullptr;
  d.grad_a = need_a ? ga.data_ptr() : nullptr;
  d.grad_b = need_b ? gb.data_ptr() : nullptr;
  at::Tensor ws = at::empty({(int64_t)gtp_lora_backward_workspace_bytes(&q)},
                            x.options().dtype(at::kByte));
  check_rc(gtp_lora_backward(&q, &d, state.data_ptr(), (size_t)state.numel(), ws.data_ptr(),
                             (size_t)ws.numel(), reinterpret_cast<void*>(stream)),
           "gtp_lora_backward");
  return {gx, ga, gb};
}

struct LoraAdd : torch::autograd::Function<LoraAdd> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& base,
                            const at::Tensor& x, const at::Tensor& a, const at::Tensor& b,
                            const c10::optional<at::Tensor>& ids,
                            const c10::optional<at::Tensor>& scales, double scale, bool check,
                            int64_t stream) {
    auto [out, state] = lora_add_state(base, x, a, b, ids, scales, scale, check, stream);
    // (the state holds the ids' order and the scales, which the caller may refill
    // before the backward)
    ctx->save_for_backward({x, a, b, state});
    ctx->saved_data["requests"] = ids.has_value() ? ids->size(0) : -1;
    ctx->saved_data["stream"] = stream;
    return out;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const char* what = "lora_add";
    check_no_tangent(grads[0], what);
    const auto saved = ctx->get_saved_variables();
    c10::optional<int64_t> requests = ctx->saved_data["requests"].toInt();
    if (*requests < 0) requests = c10::nullopt;
    const bool nx = ctx->needs_input_grad(1), na = ctx->needs_input_grad(2),
               nb = ctx->needs_input_grad(3);
    // (the engine runs a node on its forward's stream)
    auto [gx, ga, gb] = lora_backward(grads[0].detach(), saved[0].detach(), saved[1].detach(),
                                      saved[2].detach(), saved[3], requests, nx, na, nb,
                                      ctx->saved_data["stream"].toInt());
    return {ctx->needs_input_grad(0) ? grads[0] : at::Tensor(),
            once_only(gx, grads[0], what), once_only(ga, grads[0], what),
            once_only(gb, grads[0], what), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(),
            at::Tensor()};
  }
};

// What lora_add refuses whatever the device (here, and not in Python, where it
// takes 3 us of a call of 12).
void check_lora(const at::Tensor& base, const at::Tensor& x, const at::Tensor& a,
                const at::Tensor& b, const c10::optional<at::Tensor>& ids,
                const c10::optional<at::Tensor>& scales) {
  const at::ScalarType dt = x.scalar_type();
  TORCH_CHECK_VALUE(dt == at::kFloat || dt == at::kBFloat16 || dt == at::kHalf,
                    "lora_add: x must be float32, bfloat16 or float16, got ", dt);
  const std::pair<const char*, const at::Tensor*> others[] = {
      {"base", &base}, {"lora_a", &a}, {"lora_b", &b}};
  for (const auto& o : others)
    TORCH_CHECK_VALUE(o.second->scalar_type() == dt, "lora_add: ", o.first, " must be ", dt,
                      " as x, got ", o.second->scalar_type());
  TORCH_CHECK_VALUE((a.dim() == 2 || a.dim() == 3) && b.dim() == a.dim(),
                    "lora_add: expected adapters [E, r, K] and [E, N, r] (or [r, K] and [N, r]), "
                    "got ", a.sizes(), " and ", b.sizes());
  const int64_t E = a.dim() == 3 ? a.size(0) : 1, r = a.size(-2), K = a.size(-1), N = b.size(-2);
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) == K && b.size(-1) == r &&
                        (a.dim() == 2 || b.size(0) == E) && base.dim() == x.dim() &&
                        base.size(-1) == N &&
                        base.sizes().slice(0, x.dim() - 1) == x.sizes().slice(0, x.dim() - 1) &&
                        E > 0 && r > 0 && K > 0 && N > 0,
                    "lora_add: base ", base.sizes(), ", x ", x.sizes(), " and adapters ", a.sizes(),
                    ", ", b.sizes(), " do not go together");
  TORCH_CHECK_VALUE(r <= 256 && E <= 1024, "lora_add: at most 1024 adapters of rank 256, got ", E,
                    " of ", r);
  if (ids.has_value()) {
    TORCH_CHECK_VALUE(ids->scalar_type() == at::kInt || ids->scalar_type() == at::kLong,
                      "lora_add: adapter_ids must be int32 or int64, got ", ids->scalar_type());
    TORCH_CHECK_VALUE(ids->dim() >= 1 && ids->dim() < x.dim() &&
                          ids->sizes() == x.sizes().slice(0, ids->dim()),
                      "lora_add: adapter_ids ", ids->sizes(),
                      " are not of the leading dimensions of x ", x.sizes());
  } else {
    TORCH_CHECK_VALUE(E == 1, "lora_add: ", E, " adapters and no adapter_ids");
  }
  if (scales.has_value()) {
    TORCH_CHECK_VALUE(scales->scalar_type() == at::kFloat && scales->dim() == 1 &&
                          scales->size(0) == E,
                      "lora_add: scaling must be a number or float32 [", E, "], got ",
                      scales->scalar_type(), " ", scales->sizes());
    TORCH_CHECK_VALUE(!scales->requires_grad(), "lora_add: the scaling has no gradient");
  }
  TORCH_CHECK(x.is_cuda(), "graspo_tokpath: tensors must be on a GPU (got ", x.device(),
              "); there is no CPU path");
}

at::Tensor lora_add(const at::Tensor& base, const at::Tensor& x, const at::Tensor& a,
                    const at::Tensor& b, const c10::optional<at::Tensor>& ids_,
                    const c10::optional<at::Tensor>& scales_, double scale, bool check,
                    int64_t stream) {
  check_lora(base, x, a, b, ids_, scales_);
  c10::optional<at::Tensor> ids, scales;
  if (ids_.has_value()) ids = ids_->dim() == 1 ? ids_->contiguous() : ids_->reshape({-1}).contiguous();
  if (scales_.has_value()) scales = scales_->contiguous();
  bool grad = false;
  for (const at::Tensor* t : {&base, &x, &a, &b}) {
    check_no_tangent(*t, "lora_add");
    grad = grad || t->requires_grad();
  }
  grad = grad && at::GradMode::is_enabled();
  if (grad)
    for (const at::Tensor* t : {&base, &x, &a, &b}) check_leaf(*t, "lora_add", stream);
  // a single adapter without its dimension, and views of a larger tensor
  const at::Tensor a3 = (a.dim() == 2 ? a.unsqueeze(0) : a).contiguous();
  const at::Tensor b3 = (b.dim() == 2 ? b.unsqueeze(0) : b).contiguous();
  if (grad) return LoraAdd::apply(base, x, a3, b3, ids, scales, scale, check, stream);
  return std::get<0>(lora_add_state(base, x, a3, b3, ids, scales, scale, check, stream));
}

TORCH_LIBRARY(graspo_tokpath, m) {
  m.def("lora_add_state(Tensor base, Tensor x, Tensor a, Tensor b, Tensor? ids, Tensor? scales, "
        "float scale, bool check, int stream) -> (Tensor, Tensor)",
        &lora_add_state);
  m.def("lora_backward(Tensor grad, Tensor x, Tensor a, Tensor b, Tensor state, int? requests, "
        "bool need_x, bool need_a, bool need_b, int stream) -> (Tensor, Tensor, Tensor)",
        &lora_backward);
  m.def("lora_add(Tensor base, Tensor x, Tensor a, Tensor b, Tensor? ids, Tensor? scales, "
        "float scale, bool check, int stream) -> Tensor",
        &lora_add);
  m.def(
      "beam_candidates(Tensor logits, Tensor scores, int candidates, Tensor? allow_mask, "
      "Tensor? done, int stream) -> (Tensor, Tensor, Tensor, Tensor)",
      &beam_candidates);
  m.def(
      "beam_advance(Tensor c_scores, Tensor c_beams, Tensor c_tokens, Tensor scores, "
      "Tensor pool_scores, Tensor pool_rows, Tensor pool_steps, Tensor done, int eos, int pad, "
      "float length, int step, bool early, Tensor(a!)? tokens_out, Tensor(b!)? parents_out, "
      "int stream) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)",
      &beam_advance);
  m.def(
      "beam_step(Tensor logits, Tensor scores, Tensor pool_scores, Tensor pool_rows, "
      "Tensor pool_steps, Tensor done, int candidates, int eos, int pad, float length, int step, "
      "bool early, Tensor? allow_mask, Tensor(a!)? tokens_out, Tensor(b!)? parents_out, "
      "int stream) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)",
      &beam_step);
  m.def(
      "beam_finish(Tensor scores, Tensor pool_scores, Tensor pool_rows, Tensor pool_steps, "
      "Tensor done, Tensor tokens, Tensor parents, float length, int eos, int pad, int give, "
      "int stream) -> (Tensor, Tensor, Tensor)",
      &beam_finish);
  m.def("reorder_states_(Tensor(a!)[] states, Tensor parents, int beams, bool check, int stream) "
        "-> ()",
        &reorder_states_);
  m.def("expand_states(Tensor[] states, int beams, int stream) -> Tensor[]", &expand_states);
  m.def("embedding(Tensor ids, Tensor weight, float scale, bool check, bool ordered, int padding_idx, "
        "int stream) -> (Tensor, bool, Tensor)",
        &embedding);
  m.def(
      "embedding_backward(Tensor? ids, Tensor grad, int vocab, float scale, int padding_idx, "
      "Tensor(a!)? out, Tensor? order, int stream) -> Tensor",
      &embedding_backward);
  m.def("linear_loss(Tensor hidden, Tensor weight, Tensor targets, int? ignore_index, bool mean, "
        "str what, int stream) -> Tensor",
        &linear_loss);
  m.def("token_embedding(Tensor ids, Tensor weight, float scale, int padding_idx, bool check, "
        "int stream) -> Tensor",
        &token_embedding);
  m.def("grad_norm(Tensor[] tensors, float norm_type, int stream) -> Tensor", &grad_norm);
  m.def("clip_grads_(Tensor(a!)[] tensors, Tensor norm, float max_norm, int stream) -> ()",
        &clip_grads_);
  m.def(
      "clip_grad_norm_(Tensor(a!)[] tensors, float max_norm, float norm_type, int stream) -> Tensor",
      &clip_grad_norm_);
  m.def(
      "linear_logprob(Tensor hidden, Tensor weight, Tensor targets, int? ignore_index, bool mean, "
      "int stream) -> (Tensor, Tensor, Tensor, Tensor, bool)",
      &linear_logprob);
  m.def(
      "linear_logprob_backward(Tensor hidden, Tensor weight, Tensor targets, Tensor lse, "
      "Tensor grad, Tensor? mean_count, int? ignore_index, bool need_hidden, bool need_weight, "
      "int stream) -> (Tensor, Tensor)",
      &linear_logprob_backward);
  m.def(
      "sample(Tensor logits, float temperature, int top_k, float top_p, float repetition_penalty, "
      "Tensor? history, Tensor? allow_mask, Tensor? uniforms, Tensor? finished, int pad_token_id, "
      "int stream) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)",
      &sample);
  m.def(
      "sample_route(Tensor logits, float temperature, int top_k, float top_p, "
      "float repetition_penalty, int hist_len, bool has_mask) -> (int, int)",
      &sample_route);
  m.def(
      "sample_spread(Tensor logits, float temperature, int top_k, float top_p, "
      "float repetition_penalty, int hist_len, bool has_mask) -> bool",
      &sample_spread);
  m.def("logprob_entropy(Tensor logits, Tensor targets, int stream) -> (Tensor, Tensor, Tensor)",
        &logprob_entropy);
  m.def(
      "token_logprob(Tensor logits, Tensor targets, int? ignore_index, bool entropy, bool mean, "
      "int stream) -> (Tensor, Tensor, Tensor, Tensor, bool)",
      &token_logprob);
  m.def(
      "verdict_begin(Tensor targets, int vocab, Tensor? flag_a, Tensor? flag_b, int stream) -> "
      "Tensor",
      &verdict_begin);
  m.def("verdict_end(Tensor words, int stream) -> int", &verdict_end);
  m.def(
      "token_logprob_backward(Tensor logits, Tensor targets, Tensor logprob, Tensor grad, "
      "Tensor? mean_count, int? ignore_index, int stream) -> Tensor",
      &token_logprob_backward);
  m.def(
      "lse_partial(Tensor logits, Tensor? targets, int col_offset, Tensor(a!) state, "
      "bool accumulate, int stream) -> ()",
      &lse_partial);
  m.def("lse_finalize(Tensor state, int stream) -> (Tensor, Tensor)", &lse_finalize);
  m.def(
      "logprob_backward(Tensor logits, Tensor targets, Tensor grad_logprob, Tensor lse, "
      "int col_offset, Tensor(a!)? out, int stream) -> Tensor",
      &logprob_backward);
  m.def(
      "graspo_loss_forward(Tensor log_probs, Tensor old_log_probs, Tensor advantages, "
      "Tensor? action_mask, float clip_lo, float clip_hi, int stream) -> (Tensor, Tensor, Tensor)",
      &graspo_loss_forward);
  m.def(
      "graspo_loss_backward(Tensor log_probs, Tensor old_log_probs, Tensor advantages, "
      "Tensor? action_mask, Tensor inv_denom, Tensor grad_loss, float clip_lo, float clip_hi, "
      "int stream) -> Tensor",
      &graspo_loss_backward);
  m.def(
      "decode_update(Tensor(e!) ids, Tensor? status, Tensor(a!) finished, int eos_token_id, "
      "int pad_token_id, Tensor(b!)? sequences, Tensor(c!)? attention_mask, int col, "
      "Tensor(d!) flags, int stream) -> ()",
      &decode_update);
  m.def("to_bf16_exact(Tensor src, int stream) -> (Tensor, Tensor)", &to_bf16_exact);
  m.def("time_next_launch(int start_event, int stop_event) -> ()", &time_next_launch);
  m.def(
      "logprob_backward_split(Tensor logits, Tensor targets, Tensor grad_logprob, Tensor lse, "
      "int col_offset, int stream) -> (Tensor, Tensor)",
      &logprob_backward_split);
  m.def("lm_head_logprob(Tensor hidden, Tensor weight, Tensor targets, int stream) -> "
        "(Tensor, Tensor, Tensor)",
        &lm_head_logprob);
  m.def("lm_head_logprob_save(Tensor hidden, Tensor weight, Tensor targets, int stream) -> "
        "(Tensor, Tensor, Tensor, Tensor)",
        &lm_head_logprob_save);
  m.def("softmax_grad_bf16(Tensor logits_t, Tensor grad_logprob, Tensor lse, int layouts, int stream) -> (Tensor, Tensor)",
        &softmax_grad_bf16);
}
