// Python bindings of the operators for packed rows: masked attention and its form for
// single tokens, the norms and rotation of queries and keys, log probabilities.

#include "bindings.h"

#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <algorithm>
#include <cmath>
#include <limits>
#include <tuple>
#include <unordered_set>

extern "C" int ds_packed_spans(const void* ids, int wide, const int* prefix,
                               int* spans, int B, int S, int N, int causal,
                               void* stream);
extern "C" int ds_masked_attention(
    const void* q, const void* k, const void* v, void* out, float* lse,
    void* rest, const void* dout, void* dq, void* dk, void* dv, float* stat,
    float* part, int splits, const int* spans, const float* slopes,
    const long long* strides, int B, int S, int H, int Hkv, int D, int causal,
    float scale, float cap, void* stream);
extern "C" int ds_paged_shaped(const void* q, const void* kpool,
                               const void* vpool, const int* table,
                               const int* lens, const float* slopes, void* out,
                               float* part, float* part_ml, int n, int H,
                               int Hkv, int BS, int max_blocks, int blocks,
                               int splits, float scale, float cap,
                               void* stream);
extern "C" int ds_flash_bwd_splits(int B, int S, int H, int Hkv);
extern "C" int ds_qk_norm_parts(int tokens);
extern "C" int ds_qk_norm_rope(
    const void* q, const void* k, void* yq, void* yk, const void* dq,
    const void* dk, const void* wq, const void* wk, const float* cs,
    const float* sn, const int* positions, const long long* strides, int B,
    int S, int H, int Hk, int D, int rotated, int angles, int half, float eps,
    float plus, int type, float* part, int parts, void* dwq, void* dwk,
    void* stream);
extern "C" int ds_logprobs_parts(int rows, long long V, int top);
extern "C" int ds_logprobs_fwd(const void* x, long long outer_stride,
                               long long inner_stride, int inner, int type,
                               const long long* tokens, float* lp, float* ent,
                               float* stat, float* top_lp, long long* top_ids,
                               float* sums, void* lists, int rows, long long V,
                               int parts, int top, long long ignore,
                               void* stream);
extern "C" int ds_logprobs_bwd(const void* x, long long outer_stride,
                               long long inner_stride, int inner, int type,
                               const long long* tokens, const float* stat,
                               const float* ent, const float* glp,
                               const float* gent, void* dx, int rows,
                               long long V, long long ignore, void* stream);

namespace {

using Opt = c10::optional<at::Tensor>;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Threads of a launch are counted in 32 bits.
constexpr int64_t THREADS = 1ll << 32;

void* data(const Opt& t) {
  return t.has_value() && t->defined() ? t->data_ptr() : nullptr;
}

Tensor or_none(const Opt& t) { return t.has_value() ? *t : Tensor(); }

// The operators' autograd is here, not in Python: a backward pass of a few tens of us
// waits as long again for the interpreter's lock in the engine's thread (a short
// attention, there and back: 105 us so, 55 of them an empty Python function's).
// What has no gradient of its own says so when one is asked for.
variable_list no_further(variable_list results, const std::string& message) {
  if (!at::GradMode::is_enabled()) return results;
  for (auto& t : results)
    if (t.defined()) t = t.detach().requires_grad_(true);
  const int64_t n = results.size();
  auto node = std::make_shared<torch::autograd::DelayedError>(message, n);
  return node->apply(std::move(results));
}

// Gradients: a second derivative raises.
variable_list once(variable_list grads, const char* what) {
  return no_further(std::move(grads), std::string(what) + " is differentiable once");
}

// Gradients that come in: those asked for in batches have no memory of their own.
void check_single(const variable_list& grads, const char* what) {
  for (const auto& g : grads)
    TORCH_CHECK(!g.defined() || g.has_storage(), what,
                ": gradients one after another, not in batches (is_grads_batched)");
}

bool wants_grad(const Tensor& t) {
  return at::GradMode::is_enabled() && t.requires_grad();
}

// An eager graph that lives keeps the place of its leaves' gradients on the stream it
// was made on. On the default one, which no capture can take in, a captured backward
// of the same leaves ends the process: such a forward is refused. The leaves are mostly
// not the inputs themselves but the weights that these come from, so they are looked for
// through the whole graph behind the inputs, while a capture is about and only then.
void check_capture(const char* what,
                   std::initializer_list<const Tensor*> inputs) {
  using torch::autograd::Node;
  const auto now =
      c10::hip::getCurrentHIPStream((*inputs.begin())->device().index()).stream();
  if (now == nullptr) return;            // the default stream itself
  std::vector<const Node*> next;
  std::vector<std::shared_ptr<Node>> held;     // of the inputs that are leaves
  for (const auto* t : inputs) {
    if (!wants_grad(*t)) continue;
    if (t->is_leaf()) {
      held.push_back(torch::autograd::impl::try_get_grad_accumulator(*t));
      if (held.back()) next.push_back(held.back().get());
    } else {
      next.push_back(t->grad_fn().get());
    }
  }
  if (next.empty()) return;
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  TORCH_CHECK(hipStreamIsCapturing(now, &status) == hipSuccess, what,
              ": a stream of no capture status");
  if (status == hipStreamCaptureStatusNone) return;
  std::unordered_set<const Node*> seen(next.begin(), next.end());
  while (!next.empty()) {
    const Node* node = next.back();
    next.pop_back();
    if (dynamic_cast<const torch::autograd::AccumulateGrad*>(node)) {
      const auto kept = const_cast<Node*>(node)->stream();
      TORCH_CHECK(!kept || kept->id() != 0, what,
                  ": an eager graph of the same leaves lives, which a capture with "
                  "gradients cannot take in; end it before, or give the capture "
                  "leaves of its own");
    }
    for (const auto& edge : node->next_edges())
      if (edge.function && seen.insert(edge.function.get()).second)
        next.push_back(edge.function.get());
  }
}

at::Tensor packed_spans(at::Tensor ids, Opt prefix, bool causal) {
  const OneDevice on("packed_rows", ids, prefix);
  const bool wide = ids.scalar_type() == at::kLong;
  TORCH_CHECK(ids.is_cuda() && ids.dim() == 2 && ids.is_contiguous() &&
              (wide || ids.scalar_type() == at::kInt),
              "packed_rows: document_ids int32 or int64 [B, S]");
  const int64_t B = ids.size(0), S = ids.size(1);
  TORCH_CHECK(S < (1 << 30) && B <= 65535, "packed_rows: size");
  int64_t N = 0;
  if (data(prefix)) {
    TORCH_CHECK(prefix->scalar_type() == at::kInt && prefix->dim() == 2 &&
                prefix->size(0) == B && prefix->is_contiguous() && causal,
                "packed_rows: prefix_lens int32 [B, N], causal");
    N = prefix->size(1);
  }
  auto spans = at::empty({4, B, S}, ids.options().dtype(at::kInt));
  if (spans.numel() == 0) return spans;
  const int e = ds_packed_spans(
      ids.data_ptr(), wide, static_cast<const int*>(data(prefix)),
      spans.data_ptr<int>(), (int)B, (int)S, (int)N, causal, cur_stream());
  TORCH_CHECK(e == 0, "packed_rows: launch failed, hipError_t ", e);
  return spans;
}

struct MaskedArgs : FlashArgs {
  const int* spans = nullptr;
  const float* slopes = nullptr;
  MaskedArgs(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
             const Opt& spans_, const Opt& slopes_, double scale, double cap)
      : FlashArgs(q, k, v, scale, "masked_attention") {
    TORCH_CHECK((int64_t)B * H * ((S + 127) / 128) * 256 < THREADS,
                "masked_attention: size");
    if (data(spans_)) {
      TORCH_CHECK(spans_->scalar_type() == at::kInt &&
                  spans_->is_contiguous() && spans_->dim() == 3 &&
                  spans_->size(0) == 4 && spans_->size(1) == B &&
                  spans_->size(2) == S, "masked_attention: rows of another batch");
      spans = spans_->data_ptr<int>();
    }
    if (data(slopes_)) {
      TORCH_CHECK(slopes_->scalar_type() == at::kFloat &&
                  slopes_->is_contiguous() && slopes_->numel() == H,
                  "masked_attention: alibi_slopes fp32 [H]");
      slopes = slopes_->data_ptr<float>();
    }
  }
};

std::tuple<at::Tensor, at::Tensor, at::Tensor> masked_attn_fwd(
    at::Tensor q, at::Tensor k, at::Tensor v, Opt spans, Opt slopes,
    bool causal, double scale, double cap, bool with_rest) {
  const OneDevice on("masked_attention", q, k, v, spans, slopes);
  MaskedArgs a(q, k, v, spans, slopes, scale, cap);
  auto o = at::empty({a.B, a.S, a.H, a.D}, q.options());
  auto lse = at::empty({a.B, a.H, a.S}, q.options().dtype(at::kFloat));
  auto rest = at::empty({with_rest ? o.numel() : 0},
                        q.options().dtype(at::kChar));
  a.add(q, q); a.add(k, k); a.add(v, k); a.add(o, q);
  if (q.numel()) {
    const int e = ds_masked_attention(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
        lse.data_ptr<float>(), with_rest ? rest.data_ptr() : nullptr, nullptr,
        nullptr, nullptr, nullptr, nullptr, nullptr, 0, a.spans, a.slopes,
        a.strides.data(), a.B, a.S, a.H, a.Hkv, a.D, causal, (float)scale,
        (float)cap, cur_stream());
    TORCH_CHECK(e == 0, "masked_attention: launch failed, hipError_t ", e);
  }
  return {o, lse, rest};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> masked_attn_bwd(
    at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor o, at::Tensor dout,
    at::Tensor lse, at::Tensor rest, Opt spans, Opt slopes, bool causal,
    double scale, double cap) {
  const OneDevice on("masked_attention", q, k, v, o, dout, lse, rest, spans,
                     slopes);
  MaskedArgs a(q, k, v, spans, slopes, scale, cap);
  TORCH_CHECK(lse.scalar_type() == at::kFloat && lse.is_contiguous() &&
              lse.numel() == (int64_t)a.B * a.H * a.S &&
              rest.scalar_type() == at::kChar && rest.is_contiguous() &&
              rest.numel() == o.numel(), "masked_attention: lse");
  const int splits = ds_flash_bwd_splits(a.B, a.S, a.H, a.Hkv);
  auto dq = at::empty({a.B, a.S, a.H, a.D}, q.options());
  auto dk = at::empty({a.B, a.S, a.Hkv, a.D}, q.options());
  auto dv = at::empty({a.B, a.S, a.Hkv, a.D}, q.options());
  auto stat = at::empty_like(lse);
  auto part = at::empty({splits > 1 ? 2 * splits * dk.numel() : 0},
                        lse.options());
  a.add(q, q); a.add(k, k); a.add(v, k); a.add(o, q); a.add(dout, q);
  if (q.numel()) {
    const int e = ds_masked_attention(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
        lse.data_ptr<float>(), rest.data_ptr(), dout.data_ptr(), dq.data_ptr(),
        dk.data_ptr(), dv.data_ptr(), stat.data_ptr<float>(),
        part.data_ptr<float>(), splits, a.spans, a.slopes, a.strides.data(), a.B, a.S, a.H, a.Hkv, a.D, causal,
        (float)scale, (float)cap, cur_stream());
    TORCH_CHECK(e == 0, "masked_attention: launch failed, hipError_t ", e);
  }
  return {dq, dk, dv};
}

// x as the attention kernels read it: unit stride inside a head, 16-byte rows.
Tensor rows_of(const Tensor& x) {
  bool fits = x.stride(3) == 1 && (uintptr_t)x.data_ptr() % 16 == 0 &&
              x.stride(1) < (1 << 24);
  for (int d = 0; d < 3; ++d)
    fits = fits && x.stride(d) % 8 == 0 && x.stride(d) >= 0;
  return fits ? x : x.clone(at::MemoryFormat::Contiguous);
}

struct MaskedAttention : torch::autograd::Function<MaskedAttention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q_, const Tensor& k_,
                        const Tensor& v_, const Opt& spans,
                        const Opt& slopes, bool causal, double scale,
                        double cap, bool grads) {
    // the kernels take maxima of scores that a positive scale has left in order
    auto q = q_;
    double factor = 1;
    if (!(scale >= std::numeric_limits<float>::min())) {
      const bool flips = scale <= -std::numeric_limits<float>::min();
      factor = flips ? -1 : scale;      // or 0, and what is as good as that in fp32
      q = q * factor;
      scale = flips ? -scale : 1;
    }
    q = rows_of(q);
    const auto k = rows_of(k_), v = rows_of(v_);
    auto [o, lse, rest] =
        masked_attn_fwd(q, k, v, spans, slopes, causal, scale, cap, grads);
    if (grads) {
      ctx->save_for_backward({q, k, v, o, lse, rest, or_none(spans),
                              or_none(slopes)});
      ctx->saved_data["causal"] = causal;
      ctx->saved_data["scale"] = scale;
      ctx->saved_data["cap"] = cap;
      ctx->saved_data["factor"] = factor;
    }
    return o;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    check_single(g, "masked_attention");
    const auto t = ctx->get_saved_variables();
    const double factor = ctx->saved_data["factor"].toDouble();
    auto [dq, dk, dv] = masked_attn_bwd(
        t[0], t[1], t[2], t[3], rows_of(g[0]), t[4], t[5], t[6], t[7],
        ctx->saved_data["causal"].toBool(), ctx->saved_data["scale"].toDouble(),
        ctx->saved_data["cap"].toDouble());
    if (factor != 1) dq = dq * factor;
    variable_list grads = once({dq, dk, dv}, "masked_attention");
    grads.resize(9);
    return grads;
  }
};

Opt slopes_of(const Opt& t, const Tensor& q, const char* what) {
  if (!t.has_value()) return t;
  TORCH_CHECK_VALUE(!t->requires_grad(), what, ": alibi_slopes have no gradient");
  TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == q.size(-2) &&
                    t->is_floating_point(),
                    what, ": alibi_slopes is one number a query head, got ",
                    t->sizes());
  TORCH_CHECK_VALUE(t->device() == q.device(),
                    what, ": tensors on different devices");
  return t->to(at::kFloat).contiguous();
}

void check_cap(double softcap, const char* what) {
  TORCH_CHECK_VALUE(softcap == 0 || (softcap > 1e-30 && softcap < 1e30), what,
                    ": softcap is 0 (none) or positive, got ", softcap);
}

Tensor masked_attention(const Tensor& q, const Tensor& k, const Tensor& v,
                        const Opt& spans, const Opt& alibi_slopes, bool causal,
                        c10::optional<double> scale, double softcap) {
  TORCH_CHECK_VALUE(
      q.dim() == 4 && k.dim() == 4 && k.sizes() == v.sizes() &&
      q.size(0) == k.size(0) && q.size(1) == k.size(1) &&
      q.size(3) == k.size(3) && k.size(2) > 0 && q.size(2) > 0 &&
      q.size(2) % k.size(2) == 0,
      "masked_attention: q is [B, S, H, D], k and v are [B, S, Hkv, D] with H a "
      "multiple of Hkv, got ", q.sizes(), ", ", k.sizes(), ", ", v.sizes());
  TORCH_CHECK_VALUE(q.scalar_type() == k.scalar_type() &&
                    q.scalar_type() == v.scalar_type(),
                    "masked_attention: q, k and v of one type");
  TORCH_CHECK_VALUE(q.scalar_type() == at::kBFloat16 &&
                    (q.size(3) == 64 || q.size(3) == 96 || q.size(3) == 128),
                    "masked_attention: bf16 and heads of 64, 96 or 128 on a GPU, "
                    "got ", q.scalar_type(), " and ", q.size(3));
  check_cap(softcap, "masked_attention");
  TORCH_CHECK_VALUE(!spans.has_value() ||
                    (spans->dim() == 3 && spans->size(1) == q.size(0) &&
                     spans->size(2) == q.size(1) && spans->device() == q.device()),
                    "masked_attention: rows of another batch or device");
  const Opt slopes = slopes_of(alibi_slopes, q, "masked_attention");
  TORCH_CHECK_VALUE(k.device() == q.device() && v.device() == q.device(),
                    "masked_attention: tensors on different devices");
  check_capture("masked_attention", {&q, &k, &v});
  return MaskedAttention::apply(
      q, k, v, spans, slopes, causal,
      scale.has_value() ? *scale : 1.0 / std::sqrt((double)q.size(3)), softcap,
      wants_grad(q) || wants_grad(k) || wants_grad(v));
}

Tensor aligned(const Tensor& t) {     // contiguous, on 16 bytes
  const auto x = t.contiguous();
  return (uintptr_t)x.data_ptr() % 16 == 0 ? x : x.clone();
}

// Numbers of 64 bits in 32: one that does not fit is the nearest that does, which is as
// far outside of any pool or table, and not some other's that it would wrap to.
Tensor in_32_bits(const Tensor& t) {
  return (t.scalar_type() == at::kLong
              ? t.clamp(std::numeric_limits<int>::min(),
                        std::numeric_limits<int>::max())
              : t).to(at::kInt).contiguous();
}

// Parts of each request, of whose keys the table's width is all that the host knows. us
// from cold caches, whole / in these parts, groups of heads times requests by keys:
//   up to 512 keys whole: 8 x 350 8.7, in two parts 10.0
//   up to 80 groups a workgroup a CU, of 125 keys at least: 8 x 700 13.0 / 10.8, 8 x
//     4000 47 / 13, 32 x 4000 49 / 19, 72 x 12000 138 / 67
//   more: whole up to 1024 keys (136 x 700 14.7, in 5 parts 16.7), and where they come
//     to nearly one a CU (216 x 4000 58.8, in 7 parts 60.5; 256 x 2000 35.8, in 3 parts
//     40.0), but for very long ones
//   else the fewest parts, of 500 keys at least, that fill nine tenths of a round of
//     three workgroups a CU: 136 x 4000 52 / 43, 288 x 4000 96 / 77, 384 x 4000 110 /
//     99, 864 x 4000 200 / 187, 216 x 12000 157 / 140
int64_t shaped_splits(int64_t groups, int64_t keys) {
  if (keys <= 512) return 1;
  if (groups <= 80) return std::clamp<int64_t>(256 / groups, 1,
                                               std::clamp<int64_t>(keys / 125, 1, 32));
  if (keys <= 1024 || (groups >= 176 && groups <= 256 && keys < 8000)) return 1;
  const int64_t most = std::min<int64_t>(16, keys / 500);
  int64_t best = 1;
  double fill = 0;
  for (int64_t n = 1; n <= most && fill < 0.9; ++n) {
    const int64_t all = groups * n, rounds = (all + 767) / 768;
    if (all / (768.0 * rounds) > fill && (all >= 700 || n == 1)) {
      fill = all / (768.0 * rounds);
      best = n;
    }
  }
  return best;
}

// splits 0: by sizes.
Tensor paged_shaped(const Tensor& q_, const Tensor& kpool_,
                    const Tensor& vpool_, const Tensor& table_,
                    const Tensor& lens_, int64_t splits,
                    c10::optional<double> scale, double softcap,
                    const Opt& alibi_slopes) {
  const char* what = "paged_decode_attention";
  TORCH_CHECK_VALUE(q_.dim() == 3 && kpool_.dim() == 4 &&
                    kpool_.sizes() == vpool_.sizes() &&
                    q_.size(2) == kpool_.size(3) && kpool_.size(1) > 0 &&
                    q_.size(1) % kpool_.size(1) == 0 && kpool_.size(2) > 0,
                    what, ": q is [n, H, D], the pools are [blocks, Hkv, BS, D] "
                    "with H a multiple of Hkv, got ", q_.sizes(), ", ",
                    kpool_.sizes(), ", ", vpool_.sizes());
  TORCH_CHECK_VALUE(table_.dim() == 2 && table_.size(0) == q_.size(0) &&
                    lens_.dim() == 1 && lens_.size(0) == q_.size(0),
                    what, ": block_table is [n, blocks], lens [n]");
  TORCH_CHECK_VALUE(q_.scalar_type() == at::kBFloat16 &&
                    kpool_.scalar_type() == at::kBFloat16 &&
                    vpool_.scalar_type() == at::kBFloat16 &&
                    q_.size(2) == 128 && q_.size(1) <= 16 * kpool_.size(1),
                    what, ": bf16, heads of 128 and up to 16 a key head on a GPU");
  bool here = true;
  for (const auto* t : {&kpool_, &vpool_, &table_, &lens_})
    here = here && t->device() == q_.device();
  TORCH_CHECK_VALUE(here, what, ": tensors on different devices");
  check_cap(softcap, what);
  // keys and the steps behind the last of them are counted in 32 bits, and so are the
  // table's blocks
  constexpr int64_t KEYS = 1ll << 30;
  TORCH_CHECK_VALUE(kpool_.size(2) <= KEYS &&
                    table_.size(1) <= KEYS / kpool_.size(2) &&
                    table_.numel() < 2 * KEYS,
                    what, ": a table of up to 2^30 keys a request and 2^31 blocks");
  const Opt slopes = slopes_of(alibi_slopes, q_, what);
  const OneDevice on(what, q_);
  const auto q = aligned(q_), kpool = aligned(kpool_), vpool = aligned(vpool_);
  const auto table = in_32_bits(table_), lens = in_32_bits(lens_);
  const int64_t n = q.size(0), H = q.size(1), Hkv = kpool.size(1);
  const int64_t BS = kpool.size(2), groups = n * Hkv;
  auto o = at::empty_like(q);
  if (n == 0) return o;
  if (splits == 0) splits = shaped_splits(groups, table.size(1) * BS);
  TORCH_CHECK_VALUE(splits >= 1 && kpool.size(0) > 0 &&
                    kpool.size(0) < (1ll << 31) && H * 128 < (1ll << 31) &&
                    n * splits * 512 < THREADS && Hkv <= 65535,
                    what, ": size");
  const int64_t items = splits > 1 ? n * splits * Hkv * 16 : 0;
  auto part = at::empty({items * 130}, q.options().dtype(at::kFloat));
  float* p = part.data_ptr<float>();
  const int e = ds_paged_shaped(
      q.data_ptr(), kpool.data_ptr(), vpool.data_ptr(), table.data_ptr<int>(),
      lens.data_ptr<int>(), static_cast<const float*>(data(slopes)),
      o.data_ptr(), p, p + items * 128, (int)n, (int)H, (int)Hkv, (int)BS,
      (int)table.size(1), (int)kpool.size(0), (int)splits,
      (float)(scale.has_value() ? *scale : 1.0 / std::sqrt(128.0)),
      (float)softcap, cur_stream());
  TORCH_CHECK(e == 0, what, ": launch failed, hipError_t ", e);
  if (wants_grad(q_) || wants_grad(kpool_) || wants_grad(vpool_))
    return no_further({o}, std::string(what) + " has no gradient on a GPU: take "
                      "masked_attention")[0];
  return o;
}

// q [B, S, H, D], k [B, S, Hk, D], any strides but one inside a head; with dq and dk
// the backward: (dq, dk, dwq, dwk) instead of (q, k).
variable_list qk_norm_kernels(const Tensor& q, const Tensor& k, const Tensor& wq,
                              const Tensor& wk, const Tensor& cs,
                              const Tensor& sn, const Opt& positions,
                              double eps, bool half, bool one_plus, Opt dq,
                              Opt dk) {
  const OneDevice on("qk_norm_rope", q, k, wq, wk, cs, sn, positions, dq, dk);
  TORCH_CHECK(q.is_cuda() && q.dim() == 4 && k.dim() == 4 &&
              q.size(0) == k.size(0) && q.size(1) == k.size(1) &&
              q.size(3) == k.size(3), "qk_norm_rope: q [B, S, H, D], k [B, S, Hk, D]");
  const int64_t B = q.size(0), S = q.size(1), H = q.size(2), Hk = k.size(2);
  const int64_t D = q.size(3), tokens = B * S;
  const int type = dtype_code(q);
  TORCH_CHECK(D % 2 == 0 && D >= 2 && D <= 512, "qk_norm_rope: even heads up to 512");
  for (const auto& w : {wq, wk})
    TORCH_CHECK(w.dim() == 1 && w.size(0) == D && w.is_contiguous() &&
                w.scalar_type() == q.scalar_type(),
                "qk_norm_rope: weights [D] of the heads' type");
  for (const auto& t : {cs, sn})
    TORCH_CHECK(t.scalar_type() == at::kFloat && t.dim() == 2 &&
                t.is_contiguous() && t.sizes() == cs.sizes() && t.size(1) >= 1 &&
                2 * t.size(1) <= D && t.size(0) < (1ll << 31),
                "qk_norm_rope: tables fp32 [positions, rotated / 2]");
  if (data(positions)) {
    TORCH_CHECK(positions->scalar_type() == at::kInt &&
                positions->is_contiguous() && positions->numel() == tokens,
                "qk_norm_rope: positions int32, one a token");
  } else {
    TORCH_CHECK(S <= cs.size(0), "qk_norm_rope: tables shorter than the rows");
  }
  TORCH_CHECK(tokens * 64 < THREADS && H + Hk < (1 << 24), "qk_norm_rope: size");
  // (gradients of no tokens are there, but have no memory)
  const bool back = dq.has_value();
  std::vector<long long> strides;
  auto add = [&](const at::Tensor& t, const at::Tensor& like) {
    TORCH_CHECK(t.sizes() == like.sizes() &&
                (t.stride(3) == 1 || t.numel() == 0) &&
                t.scalar_type() == q.scalar_type(),
                "qk_norm_rope: heads of one type, unit stride inside them");
    for (int d = 0; d < 3; ++d) strides.push_back(t.stride(d));
  };
  add(q, q); add(k, k);
  if (back) {
    TORCH_CHECK(dk.has_value(), "qk_norm_rope: both gradients");
    add(*dq, q); add(*dk, k);
  }
  auto yq = at::empty({B, S, H, D}, q.options());
  auto yk = at::empty({B, S, Hk, D}, q.options());
  variable_list out = {yq, yk};
  const int parts = tokens ? ds_qk_norm_parts((int)tokens) : 0;
  at::Tensor part;
  if (back) {
    out.push_back(tokens ? at::empty_like(wq) : at::zeros_like(wq));
    out.push_back(tokens ? at::empty_like(wk) : at::zeros_like(wk));
    part = at::empty({parts, D}, q.options().dtype(at::kFloat));
  }
  if (tokens == 0) return out;
  const int e = ds_qk_norm_rope(
      q.data_ptr(), k.data_ptr(), yq.data_ptr(), yk.data_ptr(), data(dq),
      data(dk), wq.data_ptr(), wk.data_ptr(), cs.data_ptr<float>(),
      sn.data_ptr<float>(), static_cast<const int*>(data(positions)),
      strides.data(), (int)B, (int)S, (int)H, (int)Hk, (int)D,
      (int)(2 * cs.size(1)), (int)cs.size(0), half, (float)eps,
      one_plus ? 1.f : 0.f, type, back ? part.data_ptr<float>() : nullptr,
      parts, back ? out[2].data_ptr() : nullptr,
      back ? out[3].data_ptr() : nullptr, cur_stream());
  TORCH_CHECK(e == 0, "qk_norm_rope: launch failed, error ", e);
  return out;
}

Tensor inside(const Tensor& x) {     // unit stride inside a head
  return x.stride(-1) == 1 ? x : x.contiguous();
}

struct QkNorm : torch::autograd::Function<QkNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q_,
                               const Tensor& k_, const Tensor& wq_,
                               const Tensor& wk_, const Tensor& cs,
                               const Tensor& sn, const Opt& positions,
                               double eps, bool half, bool one_plus) {
    const auto q = inside(q_), k = inside(k_);
    const auto wq = wq_.contiguous(), wk = wk_.contiguous();
    auto out = qk_norm_kernels(q, k, wq, wk, cs, sn, positions, eps, half,
                               one_plus, c10::nullopt, c10::nullopt);
    ctx->save_for_backward({q, k, wq, wk, cs, sn, or_none(positions)});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["half"] = half;
    ctx->saved_data["one_plus"] = one_plus;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    check_single(g, "qk_norm_rope");
    const auto t = ctx->get_saved_variables();
    auto grads = once(
        qk_norm_kernels(t[0], t[1], t[2], t[3], t[4], t[5], t[6],
                        ctx->saved_data["eps"].toDouble(),
                        ctx->saved_data["half"].toBool(),
                        ctx->saved_data["one_plus"].toBool(), inside(g[0]),
                        inside(g[1])), "qk_norm_rope");
    grads.resize(10);
    return grads;
  }
};

std::tuple<Tensor, Tensor> qk_norm_rope(const Tensor& q, const Tensor& k,
                                        const Tensor& q_weight,
                                        const Tensor& k_weight,
                                        const Tensor& cos, const Tensor& sin,
                                        const Opt& positions, double eps,
                                        bool half, bool one_plus) {
  const int64_t D = q.dim() ? q.size(-1) : 0;
  TORCH_CHECK_VALUE(q.dim() == 4 && k.dim() == 4 && q.size(0) == k.size(0) &&
                    q.size(1) == k.size(1) && k.size(3) == D && D % 2 == 0 &&
                    D >= 2 && D <= 512 && q.size(2) > 0 && k.size(2) > 0,
                    "qk_norm_rope: q is [B, S, H, D], k [B, S, Hk, D], D even and "
                    "up to 512, got ", q.sizes(), " and ", k.sizes());
  TORCH_CHECK_VALUE(q_weight.dim() == 1 && q_weight.size(0) == D &&
                    k_weight.dim() == 1 && k_weight.size(0) == D,
                    "qk_norm_rope: weights are [D]");
  const auto type = q.scalar_type();
  TORCH_CHECK_VALUE(type == k.scalar_type() && type == q_weight.scalar_type() &&
                    type == k_weight.scalar_type(),
                    "qk_norm_rope: heads and weights of one type, got ", type,
                    ", ", k.scalar_type(), ", ", q_weight.scalar_type(), ", ",
                    k_weight.scalar_type());
  TORCH_CHECK_VALUE(type == at::kBFloat16 || type == at::kHalf ||
                    type == at::kFloat,
                    "qk_norm_rope: bf16, fp16 or fp32 on a GPU");
  TORCH_CHECK_VALUE(cos.dim() == 2 && cos.sizes() == sin.sizes() &&
                    cos.size(1) >= 1 && 2 * cos.size(1) <= D &&
                    cos.scalar_type() == at::kFloat &&
                    sin.scalar_type() == at::kFloat,
                    "qk_norm_rope: cos and sin are fp32 [positions, rotated / 2]");
  TORCH_CHECK_VALUE(!positions.has_value() ||
                    (positions->scalar_type() == at::kInt &&
                     positions->numel() == q.size(0) * q.size(1)),
                    "qk_norm_rope: positions are int32, one a token");
  TORCH_CHECK_VALUE(positions.has_value() || q.size(1) <= cos.size(0),
                    "qk_norm_rope: rows longer than the tables");
  bool here = true;
  for (const auto* t : {&k, &q_weight, &k_weight, &cos, &sin})
    here = here && t->device() == q.device();
  TORCH_CHECK_VALUE(here && (!positions.has_value() ||
                             positions->device() == q.device()),
                    "qk_norm_rope: tensors on different devices");
  TORCH_CHECK_VALUE(!cos.requires_grad() && !sin.requires_grad(),
                    "qk_norm_rope: cos and sin have no gradient");
  check_capture("qk_norm_rope", {&q, &k, &q_weight, &k_weight});
  Opt pos;
  if (positions.has_value()) pos = positions->contiguous();
  const auto c = cos.contiguous(), s = sin.contiguous();
  if (wants_grad(q) || wants_grad(k) || wants_grad(q_weight) ||
      wants_grad(k_weight)) {
    const auto y = QkNorm::apply(q, k, q_weight, k_weight, c, s, pos, eps, half,
                                 one_plus);
    return {y[0], y[1]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  const auto y = qk_norm_kernels(inside(q), inside(k), q_weight.contiguous(),
                                 k_weight.contiguous(), c, s, pos, eps, half,
                                 one_plus, c10::nullopt, c10::nullopt);
  return {y[0], y[1]};
}

// Logits as rows of two strides: [V], [N, V] or [B, S, V], unit stride inside.
struct LogitRows {
  int64_t rows = 1, V, inner = 1, outer_stride = 0, inner_stride = 0;
  int type;
  LogitRows(const at::Tensor& x, const at::Tensor& tokens) {
    const int64_t n = x.dim();
    TORCH_CHECK(x.is_cuda() && n >= 1 && n <= 3 &&
                (x.stride(n - 1) == 1 || x.size(n - 1) == 1 || x.numel() == 0),
                "token_logprobs: logits [.., V], unit stride inside");
    V = x.size(n - 1);
    if (n == 3) {
      rows = x.size(0) * x.size(1);
      inner = x.size(1);
      outer_stride = x.stride(0);
      inner_stride = x.stride(1);
    } else if (n == 2) {
      rows = inner = x.size(0);
      inner_stride = x.stride(0);
    }
    type = dtype_code(x);
    TORCH_CHECK(tokens.scalar_type() == at::kLong && tokens.is_contiguous() &&
                tokens.numel() == rows, "token_logprobs: tokens int64, one a row");
    TORCH_CHECK(V >= 1 && V < (1ll << 31) && rows * 256 < THREADS,
                "token_logprobs: size");
  }
};

variable_list logprobs_fwd(const Tensor& x, const Tensor& tokens, int64_t top,
                           int64_t ignore) {
  const OneDevice on("token_logprobs", x, tokens);
  const LogitRows r(x, tokens);
  const int parts = ds_logprobs_parts((int)r.rows, r.V, (int)top);
  TORCH_CHECK(top >= 0 && top <= 32 && top <= r.V && (top == 0 || parts <= 64),
              "token_logprobs: up to 32 of up to 500000 tokens");
  TORCH_CHECK(r.rows * (parts + 1) * 256 < THREADS, "token_logprobs: size");
  const auto f32 = x.options().dtype(at::kFloat);
  auto lp = at::empty(tokens.sizes(), f32), ent = at::empty(tokens.sizes(), f32);
  auto stat = at::empty({r.rows, 2}, f32);
  auto best = tokens.sizes().vec();
  best.push_back(top);
  auto top_lp = at::empty(best, f32), ids = at::empty(best, tokens.options());
  if (r.rows) {
    // the parts' sums, then on 8 bytes their lists
    const int64_t of_sums = (r.rows * parts * 3 + 1) / 2 * 2;
    auto work = at::empty({of_sums + r.rows * parts * 2 * top}, f32);
    float* sums = work.data_ptr<float>();
    const int e = ds_logprobs_fwd(
        x.data_ptr(), r.outer_stride, r.inner_stride, (int)r.inner, r.type,
        reinterpret_cast<const long long*>(tokens.data_ptr<int64_t>()),
        lp.data_ptr<float>(), ent.data_ptr<float>(), stat.data_ptr<float>(),
        top_lp.data_ptr<float>(),
        reinterpret_cast<long long*>(ids.data_ptr<int64_t>()), sums,
        sums + of_sums,
        (int)r.rows, r.V, parts, (int)top, ignore, cur_stream());
    TORCH_CHECK(e == 0, "token_logprobs: launch failed, hipError_t ", e);
  }
  return {lp, ent, stat, top_lp, ids};
}

at::Tensor logprobs_bwd(at::Tensor x, at::Tensor tokens, at::Tensor stat,
                        at::Tensor ent, Opt glp, Opt gent, int64_t ignore) {
  const OneDevice on("token_logprobs", x, tokens, stat, ent, glp, gent);
  const LogitRows r(x, tokens);
  for (const auto& g : {glp, gent})
    if (data(g))
      TORCH_CHECK(g->scalar_type() == at::kFloat && g->is_contiguous() &&
                  g->numel() == r.rows, "token_logprobs: gradients fp32, one a row");
  TORCH_CHECK(stat.numel() == 2 * r.rows && ent.numel() == r.rows,
              "token_logprobs: saved rows");
  auto dx = at::empty(x.sizes(), x.options());
  if (r.rows) {
    const int e = ds_logprobs_bwd(
        x.data_ptr(), r.outer_stride, r.inner_stride, (int)r.inner, r.type,
        reinterpret_cast<const long long*>(tokens.data_ptr<int64_t>()),
        stat.data_ptr<float>(), ent.data_ptr<float>(),
        static_cast<const float*>(data(glp)),
        static_cast<const float*>(data(gent)), dx.data_ptr(), (int)r.rows, r.V,
        ignore, cur_stream());
    TORCH_CHECK(e == 0, "token_logprobs: launch failed, hipError_t ", e);
  }
  return dx;
}

struct TokenLogprobs : torch::autograd::Function<TokenLogprobs> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits,
                               const Tensor& tokens, int64_t top,
                               int64_t ignore) {
    // up to three dimensions of any strides but one inside a row
    auto x = logits;
    if (x.dim() > 3) x = x.flatten(0, x.dim() - 3);
    if (x.size(-1) > 1 && x.stride(-1) != 1) x = x.contiguous();
    auto out = logprobs_fwd(x, tokens, top, ignore);
    ctx->save_for_backward({x, tokens, out[2], out[1]});
    ctx->saved_data["ignore"] = ignore;
    ctx->mark_non_differentiable({out[3], out[4]});
    ctx->set_materialize_grads(false);
    return {out[0], out[1], out[3], out[4]};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    check_single(g, "token_logprobs");
    variable_list grads(4);
    if (!g[0].defined() && !g[1].defined()) return grads;
    const auto t = ctx->get_saved_variables();
    for (int i = 0; i < 2; ++i)
      if (g[i].defined()) g[i] = g[i].to(at::kFloat).contiguous();
    auto shape = t[1].sizes().vec();
    shape.push_back(t[0].size(-1));
    auto dx = logprobs_bwd(t[0], t[1], t[2], t[3], g[0], g[1],
                           ctx->saved_data["ignore"].toInt());
    grads[0] = once({dx.view(shape)}, "token_logprobs")[0];
    return grads;
  }
};

std::tuple<Tensor, Tensor, Tensor, Tensor> token_logprobs(
    const Tensor& logits, const Tensor& tokens, int64_t top,
    int64_t ignore_index) {
  TORCH_CHECK_VALUE(logits.dim() >= 1 && logits.size(-1) >= 1 &&
                    logits.sizes().slice(0, logits.dim() - 1) == tokens.sizes(),
                    "token_logprobs: logits [.., V] and tokens [..], got ",
                    logits.sizes(), " and ", tokens.sizes());
  TORCH_CHECK_VALUE(tokens.scalar_type() == at::kInt ||
                    tokens.scalar_type() == at::kLong,
                    "token_logprobs: integer tokens, got ", tokens.scalar_type());
  const auto type = logits.scalar_type();
  TORCH_CHECK_VALUE(type == at::kBFloat16 || type == at::kHalf ||
                    type == at::kFloat,
                    "token_logprobs: floating logits, bf16, fp16 or fp32 on a "
                    "GPU, got ", type);
  const int64_t V = logits.size(-1);
  TORCH_CHECK_VALUE(top >= 0 && top <= 32 && top <= V &&
                    (top == 0 || V <= 500000),
                    "token_logprobs: up to 32 best of 500000 tokens at most, got ",
                    top, " of ", V);
  TORCH_CHECK_VALUE(logits.device() == tokens.device(),
                    "token_logprobs: tensors on different devices");
  check_capture("token_logprobs", {&logits});
  const auto y = TokenLogprobs::apply(
      logits, tokens.to(at::kLong).contiguous(), top, ignore_index);
  return {y[0], y[1], y[2], y[3]};
}

}  // namespace

void bind_packed(pybind11::module_& m) {
  namespace py = pybind11;
  m.def("packed_spans", &packed_spans,
        "the keys that each query sees, the queries that see each key");
  m.def("masked_attention", &masked_attention, "attention over packed rows",
        py::arg("q"), py::arg("k"), py::arg("v"), py::arg("spans"),
        py::arg("alibi_slopes"), py::arg("causal"), py::arg("scale"),
        py::arg("softcap"));
  m.def("paged_shaped", &paged_shaped,
        "attention of single tokens over the paged pool, scores shaped",
        py::arg("q"), py::arg("kpool"), py::arg("vpool"), py::arg("block_table"),
        py::arg("lens"), py::arg("splits"), py::arg("scale"), py::arg("softcap"),
        py::arg("alibi_slopes"));
  m.def("qk_norm_rope", &qk_norm_rope, "norms and rotation of queries and keys",
        py::arg("q"), py::arg("k"), py::arg("q_weight"), py::arg("k_weight"),
        py::arg("cos"), py::arg("sin"), py::arg("positions"), py::arg("eps"),
        py::arg("half"), py::arg("one_plus"));
  m.def("token_logprobs", &token_logprobs,
        "log probabilities, entropy and best tokens of rows of logits",
        py::arg("logits"), py::arg("tokens"), py::arg("top"),
        py::arg("ignore_index"));
}
