// Python bindings of the vocabulary losses (vocab_loss.cu) and of the router with a balance
// loss (router_balance.cu).
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <atomic>
#include <cmath>
#include <string>

#include "router_balance.h"
#include "vocab_loss.h"

namespace {

// Numbers go into messages through std::to_string: the stream insertion of an integer
// crashes where the extension's C++ runtime differs from the interpreter's.

// The last of an entry point's checks, so that the others speak on any machine.
void need_cuda(const at::Tensor& t, const char* name) { TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor"); }

cudaStream_t cs() { return at::cuda::getCurrentCUDAStream().stream(); }
int sms() { return at::cuda::getCurrentDeviceProperties()->multiProcessorCount; }

int vocab_dtype(const at::Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return sepx::kVocabBf16;
    case at::kHalf: return sepx::kVocabF16;
    case at::kFloat: return sepx::kVocabF32;
    default: TORCH_CHECK(false, name, " must be bf16, fp16 or fp32, not ", t.scalar_type());
  }
}

void req_rows(const at::Tensor& t, const at::Tensor& z, const char* name) {
  TORCH_CHECK(t.device() == z.device(), name, " must be on the logits' device");
  TORCH_CHECK(t.dim() == 1 && t.size(0) == z.size(0), name, " must be [", std::to_string(z.size(0)), "]");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}
void req_f32_rows(const at::Tensor& t, const at::Tensor& z, const char* name) {
  req_rows(t, z, name);
  TORCH_CHECK(t.scalar_type() == at::kFloat, name, " must be fp32");
}
bool ids_are_64(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, name, " must be int32 or int64");
  return t.scalar_type() == at::kLong;
}

// Limits of the waits in the calls to come (test_stall).
std::atomic<int64_t> g_wait_ns{2000000000}, g_stall_row{-1};

// Makes the waits for a row run out after wait_ns in every call until test_stall(-1, 0).
void test_stall(int64_t row, int64_t wait_ns) {
  TORCH_CHECK(row >= -1 && row < 0x7fffffff && wait_ns >= 0 && wait_ns <= 2000000000, "a row and at most 2 s");
  g_stall_row = row;
  g_wait_ns = wait_ns > 0 ? wait_ns : 2000000000;
}

// Common part: logits, gradient buffer and temperature.
sepx::VocabLossArgs vocab_args(const at::Tensor& z, const c10::optional<at::Tensor>& grad, double tau) {
  TORCH_CHECK(z.dim() == 2, "logits must be [T, V]");
  TORCH_CHECK(z.size(1) >= 1 && z.size(1) <= 0x7fffff00, "logits must have a vocabulary of 1 to 2^31 - 256 columns");
  TORCH_CHECK(z.size(0) <= 0x7fffffff / 8, "too many rows");
  TORCH_CHECK(z.stride(1) == 1 || z.size(1) == 1, "logits must have unit stride along the vocabulary");
  TORCH_CHECK(std::isfinite(tau) && tau > 0, "temperature must be positive and finite");
  sepx::VocabLossArgs a;
  a.wait_ns = (uint64_t)g_wait_ns.load();
  a.stall_row = (int)g_stall_row.load();
  a.z = z.data_ptr();
  a.z_stride = z.stride(0);
  a.dtype = vocab_dtype(z, "logits");
  a.T = (int)z.size(0);
  a.V = (int)z.size(1);
  // in two parts, the second above 0: a logit of -infinity has to stay one in both products
  const double c2 = 1.4426950408889634 / tau;
  a.c2 = (float)c2;
  int exponent = 0;
  const double bits = std::frexp(c2, &exponent) * 4096;  // 2048 <= bits < 4096
  a.c2_hi = (float)std::ldexp(std::ceil(bits) - 1, exponent - 12);
  a.c2_lo = (float)(c2 - (double)a.c2_hi);
  // c2_lo is at least c2 2^-53: from 1e-20 on a normal number, which -inf times stays -inf.
  TORCH_CHECK(std::isfinite(c2) && a.c2 > 1e-20f && a.c2 < 1e30f, "temperature out of range");
  a.tau = (float)tau;
  a.tau64 = tau;
  if (grad.has_value()) {
    TORCH_CHECK(grad->device() == z.device() && grad->scalar_type() == z.scalar_type() && grad->sizes() == z.sizes(),
                "the gradient buffer must be like the logits");
    TORCH_CHECK((grad->stride(1) == 1 || grad->size(1) == 1) && (grad->stride(0) >= grad->size(1) || grad->size(0) < 2),
                "the gradient buffer must have unit stride along the vocabulary and rows apart");
    a.grad = grad->data_ptr();
    a.grad_stride = grad->stride(0);
  }
  return a;
}

void set_upstream(sepx::VocabLossArgs& a, const c10::optional<at::Tensor>& up, const at::Tensor& z) {
  if (!up.has_value()) return;
  TORCH_CHECK(up->device() == z.device() && up->numel() == 1 && up->scalar_type() == at::kFloat,
              "the gradient of the loss must be one fp32 on the logits' device");
  a.up = up->data_ptr<float>();
}

// Gradient of the logits, with rows at the same places in their 16 bytes as the logits' rows,
// so that both move in whole vectors: the logits' row stride (where it costs little memory)
// and the phase of their first row. Contiguous where the logits are.
bool shares_stride(const at::Tensor& z) {
  return z.dim() == 2 && z.stride(0) >= z.size(1) && z.stride(0) <= z.size(1) + z.size(1) / 64 + 64;
}
int64_t phase_of(const at::Tensor& z) { return (int64_t)(reinterpret_cast<uintptr_t>(z.data_ptr()) % 16) / z.element_size(); }
at::Tensor gradient_storage(const at::Tensor& z) {
  TORCH_CHECK(z.dim() == 2, "logits must be [T, V]");
  if (z.is_contiguous() && phase_of(z) == 0) return at::empty(z.sizes(), z.options());
  return at::empty({z.size(0) * (shares_stride(z) ? z.stride(0) : z.size(1)) + 16 / z.element_size()}, z.options());
}
at::Tensor gradient_view(const at::Tensor& flat, const at::Tensor& z) {
  if (flat.dim() == 2) return flat;
  return flat.as_strided({z.size(0), z.size(1)}, {shares_stride(z) ? z.stride(0) : z.size(1), 1},
                         flat.storage_offset() + phase_of(z));
}

// Scratch of a call in one allocation: records, partial sums, a ticket and a count.
at::Tensor set_scratch(sepx::VocabLossArgs& a, const at::Tensor& z, int64_t partial = 0) {
  const int64_t rec = (int64_t)a.T * sepx::kRowRecordBytes;
  const int64_t part = std::max<int64_t>(sepx::vocab_finish_blocks(a.T), partial) * 8;
  at::Tensor s = at::empty({rec + part + 16}, z.options().dtype(at::kByte));
  uint8_t* p = s.data_ptr<uint8_t>();
  a.records = p;
  a.partial = reinterpret_cast<double*>(p + rec);
  a.ticket = reinterpret_cast<unsigned int*>(p + rec + part);
  return s;
}

// num_valid >= 0: the rows in the loss, known on the host; negative: counted on the device,
// into the scratch.
void set_rows(sepx::VocabLossArgs& a, int op, int64_t num_valid) {
  if (num_valid >= 0) {
    a.host_scale = 1.f / (float)std::max<int64_t>(num_valid, 1);
  } else {
    int* count = reinterpret_cast<int*>(a.ticket + 1);
    a.count = count;
    sepx::vocab_count_rows(a, op, count, cs());
  }
}

// Returns the loss; the gradient (of the loss times `up`) goes to `grad`, which may be the
// logits themselves.
at::Tensor distill_loss(const at::Tensor& z, const at::Tensor& ids, const at::Tensor& teacher, double tau,
                        int64_t num_valid, const c10::optional<at::Tensor>& grad, const c10::optional<at::Tensor>& up) {
  auto a = vocab_args(z, grad, tau);
  TORCH_CHECK(ids.device() == z.device() && teacher.device() == z.device(),
              "teacher ids and logits must be on the logits' device");
  TORCH_CHECK(ids.dim() == 2 && ids.size(0) == z.size(0), "teacher_ids must be [", std::to_string(z.size(0)), ", K]");
  TORCH_CHECK(teacher.sizes() == ids.sizes(), "teacher_logits must have the shape of teacher_ids");
  TORCH_CHECK(ids.size(1) >= 1 && ids.size(1) <= sepx::kMaxTeacher, "a row has 1 to ", std::to_string(sepx::kMaxTeacher),
              " teacher entries, not ", std::to_string(ids.size(1)));
  TORCH_CHECK(ids.is_contiguous() && teacher.is_contiguous(), "teacher_ids and teacher_logits must be contiguous");
  TORCH_CHECK(teacher.scalar_type() == at::kFloat, "teacher_logits must be fp32");
  a.ids64 = ids_are_64(ids, "teacher_ids");
  need_cuda(z, "logits");
  const c10::cuda::CUDAGuard guard(z.device());
  a.ids = ids.data_ptr();
  a.teacher = teacher.data_ptr<float>();
  a.K = (int)ids.size(1);
  set_upstream(a, up, z);
  const auto f32 = z.options().dtype(at::kFloat);
  at::Tensor loss = at::empty({}, f32);
  const at::Tensor scratch = set_scratch(a, z);
  set_rows(a, sepx::kOpDistill, num_valid);
  a.loss = loss.data_ptr<float>();
  sepx::vocab_loss(a, sepx::kOpDistill, sms(), cs());
  return loss;
}

// Returns (loss, logp [T], kl [T]).
std::vector<at::Tensor> policy_loss(const at::Tensor& z, const at::Tensor& actions, const at::Tensor& old_logp,
                                    const at::Tensor& advantages, const c10::optional<at::Tensor>& ref_logp,
                                    double clip_low, double clip_high, double kl_coef, double tau, int64_t num_valid,
                                    const c10::optional<at::Tensor>& grad, const c10::optional<at::Tensor>& up) {
  auto a = vocab_args(z, grad, tau);
  req_rows(actions, z, "actions");
  req_f32_rows(old_logp, z, "old_logp");
  req_f32_rows(advantages, z, "advantages");
  if (ref_logp.has_value()) req_f32_rows(*ref_logp, z, "ref_logp");
  TORCH_CHECK(clip_low >= 0 && clip_low <= 1 && clip_high >= 0, "clip_low must be in [0, 1], clip_high >= 0");
  TORCH_CHECK(std::isfinite(kl_coef) && kl_coef >= 0, "kl_coef must be finite and >= 0");
  TORCH_CHECK(kl_coef == 0 || ref_logp.has_value(), "a KL term needs ref_logp");
  a.ids64 = ids_are_64(actions, "actions");
  need_cuda(z, "logits");
  const c10::cuda::CUDAGuard guard(z.device());
  a.labels = actions.data_ptr();
  a.old_logp = old_logp.data_ptr<float>();
  a.adv = advantages.data_ptr<float>();
  a.ref_logp = ref_logp.has_value() ? ref_logp->data_ptr<float>() : nullptr;
  a.clip_low = (float)clip_low;
  a.clip_high = (float)clip_high;
  a.kl_coef = (float)kl_coef;
  set_upstream(a, up, z);
  const auto f32 = z.options().dtype(at::kFloat);
  at::Tensor loss = at::empty({}, f32), logp = at::empty({a.T}, f32), kl = at::empty({a.T}, f32);
  const at::Tensor scratch = set_scratch(a, z);
  set_rows(a, sepx::kOpPolicy, num_valid);
  a.loss = loss.data_ptr<float>();
  a.logp = logp.data_ptr<float>();
  a.kl = kl.data_ptr<float>();
  sepx::vocab_loss(a, sepx::kOpPolicy, sms(), cs());
  return {loss, logp, kl};
}

// Log-probability [T] of each row's label.
at::Tensor token_logp(const at::Tensor& z, const at::Tensor& labels, double tau) {
  auto a = vocab_args(z, c10::nullopt, tau);
  req_rows(labels, z, "labels");
  a.ids64 = ids_are_64(labels, "labels");
  need_cuda(z, "logits");
  const c10::cuda::CUDAGuard guard(z.device());
  a.labels = labels.data_ptr();
  at::Tensor logp = at::empty({a.T}, z.options().dtype(at::kFloat));
  a.logp = logp.data_ptr<float>();
  const at::Tensor scratch = set_scratch(a, z);
  sepx::vocab_loss(a, sepx::kOpLogp, sms(), cs());
  return logp;
}

void set_offsets(sepx::VocabLossArgs& a, const at::Tensor& offsets, const at::Tensor& z) {
  TORCH_CHECK(offsets.device() == z.device() && offsets.scalar_type() == at::kInt && offsets.is_contiguous() &&
                  offsets.dim() == 1 && offsets.size(0) % 2 == 1,
              "seq_offsets must be a contiguous int32 vector of 2 * pairs + 1 entries on the logits' device");
  a.offsets = offsets.data_ptr<int>();
  a.num_seq = (int)offsets.size(0) - 1;
}

// Returns (loss, rewards [2 * pairs], logp [T], rows [5, T]: the rows' lse as T pairs, then
// d loss / d logp, then scratch, then the sums without the labels' terms). With `grad` (may be the logits), d logp / d logits of each
// row is written there.
std::vector<at::Tensor> preference_fwd(const at::Tensor& z, const at::Tensor& labels, const at::Tensor& offsets,
                                       const at::Tensor& ref_logp, double beta, double eps,
                                       const c10::optional<at::Tensor>& grad) {
  auto a = vocab_args(z, grad, 1.0);
  req_rows(labels, z, "labels");
  req_f32_rows(ref_logp, z, "ref_logp");
  set_offsets(a, offsets, z);
  TORCH_CHECK(std::isfinite(beta) && beta > 0, "beta must be positive and finite");
  TORCH_CHECK(eps >= 0 && eps < 0.5, "label_smoothing must be in [0, 0.5)");
  a.ids64 = ids_are_64(labels, "labels");
  need_cuda(z, "logits");
  const c10::cuda::CUDAGuard guard(z.device());
  a.labels = labels.data_ptr();
  sepx::PreferenceArgs q;
  q.pairs = a.num_seq / 2;
  const auto f32 = z.options().dtype(at::kFloat);
  at::Tensor loss = at::empty({}, f32), rewards = at::empty({2 * (int64_t)q.pairs}, f32);
  at::Tensor logp = at::empty({a.T}, f32), rows = at::empty({5, a.T}, f32);
  const at::Tensor scratch = set_scratch(a, z, q.pairs);
  a.logp = logp.data_ptr<float>();
  a.lse = rows.data_ptr<float>();
  a.row_coef = a.lse + 2 * (int64_t)a.T;
  a.ratio = a.lse + 3 * (int64_t)a.T;
  a.rest = a.lse + 4 * (int64_t)a.T;
  a.ref_logp = ref_logp.data_ptr<float>();
  if (a.T > 0) sepx::vocab_loss(a, sepx::kOpLogp, sms(), cs());
  else if (q.pairs > 0) C10_CUDA_CHECK(cudaMemsetAsync(a.ticket, 0, sizeof(int), cs()));
  q.ratio = a.ratio;
  q.labels = a.labels;
  q.ids64 = a.ids64;
  q.offsets = a.offsets;
  q.T = a.T;
  q.beta = (float)beta;
  q.eps = (float)eps;
  q.rewards = rewards.data_ptr<float>();
  q.loss = loss.data_ptr<float>();
  q.row_coef = a.row_coef;
  q.partial = a.partial;
  q.ticket = a.ticket;
  sepx::preference_pairs(q, cs());
  return {loss, rewards, logp, rows};
}

// d (up * loss) / d logits from the forward's rows.
at::Tensor preference_grad(const at::Tensor& z, const at::Tensor& labels, const at::Tensor& offsets,
                           const at::Tensor& rows, const at::Tensor& up) {
  const at::Tensor grad = gradient_view(gradient_storage(z), z);
  auto a = vocab_args(z, grad, 1.0);
  req_rows(labels, z, "labels");
  TORCH_CHECK(rows.device() == z.device() && rows.scalar_type() == at::kFloat && rows.is_contiguous() &&
                  rows.numel() == 5 * z.size(0),
              "rows must be the forward's");
  set_offsets(a, offsets, z);
  a.ids64 = ids_are_64(labels, "labels");
  need_cuda(z, "logits");
  const c10::cuda::CUDAGuard guard(z.device());
  a.labels = labels.data_ptr();
  a.lse = rows.data_ptr<float>();
  a.rest = a.lse + 4 * (int64_t)a.T;
  set_upstream(a, up, z);
  sepx::preference_grad(a, a.lse + 2 * (int64_t)a.T, cs());
  return grad;
}

// grad *= up in place (nothing is read where up is 1).
void scale_grad(const at::Tensor& grad, const at::Tensor& up) {
  TORCH_CHECK(grad.is_contiguous(), "grad must be contiguous");
  TORCH_CHECK(up.device() == grad.device() && up.numel() == 1 && up.scalar_type() == at::kFloat,
              "the gradient of the loss must be one fp32 on the same device");
  need_cuda(grad, "grad");
  const c10::cuda::CUDAGuard guard(grad.device());
  TORCH_CHECK(reinterpret_cast<uintptr_t>(grad.data_ptr()) % 16 == 0, "grad must be 16-byte aligned");
  sepx::vocab_scale_grad(grad.data_ptr(), vocab_dtype(grad, "grad"), grad.numel(), up.data_ptr<float>(), sms(), cs());
}

sepx::RouterBalanceArgs router_args(const at::Tensor& x, int64_t k, bool renorm, const c10::optional<at::Tensor>& valid) {
  TORCH_CHECK(x.dim() == 2 && x.size(0) <= 0x7fffffff / 32, "router logits must be [T, E]");
  const int64_t E = x.size(1);
  TORCH_CHECK(E >= 1 && E <= sepx::kRouterMaxExperts, "1 to ", std::to_string(sepx::kRouterMaxExperts),
              " experts, not ", std::to_string(E));
  TORCH_CHECK(k >= 1 && k <= sepx::kRouterMaxK && k <= E, "k must be 1 to min(",
              std::to_string(sepx::kRouterMaxK), ", experts), not ", std::to_string(k));
  TORCH_CHECK(x.stride(1) == 1 || E == 1, "router logits must have unit stride along the experts");
  sepx::RouterBalanceArgs a;
  a.x = x.data_ptr();
  a.x_stride = x.stride(0);
  a.dtype = vocab_dtype(x, "router logits");
  a.T = (int)x.size(0);
  a.E = (int)E;
  a.k = (int)k;
  a.renorm = renorm;
  if (valid.has_value()) {
    TORCH_CHECK(valid->device() == x.device() && valid->scalar_type() == at::kBool && valid->is_contiguous() &&
                    valid->dim() == 1 && valid->size(0) == x.size(0),
                "valid must be a contiguous bool vector, one entry per token, on the logits' device");
    a.valid = reinterpret_cast<const uint8_t*>(valid->data_ptr<bool>());
  }
  return a;
}

// Returns (topk_w [T, k], topk_e [T, k] int32, loss, counts [E] int32, coef [E]).
std::vector<at::Tensor> router_balance_fwd(const at::Tensor& x, int64_t k, bool renorm,
                                           const c10::optional<at::Tensor>& bias,
                                           const c10::optional<at::Tensor>& valid) {
  auto a = router_args(x, k, renorm, valid);
  if (bias.has_value()) {
    TORCH_CHECK(bias->device() == x.device() && bias->scalar_type() == at::kFloat && bias->is_contiguous() &&
                    bias->dim() == 1 && bias->size(0) == x.size(1),
                "bias must be a contiguous fp32 vector, one entry per expert, on the logits' device");
    a.bias = bias->data_ptr<float>();
  }
  need_cuda(x, "router logits");
  const c10::cuda::CUDAGuard guard(x.device());
  const auto f32 = x.options().dtype(at::kFloat), i32 = x.options().dtype(at::kInt);
  a.blocks = sepx::router_balance_blocks(a.T, sms());
  at::Tensor w = at::empty({a.T, a.k}, f32), e = at::empty({a.T, a.k}, i32);
  at::Tensor loss = at::empty({}, f32), counts = at::empty({a.E}, i32), coef = at::empty({a.E}, f32);
  // scratch: parts of the loss, of the column sums and counts of each block, and a ticket
  at::Tensor part = at::empty({2 * (int64_t)a.E + a.blocks * (2 * (int64_t)a.E + 1) + 1}, f32);
  a.topk_w = w.data_ptr<float>();
  a.topk_e = e.data_ptr<int>();
  a.loss = loss.data_ptr<float>();
  a.counts = counts.data_ptr<int>();
  a.coef = coef.data_ptr<float>();
  a.part_l = reinterpret_cast<double*>(part.data_ptr<float>());
  a.part_p = part.data_ptr<float>() + 2 * a.E;
  a.part_c = reinterpret_cast<int*>(a.part_p + (int64_t)a.blocks * a.E);
  a.part_n = a.part_c + (int64_t)a.blocks * a.E;
  a.ticket = reinterpret_cast<unsigned int*>(a.part_n + a.blocks);
  sepx::router_balance_fwd(a, cs());
  return {w, e, loss, counts, coef};
}

// d logits from the gradients of topk_w and of the loss (either may be absent).
at::Tensor router_balance_bwd(const at::Tensor& x, const at::Tensor& topk_e, const at::Tensor& coef, bool renorm,
                              const c10::optional<at::Tensor>& valid, const c10::optional<at::Tensor>& dw,
                              const c10::optional<at::Tensor>& dloss) {
  TORCH_CHECK(topk_e.dim() == 2 && topk_e.scalar_type() == at::kInt && topk_e.is_contiguous() &&
                  topk_e.device() == x.device() && topk_e.size(0) == x.size(0),
              "topk_e must be the forward's");
  auto a = router_args(x, topk_e.size(1), renorm, valid);
  TORCH_CHECK(coef.device() == x.device() && coef.scalar_type() == at::kFloat && coef.is_contiguous() &&
                  coef.numel() == x.size(1),
              "coef must be the forward's");
  if (dw.has_value()) {
    TORCH_CHECK(dw->device() == x.device() && dw->scalar_type() == at::kFloat && dw->is_contiguous() &&
                    dw->sizes() == topk_e.sizes(),
                "dw must be a contiguous fp32 tensor of topk_w's shape");
    a.dw = dw->data_ptr<float>();
  }
  if (dloss.has_value()) {
    TORCH_CHECK(dloss->device() == x.device() && dloss->scalar_type() == at::kFloat && dloss->numel() == 1,
                "the gradient of the loss must be one fp32 on the logits' device");
    a.dloss = dloss->data_ptr<float>();
  }
  need_cuda(x, "router logits");
  const c10::cuda::CUDAGuard guard(x.device());
  at::Tensor dx = at::empty(x.sizes(), x.options());
  a.topk_e = topk_e.data_ptr<int>();
  a.coef = coef.data_ptr<float>();
  a.dx = dx.data_ptr();
  sepx::router_balance_bwd(a, sms(), cs());
  return dx;
}

// ------------------------------------------------------------------------------------
// Autograd. The nodes are C++ ones: a Python node would take the interpreter lock on the
// engine's thread, which costs as much as a small batch's kernels.
// ------------------------------------------------------------------------------------
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Also a forward-mode tangent takes the way through autograd, which refuses it: the kernels
// alone would drop it.
bool wants_grad(const at::Tensor& z) {
  return (at::GradMode::is_enabled() && z.requires_grad()) || z._fw_grad(/*level=*/0).defined();
}

// Gradients here are not themselves differentiable: whoever tries, through the logits that
// they depend on, gets an error.
at::Tensor once(AutogradContext* ctx, const at::Tensor& g) {
  if (!at::GradMode::is_enabled()) return g;
  auto error = std::make_shared<torch::autograd::DelayedError>("this loss can only be differentiated once", 2);
  return (*error)({g, ctx->get_saved_variables()[0]})[0];
}

// A loss whose forward has formed the gradient in its pass over the logits. It is handed out
// once, scaled in place (not touched where the upstream gradient is 1). A second backward
// through the same graph, and fp16 logits, whose unscaled gradient could leave the type's
// range, compute it from the logits. So does a backward that is captured apart from its forward:
// every replay would scale the kept gradient again.
bool formed_in_forward(const at::Tensor& z) { return z.scalar_type() != at::kHalf; }
// The capture that the current stream is in, 0 for none.
int64_t capture_id() {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  C10_CUDA_CHECK(cudaStreamGetCaptureInfo(cs(), &status, &id));
  return status == cudaStreamCaptureStatusActive ? (int64_t)id : 0;
}
// Keeps a buffer for the gradient and returns its view.
at::Tensor keep_gradient(AutogradContext* ctx, const at::Tensor& z) {
  if (z.is_cuda()) {  // others are refused with the checks of the call
    const c10::cuda::CUDAGuard guard(z.device());
    ctx->saved_data["capture"] = capture_id();
  }
  const at::Tensor flat = gradient_storage(z), g = gradient_view(flat, z);
  ctx->saved_data["grad"] = flat;
  if (flat.dim() != 2)
    ctx->saved_data["at"] = std::vector<int64_t>{g.size(0), g.size(1), g.stride(0), g.storage_offset()};
  return g;
}
at::Tensor take_formed(AutogradContext* ctx, const at::Tensor& up) {
  auto& kept = ctx->saved_data["grad"];
  if (!kept.isTensor() || ctx->saved_data["capture"].toInt() != capture_id()) return {};
  at::Tensor flat = kept.toTensor();
  kept = c10::IValue();
  scale_grad(flat, up);  // with what lies between the rows, which nothing reads
  if (flat.dim() == 2) return flat;
  const auto at = ctx->saved_data["at"].toIntVector();
  return flat.as_strided({at[0], at[1]}, {at[2], 1}, at[3]);
}

struct DistillFn : torch::autograd::Function<DistillFn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& z, const at::Tensor& ids, const at::Tensor& teacher,
                            double tau, int64_t num_valid) {
    c10::optional<at::Tensor> grad;
    if (formed_in_forward(z)) grad = keep_gradient(ctx, z);
    at::Tensor loss = distill_loss(z, ids, teacher, tau, num_valid, grad, c10::nullopt);
    ctx->save_for_backward({z, ids, teacher});
    ctx->saved_data["tau"] = tau;
    ctx->saved_data["num_valid"] = num_valid;
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list up) {
    at::Tensor g = take_formed(ctx, up[0]);
    if (!g.defined()) {
      const auto s = ctx->get_saved_variables();
      g = gradient_view(gradient_storage(s[0]), s[0]);
      distill_loss(s[0], s[1], s[2], ctx->saved_data["tau"].toDouble(), ctx->saved_data["num_valid"].toInt(), g, up[0]);
    }
    return {once(ctx, g), {}, {}, {}, {}};
  }
};

at::Tensor topk_distill(const at::Tensor& z, const at::Tensor& ids, const at::Tensor& teacher, double tau,
                        int64_t num_valid) {
  if (!wants_grad(z)) return distill_loss(z, ids, teacher, tau, num_valid, c10::nullopt, c10::nullopt);
  return DistillFn::apply(z, ids, teacher, tau, num_valid);
}

struct PolicyFn : torch::autograd::Function<PolicyFn> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& z, const at::Tensor& actions,
                               const at::Tensor& old_logp, const at::Tensor& advantages,
                               const c10::optional<at::Tensor>& ref_logp, double clip_low, double clip_high,
                               double kl_coef, double tau, int64_t num_valid) {
    c10::optional<at::Tensor> grad;
    if (formed_in_forward(z)) grad = keep_gradient(ctx, z);
    auto out = policy_loss(z, actions, old_logp, advantages, ref_logp, clip_low, clip_high, kl_coef, tau, num_valid,
                           grad, c10::nullopt);
    ctx->save_for_backward({z, actions, old_logp, advantages, ref_logp.value_or(at::Tensor())});
    ctx->saved_data["cfg"] = std::vector<double>{clip_low, clip_high, kl_coef, tau};
    ctx->saved_data["num_valid"] = num_valid;
    ctx->mark_non_differentiable({out[1], out[2]});
    ctx->set_materialize_grads(false);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list up) {
    at::Tensor g;
    if (up[0].defined()) {
      g = take_formed(ctx, up[0]);
      if (!g.defined()) {
        const auto s = ctx->get_saved_variables();
        const auto c = ctx->saved_data["cfg"].toDoubleVector();
        g = gradient_view(gradient_storage(s[0]), s[0]);
        policy_loss(s[0], s[1], s[2], s[3], s[4].defined() ? c10::optional<at::Tensor>(s[4]) : c10::nullopt, c[0], c[1],
                    c[2], c[3], ctx->saved_data["num_valid"].toInt(), g, up[0]);
      }
      g = once(ctx, g);
    }
    return {g, {}, {}, {}, {}, {}, {}, {}, {}, {}};
  }
};

std::vector<at::Tensor> clipped_policy(const at::Tensor& z, const at::Tensor& actions, const at::Tensor& old_logp,
                                       const at::Tensor& advantages, const c10::optional<at::Tensor>& ref_logp,
                                       double clip_low, double clip_high, double kl_coef, double tau,
                                       int64_t num_valid) {
  if (!wants_grad(z))
    return policy_loss(z, actions, old_logp, advantages, ref_logp, clip_low, clip_high, kl_coef, tau, num_valid,
                       c10::nullopt, c10::nullopt);
  return PolicyFn::apply(z, actions, old_logp, advantages, ref_logp, clip_low, clip_high, kl_coef, tau, num_valid);
}

struct PreferenceFn : torch::autograd::Function<PreferenceFn> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& z, const at::Tensor& labels,
                               const at::Tensor& offsets, const at::Tensor& ref_logp, double beta, double eps) {
    auto out = preference_fwd(z, labels, offsets, ref_logp, beta, eps, c10::nullopt);
    ctx->save_for_backward({z, labels, offsets, out[3]});
    out.resize(3);
    ctx->mark_non_differentiable({out[1], out[2]});
    ctx->set_materialize_grads(false);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list up) {
    at::Tensor g;
    if (up[0].defined()) {
      const auto s = ctx->get_saved_variables();
      g = once(ctx, preference_grad(s[0], s[1], s[2], s[3], up[0]));
    }
    return {g, {}, {}, {}, {}, {}};
  }
};

// Returns (loss, rewards, logp).
std::vector<at::Tensor> preference(const at::Tensor& z, const at::Tensor& labels, const at::Tensor& offsets,
                                   const at::Tensor& ref_logp, double beta, double eps) {
  if (wants_grad(z)) return PreferenceFn::apply(z, labels, offsets, ref_logp, beta, eps);
  auto out = preference_fwd(z, labels, offsets, ref_logp, beta, eps, c10::nullopt);
  out.resize(3);
  return out;
}

struct RouterBalanceFn : torch::autograd::Function<RouterBalanceFn> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, int64_t k, bool renorm,
                               const c10::optional<at::Tensor>& bias, const c10::optional<at::Tensor>& valid) {
    auto out = router_balance_fwd(x, k, renorm, bias, valid);
    ctx->save_for_backward({x, out[1], out[4], valid.value_or(at::Tensor())});
    ctx->saved_data["renorm"] = renorm;
    out.resize(4);
    ctx->mark_non_differentiable({out[1], out[3]});
    ctx->set_materialize_grads(false);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list up) {
    at::Tensor g;
    if (up[0].defined() || up[2].defined()) {
      const auto s = ctx->get_saved_variables();
      auto opt = [](const at::Tensor& t) { return t.defined() ? c10::optional<at::Tensor>(t) : c10::nullopt; };
      g = once(ctx, router_balance_bwd(s[0], s[1], s[2], ctx->saved_data["renorm"].toBool(), opt(s[3]),
                                  opt(up[0].defined() ? up[0].contiguous() : up[0]), opt(up[2])));
    }
    return {g, {}, {}, {}, {}};
  }
};

// Returns (topk_w, topk_e, loss, counts).
std::vector<at::Tensor> router_balanced(const at::Tensor& x, int64_t k, bool renorm,
                                        const c10::optional<at::Tensor>& bias,
                                        const c10::optional<at::Tensor>& valid) {
  if (wants_grad(x)) return RouterBalanceFn::apply(x, k, renorm, bias, valid);
  auto out = router_balance_fwd(x, k, renorm, bias, valid);
  out.resize(4);
  return out;
}

}  // namespace

void register_losses(pybind11::module& m) {
  m.def("topk_distill", &topk_distill);
  m.def("clipped_policy", &clipped_policy);
  m.def("preference", &preference);
  m.def("router_balanced", &router_balanced);
  m.def("token_logp", &token_logp);
  // without autograd; the gradient may overwrite the logits
  m.def("distill_loss", &distill_loss);
  m.def("policy_loss", &policy_loss);
  m.def("preference_fwd", &preference_fwd);
  m.def("scale_grad", &scale_grad);
  m.def("test_stall", &test_stall, "tests: the waits for this row of the vocabulary losses run out");
}
