// Losses over a vocabulary's logits and the balanced router: launch parameters and
// launchers (vocab_loss.cu, router_balance.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace sepx {

enum VocabDtype : int { kVocabBf16 = 0, kVocabF16 = 1, kVocabF32 = 2 };
enum VocabOp : int {
  kOpDistill = 0,  // soft targets: a teacher's top logits
  kOpPolicy = 1,   // one chosen token per row, clipped ratio loss with a KL term
  kOpLogp = 2,     // one token per row: its log-probability (and the unit gradient)
};

constexpr int kMaxTeacher = 1024;  // teacher entries per row

struct VocabLossArgs {
  const void* z = nullptr;  // [T, V] logits, unit column stride
  int64_t z_stride = 0;     // elements between rows
  void* grad = nullptr;     // [T, V] gradient, may be z; null: loss only
  int64_t grad_stride = 0;
  int dtype = kVocabBf16;
  int T = 0, V = 0;
  float c2 = 0.f, c2_hi = 0.f, c2_lo = 0.f;  // log2(e) / temperature; its first 12 bits and the rest
  float tau = 1.f;           // temperature, and unrounded
  double tau64 = 1.0;
  float host_scale = 1.f;    // 1 / rows in the loss, when the host knows it ...
  const int* count = nullptr;  // ... else the number of rows, on the device
  const float* up = nullptr;   // optional gradient of the loss, on the device
  // kOpDistill
  const void* ids = nullptr;  // [T, K] int32 / int64; negative: no entry
  const float* teacher = nullptr;  // [T, K] logits
  int K = 0;
  // kOpPolicy / kOpLogp
  const void* labels = nullptr;  // [T] int32 / int64; negative: row not in the loss
  bool ids64 = false;            // ids / labels are int64
  const float* old_logp = nullptr;
  const float* adv = nullptr;
  const float* ref_logp = nullptr;  // may be null (no KL term)
  float clip_low = 0.f, clip_high = 0.f, kl_coef = 0.f;
  const int* offsets = nullptr;  // kOpLogp: rows outside [offsets[0], offsets[num_seq]) are not in the loss
  int num_seq = 0;
  // How long a wait between warps or blocks may last, and a row (-1: none) that is never
  // announced to those who wait for it: a test makes the waits run out.
  uint64_t wait_ns = 2000000000;
  int stall_row = -1;
  // scratch
  void* records = nullptr;     // [T] records of kRowRecordBytes each
  double* partial = nullptr;   // [vocab_finish_blocks(T)]
  unsigned int* ticket = nullptr;  // [1], needs no value
  // outputs, fp32
  float* loss = nullptr;  // [1], kOpDistill / kOpPolicy: the mean over rows
  float* logp = nullptr;  // [T], kOpPolicy / kOpLogp
  float* kl = nullptr;    // [T], kOpPolicy
  float* ratio = nullptr;  // [T], kOpLogp: logp - ref_logp, 0 for rows not in the loss (optional)
  float* row_coef = nullptr;  // [T], kOpLogp with ratio: set to 0
  float* lse = nullptr;    // [T, 2], kOpLogp: a reference m of the row and its sum of 2^((z - m) c2) (optional) ...
  float* rest = nullptr;   // [T], with lse: the sum without the label's term
};
constexpr int kRowRecordBytes = 32;
int vocab_finish_blocks(int T);

// *count = rows in the loss: with a label >= 0 (labels [T]), or with a teacher entry (ids /
// teacher [T, K]).
void vocab_count_rows(const VocabLossArgs& a, int op, int* count, cudaStream_t st);
void vocab_loss(const VocabLossArgs& a, int op, int num_sms, cudaStream_t st);
// grad *= *up, in place; nothing is touched where *up is 1.
void vocab_scale_grad(void* grad, int dtype, int64_t n, const float* up, int num_sms, cudaStream_t st);

struct PreferenceArgs {
  const float* ratio = nullptr;  // [T] logp - ref_logp, 0 for rows not in the loss
  const void* labels = nullptr;  // [T]
  bool ids64 = false;
  const int* offsets = nullptr;  // [2 * pairs + 1]
  int T = 0, pairs = 0;
  float beta = 0.f, eps = 0.f;
  float* rewards = nullptr;    // [2 * pairs]
  float* loss = nullptr;       // [1], the mean over pairs
  float* row_coef = nullptr;   // [T] d loss / d logp; written for the pairs' rows with a label
  double* partial = nullptr;   // [pairs] scratch
  unsigned int* ticket = nullptr;  // [1], zero before the call
};
void preference_pairs(const PreferenceArgs& a, cudaStream_t st);
// grad[t] = up * row_coef[t] * (onehot(labels[t]) - softmax(z[t])), zeros where row_coef is 0.
void preference_grad(const VocabLossArgs& a, const float* row_coef, cudaStream_t st);

}  // namespace sepx
