// Router with a balance loss (router_balance.cu): launch parameters and launchers.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace sepx {

struct RouterBalanceArgs {
  const void* x = nullptr;  // [T, E] router logits, unit column stride
  int64_t x_stride = 0;     // elements between rows
  int dtype = 0;            // 0 bf16, 1 fp16, 2 fp32
  int T = 0, E = 0, k = 0;
  bool renorm = true;
  const float* bias = nullptr;     // [E], shifts the selection scores only
  const uint8_t* valid = nullptr;  // [T], tokens in the statistics; null: all
  int* topk_e = nullptr;           // [T, k]
  float* topk_w = nullptr;         // [T, k]
  // per-block partial sums, [blocks][E] each, and [blocks]
  float* part_p = nullptr;
  int* part_c = nullptr;
  int* part_n = nullptr;
  int blocks = 0;
  double* part_l = nullptr;          // [E] each expert's part of the loss
  unsigned int* ticket = nullptr;    // [1], needs no value
  int* counts = nullptr;   // [E] tokens of the mask that chose each expert
  float* coef = nullptr;   // [E] d loss / d p of a token in the mask
  float* loss = nullptr;   // [1]
  // backward
  const float* dw = nullptr;     // [T, k], may be null
  const float* dloss = nullptr;  // [1], may be null
  void* dx = nullptr;            // [T, E] contiguous, of x's type
};

constexpr int kRouterMaxExperts = 512, kRouterMaxK = 32;
int router_balance_blocks(int T, int num_sms);
void router_balance_fwd(const RouterBalanceArgs& a, cudaStream_t st);
void router_balance_bwd(const RouterBalanceArgs& a, int num_sms, cudaStream_t st);

}  // namespace sepx
