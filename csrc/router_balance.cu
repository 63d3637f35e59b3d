// Router with a balance loss:
//   p = softmax(x) per token, the k largest scores (p, or p + bias), w = p there
//   (renormalised to sum 1), counts c_e of the tokens in the mask (N of them) that chose e,
//   loss = E sum_e f_e P_e   with f_e = c_e / (k N) and P_e = the mean of p_e over the mask
//   d loss / d p_te = E c_e / (k N^2) for tokens in the mask (counts are constants)
//   dx_te = p_te (g_te - sum_j p_tj g_tj), g = the gradient of p from w and from the loss.
// One warp per token. A warp keeps its lanes' column sums of p in registers over its
// tokens; blocks write partial sums and a second kernel adds them in a fixed order, so the
// loss has the same bits on every run. The backward recomputes p from the logits instead of
// reading it back: T x E fp32 probabilities are never stored.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <stdexcept>
#include <string>

#include "kernels.h"
#include "router_balance.h"

namespace sepx {
namespace {

constexpr int kWarps = 8;

void check_launch(const char* what) {
  note_launch();
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) throw std::runtime_error(std::string(what) + ": " + cudaGetErrorString(e));
}

__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(float v) { return v; }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16(v); }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half(v); }
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Order of floats as unsigned numbers (NaN above everything, -0 equal to +0); 0 is below
// every value and marks what is taken or outside the row.
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);
  const uint32_t k = u ^ ((u & 0x80000000u) ? 0xffffffffu : 0x80000000u);
  return k ? k : 1u;
}

// softmax of one row: lane l holds experts l, l + 32, ...
template <typename T, int EPL>
__device__ __forceinline__ void row_softmax(const T* row, int E, int lane, float (&l)[EPL], float (&p)[EPL], float* mx_out,
                                            float* inv_out) {
  float mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const int e = i * 32 + lane;
    l[i] = e < E ? to_f(row[e]) : -INFINITY;
    mx = fmaxf(mx, l[i]);
  }
  mx = warp_max(mx);
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    p[i] = i * 32 + lane < E ? __expf(l[i] - mx) : 0.f;
    s += p[i];
  }
  const float inv = 1.f / warp_sum(s);
#pragma unroll
  for (int i = 0; i < EPL; ++i) p[i] *= inv;
  *mx_out = mx;
  *inv_out = inv;
}

template <typename T, int EPL>
__global__ void __launch_bounds__(kWarps * 32) router_balance_fwd_kernel(const RouterBalanceArgs a) {
  __shared__ int s_cnt[EPL * 32];
  __shared__ float s_p[kWarps][EPL * 32];
  __shared__ int s_n;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int e = threadIdx.x; e < EPL * 32; e += blockDim.x) s_cnt[e] = 0;
  if (threadIdx.x == 0) s_n = 0;
  __syncthreads();
  float acc[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i) acc[i] = 0.f;
  int n = 0;
  for (int t = blockIdx.x * kWarps + warp; t < a.T; t += gridDim.x * kWarps) {
    float l[EPL], p[EPL], mx, inv;
    row_softmax<T, EPL>(reinterpret_cast<const T*>(a.x) + (int64_t)t * a.x_stride, a.E, lane, l, p, &mx, &inv);
    const bool on = !a.valid || a.valid[t];
    if (on) {
      ++n;
#pragma unroll
      for (int i = 0; i < EPL; ++i) acc[i] += p[i];
    }
    // p grows with the logit, so without a bias the logits themselves are compared: equal
    // logits are equal scores, and the lowest index wins
    uint32_t key[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const int e = i * 32 + lane;
      key[i] = e < a.E ? order_key(a.bias ? p[i] + a.bias[e] : l[i]) : 0u;
    }
    int my_e = 0;
    float my_p = 0.f, S = 0.f;
    for (int j = 0; j < a.k; ++j) {
      uint32_t best = 0;
#pragma unroll
      for (int i = 0; i < EPL; ++i) best = max(best, key[i]);
      best = __reduce_max_sync(0xffffffffu, best);
      int be = 0x7fffffff;
#pragma unroll
      for (int i = EPL - 1; i >= 0; --i)
        if (key[i] == best) be = i * 32 + lane;
      be = __reduce_min_sync(0xffffffffu, be);
      float pw = 0.f;
#pragma unroll
      for (int i = 0; i < EPL; ++i)
        if (i * 32 + lane == be) {
          pw = p[i];
          key[i] = 0u;
        }
      pw = __shfl_sync(0xffffffffu, pw, be & 31);
      S += pw;
      if (lane == j) {
        my_e = be;
        my_p = pw;
      }
    }
    if (lane < a.k) {
      a.topk_e[(int64_t)t * a.k + lane] = my_e;
      a.topk_w[(int64_t)t * a.k + lane] = a.renorm ? my_p / S : my_p;
      if (on) atomicAdd(&s_cnt[my_e], 1);
    }
  }
#pragma unroll
  for (int i = 0; i < EPL; ++i) s_p[warp][i * 32 + lane] = acc[i];
  if (lane == 0 && n) atomicAdd(&s_n, n);
  __syncthreads();
  for (int e = threadIdx.x; e < a.E; e += blockDim.x) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) s += s_p[w][e];
    a.part_p[(int64_t)blockIdx.x * a.E + e] = s;
    a.part_c[(int64_t)blockIdx.x * a.E + e] = s_cnt[e];
  }
  if (threadIdx.x == 0) a.part_n[blockIdx.x] = s_n;
}

// One block: the blocks' partial sums in order, in 64 bits.
__global__ void __launch_bounds__(1024) router_balance_sum_kernel(const RouterBalanceArgs a) {
  __shared__ double s_p[1024];
  __shared__ int s_c[1024];
  __shared__ int s_n;
  if (threadIdx.x == 0) s_n = 0;
  __syncthreads();
  int n = 0;
  for (int b = threadIdx.x; b < a.blocks; b += blockDim.x) n += a.part_n[b];
  if (n) atomicAdd(&s_n, n);
  const int groups = 1024 / a.E;  // E <= 512
  const int g = threadIdx.x / a.E, e = threadIdx.x % a.E;
  double p = 0.0;
  int c = 0;
  if (g < groups)
    for (int b = g; b < a.blocks; b += groups) {
      p += a.part_p[(int64_t)b * a.E + e];
      c += a.part_c[(int64_t)b * a.E + e];
    }
  s_p[threadIdx.x] = p;
  s_c[threadIdx.x] = c;
  __syncthreads();
  const double N = max(s_n, 1);
  double v = 0.0;
  if (threadIdx.x < a.E) {
    for (int i = 1; i < groups; ++i) {
      p += s_p[i * a.E + threadIdx.x];
      c += s_c[i * a.E + threadIdx.x];
    }
    const double f = (double)a.E * c / (a.k * N);
    a.counts[threadIdx.x] = c;
    a.coef[threadIdx.x] = (float)(f / N);
    v = f * (p / N);
  }
  __syncthreads();
  s_p[threadIdx.x] = v;
  __syncthreads();
  for (int o = 512; o > 0; o >>= 1) {
    if (threadIdx.x < o) s_p[threadIdx.x] += s_p[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) *a.loss = (float)s_p[0];
}

template <typename T, int EPL>
__global__ void __launch_bounds__(kWarps * 32) router_balance_bwd_kernel(const RouterBalanceArgs a) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float gl = a.dloss ? *a.dloss : 0.f;
  float coef[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i) coef[i] = i * 32 + lane < a.E && a.dloss ? gl * a.coef[i * 32 + lane] : 0.f;
  for (int t = blockIdx.x * kWarps + warp; t < a.T; t += gridDim.x * kWarps) {
    float l[EPL], p[EPL], mx, inv;
    const T* row = reinterpret_cast<const T*>(a.x) + (int64_t)t * a.x_stride;
    row_softmax<T, EPL>(row, a.E, lane, l, p, &mx, &inv);
    const float on = a.dloss && (!a.valid || a.valid[t]) ? 1.f : 0.f;
    // chosen experts: lane j holds choice j
    int e = 0;
    float pe = 0.f, ge = 0.f, ce = 0.f;
    if (lane < a.k && a.dw) {
      e = a.topk_e[(int64_t)t * a.k + lane];
      ge = a.dw[(int64_t)t * a.k + lane];
      pe = __expf(to_f(row[e]) - mx) * inv;
      ce = a.dloss ? on * gl * a.coef[e] : 0.f;
    }
    if (a.renorm && a.dw) {  // w = p / S: d / dp_i = (g_i - sum_j g_j w_j) / S
      const float S = warp_sum(pe), gw = warp_sum(ge * pe) / S;
      ge = lane < a.k ? (ge - gw) / S : 0.f;
    }
    float dot = pe * ge;
#pragma unroll
    for (int i = 0; i < EPL; ++i) dot += p[i] * (on * coef[i]);
    dot = warp_sum(dot);
    T* out = reinterpret_cast<T*>(a.dx) + (int64_t)t * a.E;
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (i * 32 + lane < a.E) out[i * 32 + lane] = from_f<T>(p[i] * (on * coef[i] - dot));
    __syncwarp();  // the chosen experts' values replace those
    if (lane < a.k && a.dw) out[e] = from_f<T>(pe * (ce + ge - dot));
    __syncwarp();
  }
}

template <typename T>
void fwd(const RouterBalanceArgs& a, cudaStream_t st) {
  const int epl = (a.E + 31) / 32;
  if (epl <= 1) router_balance_fwd_kernel<T, 1><<<a.blocks, kWarps * 32, 0, st>>>(a);
  else if (epl <= 2) router_balance_fwd_kernel<T, 2><<<a.blocks, kWarps * 32, 0, st>>>(a);
  else if (epl <= 4) router_balance_fwd_kernel<T, 4><<<a.blocks, kWarps * 32, 0, st>>>(a);
  else if (epl <= 8) router_balance_fwd_kernel<T, 8><<<a.blocks, kWarps * 32, 0, st>>>(a);
  else router_balance_fwd_kernel<T, 16><<<a.blocks, kWarps * 32, 0, st>>>(a);
}
template <typename T>
void bwd(const RouterBalanceArgs& a, int blocks, cudaStream_t st) {
  const int epl = (a.E + 31) / 32;
  if (epl <= 1) router_balance_bwd_kernel<T, 1><<<blocks, kWarps * 32, 0, st>>>(a);
  else if (epl <= 2) router_balance_bwd_kernel<T, 2><<<blocks, kWarps * 32, 0, st>>>(a);
  else if (epl <= 4) router_balance_bwd_kernel<T, 4><<<blocks, kWarps * 32, 0, st>>>(a);
  else if (epl <= 8) router_balance_bwd_kernel<T, 8><<<blocks, kWarps * 32, 0, st>>>(a);
  else router_balance_bwd_kernel<T, 16><<<blocks, kWarps * 32, 0, st>>>(a);
}
void check_args(const RouterBalanceArgs& a) {
  if (a.E < 1 || a.E > kRouterMaxExperts) throw std::runtime_error("router: 1 to 512 experts");
  if (a.k < 1 || a.k > kRouterMaxK || a.k > a.E) throw std::runtime_error("router: top-k must be 1 to min(32, experts)");
}

}  // namespace

int router_balance_blocks(int T, int num_sms) { return std::max(1, std::min((T + kWarps - 1) / kWarps, num_sms * 4)); }

void router_balance_fwd(const RouterBalanceArgs& a, cudaStream_t st) {
  check_args(a);
  if (a.dtype == 0) fwd<__nv_bfloat16>(a, st);
  else if (a.dtype == 1) fwd<__half>(a, st);
  else fwd<float>(a, st);
  check_launch("router_balance_fwd");
  router_balance_sum_kernel<<<1, 1024, 0, st>>>(a);
  check_launch("router_balance_sum");
}

void router_balance_bwd(const RouterBalanceArgs& a, int num_sms, cudaStream_t st) {
  check_args(a);
  if (a.T <= 0) return;
  const int blocks = std::max(1, std::min((a.T + kWarps - 1) / kWarps, num_sms * 8));
  if (a.dtype == 0) bwd<__nv_bfloat16>(a, blocks, st);
  else if (a.dtype == 1) bwd<__half>(a, blocks, st);
  else bwd<float>(a, blocks, st);
  check_launch("router_balance_bwd");
}

}  // namespace sepx
