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
//
// What bounds it: arithmetic, not memory. 65537 tokens x 256 experts in fp32 would take 10 us
// (forward) and 21 us (backward) at 6.55 TB/s; measured 48 us with the sum kernel and 32 us.
// The forward executes 480 instructions per token and warp (sorting, 8 choices, softmax),
// the integer pipe 63% busy; the backward 295. Choosing by scanning all scores for every
// choice took 80 us, with the experts' indices carried beside the keys 72 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <stdexcept>
#include <string>
#include <type_traits>

#include "kernels.h"
#include "router_balance.h"

namespace sepx {
namespace {

constexpr int kWarps = 8, kFwdWarps = 32;

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
__device__ __forceinline__ float warp_max(float v) {  // NaN gives way
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// Order of floats as unsigned numbers (NaN above everything, -0 equal to +0); 0 is below
// every value and marks what is taken or outside the row. The addition turns -0 into +0, and
// any NaN, of either sign, into the one positive NaN that fp32 arithmetic returns.
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);
  const uint32_t k = u ^ ((u & 0x80000000u) ? 0xffffffffu : 0x80000000u);
  return k ? k : 1u;
}

// A row's experts over the lanes: in groups of VEC neighbours (one vector load) where the
// row allows it, else one by one.
template <int VEC>
__device__ __forceinline__ int expert_of(int i, int lane) {
  return (i / VEC) * (32 * VEC) + lane * VEC + i % VEC;
}
// VEC neighbours as one load: 4 floats, or 4 16-bit numbers
__device__ __forceinline__ void unpack4(const float* p, float* o) {
  const float4 v = *reinterpret_cast<const float4*>(p);
  o[0] = v.x; o[1] = v.y; o[2] = v.z; o[3] = v.w;
}
__device__ __forceinline__ void unpack4(const __nv_bfloat16* p, float* o) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  o[0] = __uint_as_float(v.x << 16); o[1] = __uint_as_float(v.x & 0xffff0000u);
  o[2] = __uint_as_float(v.y << 16); o[3] = __uint_as_float(v.y & 0xffff0000u);
}
__device__ __forceinline__ void unpack4(const __half* p, float* o) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&v.x));
  const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
  o[0] = a.x; o[1] = a.y; o[2] = b.x; o[3] = b.y;
}
__device__ __forceinline__ void pack4(float* p, const float* o) {
  *reinterpret_cast<float4*>(p) = make_float4(o[0], o[1], o[2], o[3]);
}
__device__ __forceinline__ void pack4(__nv_bfloat16* p, const float* o) {
  const __nv_bfloat162 a = __floats2bfloat162_rn(o[0], o[1]), b = __floats2bfloat162_rn(o[2], o[3]);
  *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}
__device__ __forceinline__ void pack4(__half* p, const float* o) {
  const __half2 a = __floats2half2_rn(o[0], o[1]), b = __floats2half2_rn(o[2], o[3]);
  *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}
template <typename T, int EPL, int VEC>
__device__ __forceinline__ void load_row(const T* row, int E, int lane, float (&l)[EPL]) {
#pragma unroll
  for (int i = 0; i < EPL; i += VEC) {
    const int e = expert_of<VEC>(i, lane);
    if constexpr (VEC == 1) l[i] = e < E ? to_f(row[e]) : -INFINITY;
    else unpack4(row + e, l + i);
  }
}
template <typename T, int EPL, int VEC>
__device__ __forceinline__ void store_row(T* row, int E, int lane, const float (&o)[EPL]) {
#pragma unroll
  for (int i = 0; i < EPL; i += VEC) {
    const int e = expert_of<VEC>(i, lane);
    if constexpr (VEC == 1) {
      if (e < E) row[e] = from_f<T>(o[i]);
    } else {
      pack4(row + e, o + i);
    }
  }
}

// e^x as 2^(x log2 e), hardware approximation (results below 2^-126 flush to 0)
__device__ __forceinline__ float fast_exp(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.4426950408889634f));
  return y;
}

// softmax of a row from its logits (experts past E: -infinity, p = 0)
template <int EPL>
__device__ __forceinline__ void row_softmax(const float (&l)[EPL], float (&p)[EPL], float* mx_out, float* inv_out) {
  float mx = -INFINITY, s = 0.f;
#pragma unroll
  for (int i = 0; i < EPL; ++i) mx = fmaxf(mx, l[i]);
  mx = warp_max(mx);
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    p[i] = fast_exp(l[i] - mx);
    s += p[i];
  }
  const float inv = __fdividef(1.f, warp_sum(s));
#pragma unroll
  for (int i = 0; i < EPL; ++i) p[i] *= inv;
  *mx_out = mx;
  *inv_out = inv;
}

// Sorts descending (Batcher's odd-even merge exchange).
template <int N>
__device__ __forceinline__ void sort_descending(uint32_t (&v)[N]) {
#pragma unroll
  for (int p = 1; p < N; p *= 2)
#pragma unroll
    for (int k = p; k >= 1; k /= 2)
#pragma unroll
      for (int j = k % p; j + k < N; j += 2 * k)
#pragma unroll
        for (int i = 0; i < k; ++i)
          if (i + j + k < N && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
            const uint32_t a = v[i + j], b = v[i + j + k];
            v[i + j] = max(a, b);
            v[i + j + k] = min(a, b);
          }
}

// The k best of a row's scores, lane j the j-th expert. Scores are compared as 32-bit numbers
// that hold the score's order key in their high bits and the expert in the low 9 (lower
// expert, larger number): one warp maximum gives the winner, and equal scores go to the
// lowest index. Each lane sorts its experts once; a choice pops the winner's list. The key's
// own low 9 bits are dropped: exact for scores whose low 9 bits are all zero (any that came
// from 16 bits), and wherever the first k + 1 numbers differ above the expert's bits.
// Anything else takes the slow selection on whole keys.
template <int EPL, int VEC, bool FROM16>
__device__ __forceinline__ int choose(int E, int k, int lane, const float (&score)[EPL], bool from16) {
  uint32_t v[EPL];
  bool exact = FROM16 && from16;
  if (!exact) {
    uint32_t low = 0;
#pragma unroll
    for (int i = 0; i < EPL; ++i) low |= __float_as_uint(score[i]);
    exact = !__any_sync(0xffffffffu, (low & 511u) != 0);
  }
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const int e = expert_of<VEC>(i, lane);
    // a score's number is above 511 (the smallest keys share one order); 0 past the row's end
    const uint32_t key = max(order_key(score[i]), 512u);
    v[i] = (VEC > 1 || e < E) ? (key & ~511u) | (511u - (uint32_t)e) : 0u;
  }
  sort_descending(v);
  int my_e = 0;
  uint32_t prev = 0;
  bool clash = false;
  const int n = exact ? k : min(k + 1, E);
  for (int j = 0; j < n; ++j) {
    const uint32_t best = __reduce_max_sync(0xffffffffu, v[0]);
    if (lane == j) my_e = 511 - (int)(best & 511u);
    clash |= j > 0 && ((best ^ prev) & ~511u) == 0;
    prev = best;
    if (v[0] == best) {
#pragma unroll
      for (int i = 0; i + 1 < EPL; ++i) v[i] = v[i + 1];
      v[EPL - 1] = 0u;
    }
  }
  if (!exact && clash) {
    uint32_t key[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) key[i] = expert_of<VEC>(i, lane) < E ? order_key(score[i]) : 0u;
    for (int j = 0; j < k; ++j) {
      uint32_t best = 0;
#pragma unroll
      for (int i = 0; i < EPL; ++i) best = max(best, key[i]);
      best = __reduce_max_sync(0xffffffffu, best);
      int be = 0x7fffffff;
#pragma unroll
      for (int i = EPL - 1; i >= 0; --i)
        if (key[i] == best) be = min(be, expert_of<VEC>(i, lane));
      be = __reduce_min_sync(0xffffffffu, be);
#pragma unroll
      for (int i = 0; i < EPL; ++i)
        if (expert_of<VEC>(i, lane) == be) key[i] = 0u;
      if (lane == j) my_e = be;
    }
  }
  return my_e;
}

template <typename T, int EPL, int VEC>
__global__ void __launch_bounds__(kFwdWarps * 32) router_balance_fwd_kernel(const RouterBalanceArgs a) {
  __shared__ int s_cnt[EPL * 32];
  __shared__ float s_p[kFwdWarps / 2][EPL * 32];
  __shared__ int s_n;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int e = threadIdx.x; e < EPL * 32; e += blockDim.x) s_cnt[e] = 0;
  if (threadIdx.x == 0) s_n = 0;
  __syncthreads();
  float acc[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i) acc[i] = 0.f;
  int n = 0;
  const int step = gridDim.x * kFwdWarps;
  int t = blockIdx.x * kFwdWarps + warp;
  auto row_of = [&](int tt) { return reinterpret_cast<const T*>(a.x) + (int64_t)tt * a.x_stride; };
  float next[EPL];  // the next token's row, loaded while this one is worked on
  bool next_on = false;
  if (t < a.T) {
    load_row<T, EPL, VEC>(row_of(t), a.E, lane, next);
    next_on = !a.valid || a.valid[t];
  }
  for (; t < a.T; t += step) {
    float l[EPL], p[EPL], mx, inv;
#pragma unroll
    for (int i = 0; i < EPL; ++i) l[i] = next[i];
    const bool on = next_on;
    if (t + step < a.T) {
      load_row<T, EPL, VEC>(row_of(t + step), a.E, lane, next);
      next_on = !a.valid || a.valid[t + step];
    }
    row_softmax<EPL>(l, p, &mx, &inv);
    if (on) {
      ++n;
#pragma unroll
      for (int i = 0; i < EPL; ++i) acc[i] += p[i];
    }
    // p grows with the logit, so without a bias the logits themselves are compared
    if (a.bias) {
#pragma unroll
      for (int i = 0; i < EPL; ++i) {
        const int e = expert_of<VEC>(i, lane);
        l[i] = e < a.E ? p[i] + a.bias[e] : -INFINITY;
      }
    }
    const int my_e = choose<EPL, VEC, sizeof(T) == 2>(a.E, a.k, lane, l, !a.bias);
    const float my_p = lane < a.k ? fast_exp(to_f(row_of(t)[my_e]) - mx) * inv : 0.f;
    const float S = a.renorm ? warp_sum(my_p) : 1.f;
    if (lane < a.k) {
      a.topk_e[(int64_t)t * a.k + lane] = my_e;
      a.topk_w[(int64_t)t * a.k + lane] = my_p / S;
      if (on) atomicAdd(&s_cnt[my_e], 1);
    }
  }
  // the warps' sums in a fixed order: the upper half onto the lower one, then down the rows
  if (warp >= kFwdWarps / 2)
#pragma unroll
    for (int i = 0; i < EPL; ++i) s_p[warp - kFwdWarps / 2][expert_of<VEC>(i, lane)] = acc[i];
  if (lane == 0 && n) atomicAdd(&s_n, n);
  __syncthreads();
  if (warp < kFwdWarps / 2)
#pragma unroll
    for (int i = 0; i < EPL; ++i) s_p[warp][expert_of<VEC>(i, lane)] += acc[i];
  __syncthreads();
  for (int e = threadIdx.x; e < a.E; e += blockDim.x) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kFwdWarps / 2; ++w) s += s_p[w][e];
    a.part_p[(int64_t)blockIdx.x * a.E + e] = s;
    a.part_c[(int64_t)blockIdx.x * a.E + e] = s_cnt[e];
  }
  if (threadIdx.x == 0) {
    a.part_n[blockIdx.x] = s_n;
    if (blockIdx.x == 0) *a.ticket = 0;  // for the kernel that adds the parts
  }
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The blocks' partial sums, one warp per expert, in a fixed order and in 64 bits; the last
// block to finish adds the experts' products to the loss.
constexpr int kSumWarps = 8;
__global__ void __launch_bounds__(kSumWarps * 32) router_balance_sum_kernel(const RouterBalanceArgs a) {
  __shared__ double s_v[kSumWarps];
  __shared__ bool last;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int e = blockIdx.x * kSumWarps + warp;
  if (e < a.E) {
    int n = 0, c = 0;
    double p = 0.0;
#pragma unroll 10
    for (int b = lane; b < a.blocks; b += 32) {
      n += a.part_n[b];
      c += a.part_c[(int64_t)b * a.E + e];
      p += a.part_p[(int64_t)b * a.E + e];
    }
    n = __reduce_add_sync(0xffffffffu, n);
    c = __reduce_add_sync(0xffffffffu, c);
    p = warp_sum(p);
    if (lane == 0) {
      const double N = max(n, 1);
      const double f = (double)a.E * c / (a.k * N);
      a.counts[e] = c;
      a.coef[e] = (float)(f / N);
      a.part_l[e] = f * (p / N);
      __threadfence();
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(a.ticket, 1u) == gridDim.x - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  double v = 0.0;
  for (int i = threadIdx.x; i < a.E; i += kSumWarps * 32) v += __ldcg(a.part_l + i);
  v = warp_sum(v);
  if (lane == 0) s_v[warp] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kSumWarps; ++w) v += s_v[w];
    *a.loss = (float)v;
  }
}

template <typename T, int EPL, int VEC>
__global__ void __launch_bounds__(kWarps * 32) router_balance_bwd_kernel(const RouterBalanceArgs a) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float gl = a.dloss ? *a.dloss : 0.f;
  float coef[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i)
    coef[i] = expert_of<VEC>(i, lane) < a.E && a.dloss ? gl * a.coef[expert_of<VEC>(i, lane)] : 0.f;
  const int step = gridDim.x * kWarps;
  int t = blockIdx.x * kWarps + warp;
  auto row_of = [&](int tt) { return reinterpret_cast<const T*>(a.x) + (int64_t)tt * a.x_stride; };
  // the next token's row and choices, loaded while this one is worked on; lane j holds choice j
  float next[EPL], next_g = 0.f;
  int next_e = 0;
  bool next_on = false;
  auto load_next = [&](int tt) {
    load_row<T, EPL, VEC>(row_of(tt), a.E, lane, next);
    if (lane < a.k && a.dw) {
      next_e = a.topk_e[(int64_t)tt * a.k + lane];
      next_g = a.dw[(int64_t)tt * a.k + lane];
    }
    next_on = a.dloss && (!a.valid || a.valid[tt]);
  };
  if (t < a.T) load_next(t);
  for (; t < a.T; t += step) {
    float l[EPL], p[EPL], mx, inv;
#pragma unroll
    for (int i = 0; i < EPL; ++i) l[i] = next[i];
    const float on = next_on ? 1.f : 0.f;
    const int e = next_e;
    float ge = next_g, pe = 0.f, ce = 0.f;
    if (lane < a.k && a.dw) {
      pe = to_f(row_of(t)[e]);
      ce = a.dloss ? on * gl * a.coef[e] : 0.f;
    }
    if (t + step < a.T) load_next(t + step);
    row_softmax<EPL>(l, p, &mx, &inv);
    pe = lane < a.k && a.dw ? fast_exp(pe - mx) * inv : 0.f;
    float dot = 0.f;  // sum p g: zero over the chosen experts where their weights sum to 1
    if (a.dw) {
      if (a.renorm) {
        // w = p / S: d / dp_i = (g_i - sum_j g_j w_j) / S. The weights sum to 1, so the g may be
        // counted from the first choice's: where it has nearly all the weight (all of it at
        // k = 1, where the result is 0) nothing large is left to cancel.
        ge -= __shfl_sync(0xffffffffu, ge, 0);
        float S = pe, gw = ge * pe;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          S += __shfl_xor_sync(0xffffffffu, S, o);
          gw += __shfl_xor_sync(0xffffffffu, gw, o);
        }
        ge = lane < a.k ? (ge - gw / S) / S : 0.f;
      } else {
        dot = pe * ge;
      }
    }
#pragma unroll
    for (int i = 0; i < EPL; ++i) dot += p[i] * (on * coef[i]);
    dot = warp_sum(dot);
    T* out = reinterpret_cast<T*>(a.dx) + (int64_t)t * a.E;
#pragma unroll
    for (int i = 0; i < EPL; ++i) l[i] = p[i] * (on * coef[i] - dot);
    store_row<T, EPL, VEC>(out, a.E, lane, l);
    __syncwarp();  // the chosen experts' values replace those
    if (lane < a.k && a.dw) out[e] = from_f<T>(pe * (ce + ge - dot));
    __syncwarp();
  }
}

// Calls f(EPL, VEC) as compile-time numbers: experts per lane, and neighbours per load where
// rows are whole vectors at aligned addresses.
template <typename T, typename F>
void with_layout(const RouterBalanceArgs& a, const void* out, F f) {
  auto aligned = [&](int vec) {
    const uintptr_t b = sizeof(T) * (uintptr_t)vec;
    return a.E % (32 * vec) == 0 && reinterpret_cast<uintptr_t>(a.x) % b == 0 &&
           (uintptr_t)a.x_stride * sizeof(T) % b == 0 && reinterpret_cast<uintptr_t>(out) % b == 0;
  };
  using std::integral_constant;
  const int epl = (a.E + 31) / 32;
  if (epl <= 1) f(integral_constant<int, 1>(), integral_constant<int, 1>());
  else if (epl <= 2) f(integral_constant<int, 2>(), integral_constant<int, 1>());
  else if (epl == 4 && aligned(4)) f(integral_constant<int, 4>(), integral_constant<int, 4>());
  else if (epl <= 4) f(integral_constant<int, 4>(), integral_constant<int, 1>());
  else if (epl == 8 && aligned(4)) f(integral_constant<int, 8>(), integral_constant<int, 4>());
  else if (epl <= 8) f(integral_constant<int, 8>(), integral_constant<int, 1>());
  else if (epl == 16 && aligned(4)) f(integral_constant<int, 16>(), integral_constant<int, 4>());
  else f(integral_constant<int, 16>(), integral_constant<int, 1>());
}
template <typename T>
void fwd(const RouterBalanceArgs& a, cudaStream_t st) {
  with_layout<T>(a, nullptr, [&](auto epl, auto vec) {
    router_balance_fwd_kernel<T, decltype(epl)::value, decltype(vec)::value><<<a.blocks, kFwdWarps * 32, 0, st>>>(a);
  });
}
template <typename T>
void bwd(const RouterBalanceArgs& a, int blocks, cudaStream_t st) {
  with_layout<T>(a, a.dx, [&](auto epl, auto vec) {
    router_balance_bwd_kernel<T, decltype(epl)::value, decltype(vec)::value><<<blocks, kWarps * 32, 0, st>>>(a);
  });
}
void check_args(const RouterBalanceArgs& a) {
  if (a.E < 1 || a.E > kRouterMaxExperts) throw std::runtime_error("router: 1 to 512 experts");
  if (a.k < 1 || a.k > kRouterMaxK || a.k > a.E) throw std::runtime_error("router: top-k must be 1 to min(32, experts)");
}

}  // namespace

int router_balance_blocks(int T, int num_sms) { return std::max(1, std::min((T + kFwdWarps - 1) / kFwdWarps, num_sms)); }

void router_balance_fwd(const RouterBalanceArgs& a, cudaStream_t st) {
  check_args(a);
  if (a.dtype == 0) fwd<__nv_bfloat16>(a, st);
  else if (a.dtype == 1) fwd<__half>(a, st);
  else fwd<float>(a, st);
  check_launch("router_balance_fwd");
  router_balance_sum_kernel<<<(a.E + kSumWarps - 1) / kSumWarps, kSumWarps * 32, 0, st>>>(a);
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
