// Losses over a vocabulary's logits, each with its gradient:
//   distillation   p = softmax of the teacher's listed logits / tau, q = softmax(z / tau):
//                  loss_t = tau^2 sum_k p_k (ln p_k - ln q_k),  dz = tau (q - P)
//   policy         l = ln softmax(z / tau)[a], r = e^(l - old):
//                  loss_t = -min(r A, clip(r) A) + beta (e^(ref-l) - (ref-l) - 1)
//                  dz = -(1 / tau) dloss/dl (q - onehot(a))
//   log-prob       l = ln softmax(z)[y] for the preference loss
// All three need the row's log-sum-exp and one gradient form, A (q - P) with a P of few
// entries, so one kernel body serves them. Exponentials are 2^((z - max) c2) with
// c2 = log2(e) / tau: the difference first, so a row of the type's lowest or highest values
// does not overflow on the way. Logits are read as they are (bf16, fp16 or fp32), everything
// is computed in fp32, and the gradient is rounded once, to the logits' type.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <stdexcept>
#include <string>

#include "kernels.h"
#include "vocab_loss.h"

namespace sepx {
namespace {

constexpr float kLn2 = 0.69314718055994531f;

void check_launch(const char* what) {
  note_launch();
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) throw std::runtime_error(std::string(what) + ": " + cudaGetErrorString(e));
}

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
__device__ __forceinline__ float block_sum(float v, float* s) {  // s: 32 floats
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  const int nw = blockDim.x >> 5;
  return warp_sum((int)(threadIdx.x & 31) < nw ? s[threadIdx.x & 31] : 0.f);
}
__device__ __forceinline__ float block_max(float v, float* s) {
  v = warp_max(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  const int nw = blockDim.x >> 5;
  return warp_max((int)(threadIdx.x & 31) < nw ? s[threadIdx.x & 31] : -INFINITY);
}

// 2^x, hardware approximation (results below 2^-126 flush to 0: nothing beside a sum >= 1)
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ------------------------------------------------------------------------------------
// 16-byte vectors of one element type
// ------------------------------------------------------------------------------------
template <typename T>
struct Elem;
template <>
struct Elem<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ float f(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 t(float v) { return __float2bfloat16(v); }
  static __device__ __forceinline__ void unpack(const uint4& v, float (&o)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      o[2 * i] = __uint_as_float(w[i] << 16);
      o[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&o)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      __nv_bfloat162 h = __floats2bfloat162_rn(o[2 * i], o[2 * i + 1]);
      w[i] = *reinterpret_cast<uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <>
struct Elem<__half> {
  static constexpr int N = 8;
  static __device__ __forceinline__ float f(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half t(float v) { return __float2half(v); }
  static __device__ __forceinline__ void unpack(const uint4& v, float (&o)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      o[2 * i] = p.x;
      o[2 * i + 1] = p.y;
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&o)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      __half2 h = __floats2half2_rn(o[2 * i], o[2 * i + 1]);
      w[i] = *reinterpret_cast<uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <>
struct Elem<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ float f(float v) { return v; }
  static __device__ __forceinline__ float t(float v) { return v; }
  static __device__ __forceinline__ void unpack(const uint4& v, float (&o)[4]) {
    o[0] = __uint_as_float(v.x); o[1] = __uint_as_float(v.y); o[2] = __uint_as_float(v.z); o[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ uint4 pack(const float (&o)[4]) {
    return make_uint4(__float_as_uint(o[0]), __float_as_uint(o[1]), __float_as_uint(o[2]), __float_as_uint(o[3]));
  }
};

// A row as 16-byte vectors on the memory's own 16-byte grid: the row may start anywhere in
// its first vector, so odd vocabularies and any row stride keep full-width accesses, and
// only the first and the last vector of a row are touched element by element.
template <typename T>
struct RowVec {
  static constexpr int N = Elem<T>::N;
  T* p;  // first element of the row
  int a;  // elements of the first vector that lie before the row
  int V, nv;
  __device__ __forceinline__ RowVec(T* row, int V_) : p(row), V(V_) {
    a = (int)((reinterpret_cast<uintptr_t>(row) / sizeof(T)) % N);
    nv = (int)(((int64_t)a + V + N - 1) / N);
  }
  __device__ __forceinline__ int64_t first(int j) const { return (int64_t)j * N - a; }
  __device__ __forceinline__ bool full(int j) const { return first(j) >= 0 && first(j) + N <= V; }
  // elements outside the row read as -infinity
  __device__ __forceinline__ uint4 load(int j) const {
    const int64_t e0 = first(j);
    if (full(j)) return *reinterpret_cast<const uint4*>(p + e0);
    float o[N];
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = (e0 + i >= 0 && e0 + i < V) ? Elem<T>::f(p[e0 + i]) : -INFINITY;
    return Elem<T>::pack(o);
  }
  // o[i] belongs to element e0 + i (e0 may come from a row with another phase)
  __device__ __forceinline__ void store(int64_t e0, const float (&o)[N]) const {
    if (e0 >= 0 && e0 + N <= V && (e0 + a) % N == 0) {
      *reinterpret_cast<uint4*>(p + e0) = Elem<T>::pack(o);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (e0 + i >= 0 && e0 + i < V) p[e0 + i] = Elem<T>::t(o[i]);
    }
  }
};

__device__ __forceinline__ int64_t load_id(const void* p, int64_t i, bool is64) {
  return is64 ? reinterpret_cast<const int64_t*>(p)[i] : (int64_t) reinterpret_cast<const int*>(p)[i];
}

// ------------------------------------------------------------------------------------
// The sparse side of a row: its entries in shared memory, K of them (1 for a token)
// ------------------------------------------------------------------------------------
struct Entries {
  int* id;    // -1: not an entry
  float* p;   // weight P; where ids repeat, the gradient takes the sum of their weights
  float* lp;  // ln P (distillation)
  float* z;   // the row's logit at id
};
__host__ __device__ inline size_t entries_bytes(int op, int K) { return op == kOpDistill ? (size_t)K * 16 : 16; }
__device__ __forceinline__ Entries entries_at(void* smem, int K) {
  float* f = reinterpret_cast<float*>(smem);
  return {reinterpret_cast<int*>(f), f + K, f + 2 * K, f + 3 * K};
}

// A row's part in the loss. Bad: an id outside the vocabulary, which turns the row's
// outputs into NaN (and is never used as an index).
enum RowState : int { kRowOff = 0, kRowOn = 1, kRowBad = 2 };

// Fills id / p / lp of row t; called by all threads, which all get the row's state.
template <int OP>
__device__ __forceinline__ int row_entries(const VocabLossArgs& a, int t, const Entries& s, float* red) {
  if constexpr (OP == kOpDistill) {
    float top = -INFINITY;
    int any = 0, bad = 0;
    for (int k = threadIdx.x; k < a.K; k += blockDim.x) {
      const int64_t id = load_id(a.ids, (int64_t)t * a.K + k, a.ids64);
      const float v = a.teacher[(int64_t)t * a.K + k];
      const bool has = id >= 0 && v != -INFINITY;
      any |= has;
      bad |= has && id >= a.V;
      s.id[k] = has ? (int)(id < a.V ? id : 0) : -1;
      s.p[k] = v;
      if (has) top = fmaxf(top, v);
    }
    any = __syncthreads_or(any);
    bad = __syncthreads_or(bad);
    if (!any) return kRowOff;
    top = block_max(top, red);
    float sum = 0.f;
    for (int k = threadIdx.x; k < a.K; k += blockDim.x)
      if (s.id[k] >= 0) sum += expf((s.p[k] - top) / a.tau);
    sum = block_sum(sum, red);
    const float lsum = logf(sum);
    for (int k = threadIdx.x; k < a.K; k += blockDim.x) {
      const bool has = s.id[k] >= 0;
      const float lp = has ? (s.p[k] - top) / a.tau - lsum : 0.f;
      s.lp[k] = lp;
      s.p[k] = has ? expf(lp) : 0.f;
    }
    __syncthreads();
    return bad ? kRowBad : kRowOn;
  } else {
    const int64_t id = load_id(a.labels, t, a.ids64);
    bool on = id >= 0;
    if (OP == kOpLogp && a.offsets) on = on && t >= a.offsets[0] && t < a.offsets[a.num_seq];
    if (threadIdx.x == 0) {
      s.id[0] = on && id < a.V ? (int)id : (on ? 0 : -1);
      s.p[0] = 1.f;
    }
    __syncthreads();
    return !on ? kRowOff : id < a.V ? kRowOn : kRowBad;
  }
}

// 1 / rows in the loss
__device__ __forceinline__ float rows_scale(const VocabLossArgs& a) {
  return a.count ? 1.f / (float)max(*a.count, 1) : a.host_scale;
}

// Outputs of a row that is not in the loss (one thread).
template <int OP>
__device__ __forceinline__ void row_off(const VocabLossArgs& a, int t) {
  if (OP != kOpLogp) a.row_loss[t] = 0.f;
  if (OP != kOpDistill) a.logp[t] = 0.f;
  if (OP == kOpPolicy) a.kl[t] = 0.f;
  if (OP == kOpLogp && a.lse) reinterpret_cast<float2*>(a.lse)[t] = make_float2(0.f, 0.f);
}

// Outputs of a row in the loss (from the threads of the block that has `write`), and the
// factor A of its gradient A (q - P) (all threads). mx = the row's maximum, l2s = log2 of
// sum 2^((z - mx) c2).
template <int OP>
__device__ __forceinline__ float row_on(const VocabLossArgs& a, int t, int state, const Entries& s, float mx, float l2s,
                                        float* red, bool write) {
  const float nan = __int_as_float(0x7fffffff);
  if constexpr (OP == kOpDistill) {
    if (write) {
      float d = 0.f;
      for (int k = threadIdx.x; k < a.K; k += blockDim.x)
        if (s.id[k] >= 0 && s.p[k] != 0.f) d += s.p[k] * (s.lp[k] - kLn2 * fmaf(s.z[k] - mx, a.c2, -l2s));
      d = block_sum(d, red);
      if (threadIdx.x == 0) a.row_loss[t] = state == kRowBad ? nan : a.tau * a.tau * d;
    }
    if (state == kRowBad) return nan;
    return a.tau * rows_scale(a) * (a.up ? *a.up : 1.f);
  } else {
    const float logp = state == kRowBad ? nan : kLn2 * fmaf(s.z[0] - mx, a.c2, -l2s);
    if constexpr (OP == kOpLogp) {
      if (write && threadIdx.x == 0) {
        a.logp[t] = logp;
        if (a.lse) reinterpret_cast<float2*>(a.lse)[t] = make_float2(mx, l2s);
      }
      return -1.f;
    } else {
      const float A = a.adv[t], r = expf(logp - a.old_logp[t]);
      // an advantage of 0 asks for nothing, also where the ratio overflows
      const float u = A == 0.f ? 0.f : r * A;
      const float v = A == 0.f ? 0.f : fminf(fmaxf(r, 1.f - a.clip_low), 1.f + a.clip_high) * A;
      float loss = -(u <= v ? u : v), dl = u <= v ? -u : 0.f, kl = 0.f;
      if (r != r) loss = dl = nan;  // the clamp drops NaN
      if (a.ref_logp) {
        const float d = a.ref_logp[t] - logp, em = expm1f(d);
        kl = em - d;
        if (a.kl_coef != 0.f) {
          loss += a.kl_coef * kl;
          dl -= a.kl_coef * em;
        }
      }
      if (write && threadIdx.x == 0) {
        a.row_loss[t] = loss;
        a.logp[t] = logp;
        a.kl[t] = kl;
      }
      return -dl / a.tau * rows_scale(a) * (a.up ? *a.up : 1.f);
    }
  }
}

// The weight at entry k's id: the sum over the entries with the same id, in their order.
template <int OP>
__device__ __forceinline__ float weight_at(const Entries& s, int K, int k) {
  if (OP != kOpDistill) return 1.f;
  const int id = s.id[k];
  float p = 0.f;
  for (int j = 0; j < K; ++j)
    if (s.id[j] == id) p += s.p[j];
  return p;
}

// One block per row, any vocabulary: the row is read for its maximum, and again (from L2
// where it fits) for the sum and for the gradient.
template <typename T, int OP>
__global__ void __launch_bounds__(512) vocab_row_kernel(const VocabLossArgs a) {
  constexpr int N = Elem<T>::N;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float red[32];
  const int t = blockIdx.x;
  const int K = OP == kOpDistill ? a.K : 1;
  const Entries s = entries_at(smem, K);
  const RowVec<T> z(const_cast<T*>(reinterpret_cast<const T*>(a.z)) + (int64_t)t * a.z_stride, a.V);
  const RowVec<T> g(reinterpret_cast<T*>(a.grad) + (a.grad ? (int64_t)t * a.grad_stride : 0), a.V);
  const int state = row_entries<OP>(a, t, s, red);
  if (state == kRowOff) {
    if (threadIdx.x == 0) row_off<OP>(a, t);
    if (a.grad) {
      const float o[N] = {};
      for (int j = threadIdx.x; j < g.nv; j += blockDim.x) g.store(g.first(j), o);
    }
    return;
  }
  for (int k = threadIdx.x; k < K; k += blockDim.x) s.z[k] = s.id[k] >= 0 ? Elem<T>::f(z.p[s.id[k]]) : 0.f;
  float mx = -INFINITY, sum = 0.f;
  for (int j = threadIdx.x; j < z.nv; j += blockDim.x) {
    float o[N];
    Elem<T>::unpack(z.load(j), o);
#pragma unroll
    for (int i = 0; i < N; ++i) mx = fmaxf(mx, o[i]);
  }
  mx = block_max(mx, red);
  for (int j = threadIdx.x; j < z.nv; j += blockDim.x) {
    float o[N];
    Elem<T>::unpack(z.load(j), o);
#pragma unroll
    for (int i = 0; i < N; ++i) sum += ex2((o[i] - mx) * a.c2);
  }
  sum = block_sum(sum, red);
  const float l2s = log2f(sum);
  __syncthreads();  // s.z
  const float A = row_on<OP>(a, t, state, s, mx, l2s, red, true);
  if (!a.grad) return;
  __syncthreads();
  for (int j = threadIdx.x; j < z.nv; j += blockDim.x) {
    float o[N];
    Elem<T>::unpack(z.load(j), o);
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = A * ex2(fmaf(o[i] - mx, a.c2, -l2s));
    g.store(z.first(j), o);
  }
  __syncthreads();
  for (int k = threadIdx.x; k < K; k += blockDim.x)
    if (s.id[k] >= 0) g.p[s.id[k]] = Elem<T>::t(A * (ex2(fmaf(s.z[k] - mx, a.c2, -l2s)) - weight_at<OP>(s, K, k)));
}

// ------------------------------------------------------------------------------------
// rows in the loss, sums over rows, scaling
// ------------------------------------------------------------------------------------
__global__ void __launch_bounds__(256) count_labels_kernel(const void* labels, bool is64, int T, int* count) {
  int n = 0;
  for (int t = blockIdx.x * blockDim.x + threadIdx.x; t < T; t += gridDim.x * blockDim.x)
    n += load_id(labels, t, is64) >= 0;
  n = __reduce_add_sync(0xffffffffu, n);
  if ((threadIdx.x & 31) == 0 && n) atomicAdd(count, n);
}
// one warp per row
__global__ void __launch_bounds__(256) count_teacher_kernel(const void* ids, bool is64, const float* teacher, int T,
                                                            int K, int* count) {
  const int lane = threadIdx.x & 31;
  const int warps = gridDim.x * (blockDim.x >> 5);
  int n = 0;
  for (int t = (blockIdx.x * blockDim.x + threadIdx.x) >> 5; t < T; t += warps) {
    bool any = false;
    for (int k = lane; k < K && !any; k += 32)
      any = load_id(ids, (int64_t)t * K + k, is64) >= 0 && teacher[(int64_t)t * K + k] != -INFINITY;
    n += __any_sync(0xffffffffu, any) ? 1 : 0;
  }
  if (lane == 0 && n) atomicAdd(count, n);
}

__device__ __forceinline__ double block_sum_d(double v, double* s) {  // s: 32 doubles
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  const int nw = blockDim.x >> 5;
  v = (int)(threadIdx.x & 31) < nw ? s[threadIdx.x & 31] : 0.0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// One block: the same order of additions on every run, in 64 bits (a long sum of terms of
// both signs).
__global__ void __launch_bounds__(1024) rows_sum_kernel(const float* __restrict__ x, int n, float host_scale,
                                                        const int* count, float* out) {
  __shared__ double red[32];
  double v = 0.0;
  for (int i = threadIdx.x; i < n; i += blockDim.x) v += x[i];
  v = block_sum_d(v, red);
  if (threadIdx.x == 0) *out = (float)(count ? v / max(*count, 1) : v * host_scale);
}

// The gradient is already in its type: one more rounding where the loss's own gradient is
// not 1 (exact for powers of two).
template <typename T>
__global__ void __launch_bounds__(256) scale_grad_kernel(T* g, int64_t n, const float* up) {
  const float u = *up;
  if (u == 1.f) return;
  constexpr int N = Elem<T>::N;
  const int64_t step = (int64_t)gridDim.x * blockDim.x, i0 = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  for (int64_t i = i0; i < n / N; i += step) {
    float o[N];
    Elem<T>::unpack(reinterpret_cast<uint4*>(g)[i], o);
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] *= u;
    reinterpret_cast<uint4*>(g)[i] = Elem<T>::pack(o);
  }
  for (int64_t i = n / N * N + i0; i < n; i += step) g[i] = Elem<T>::t(Elem<T>::f(g[i]) * u);
}

// ------------------------------------------------------------------------------------
// Preference pairs: sequence 2 i is the chosen, 2 i + 1 the rejected one of pair i.
// ------------------------------------------------------------------------------------
// One block per pair. Log-ratios are summed in 64 bits: the margin is the difference of
// two sums over whole sequences.
__global__ void __launch_bounds__(256) preference_pairs_kernel(const PreferenceArgs a) {
  __shared__ double red[32];
  const int i = blockIdx.x;
  int lo[2], hi[2];
  double R[2];
  for (int s = 0; s < 2; ++s) {  // offsets are clamped: a wrong one reads no other memory
    lo[s] = min(max(a.offsets[2 * i + s], 0), a.T);
    hi[s] = min(max(a.offsets[2 * i + s + 1], 0), a.T);
    double v = 0.0;
    for (int t = lo[s] + threadIdx.x; t < hi[s]; t += blockDim.x)
      if (load_id(a.labels, t, a.ids64) >= 0) v += (double)a.logp[t] - (double)a.ref_logp[t];
    R[s] = (double)a.beta * block_sum_d(v, red);
  }
  const double m = R[0] - R[1], e = exp(-fabs(m));
  const double sp = log1p(e);  // softplus(-|m|)
  const double neg = m > 0 ? sp : sp - m, pos = m > 0 ? sp + m : sp;  // softplus(-m), softplus(m)
  const double sig_neg = m > 0 ? e / (1.0 + e) : 1.0 / (1.0 + e), sig_pos = 1.0 - sig_neg;
  const double dm = ((double)a.eps * sig_pos - (1.0 - (double)a.eps) * sig_neg) / a.pairs;
  if (threadIdx.x == 0) {
    a.rewards[2 * i] = (float)R[0];
    a.rewards[2 * i + 1] = (float)R[1];
    a.pair_loss[i] = (float)((1.0 - (double)a.eps) * neg + (double)a.eps * pos);
  }
  for (int s = 0; s < 2; ++s) {
    const float c = (float)((s ? -dm : dm) * (double)a.beta);
    for (int t = lo[s] + threadIdx.x; t < hi[s]; t += blockDim.x)
      if (load_id(a.labels, t, a.ids64) >= 0) a.row_coef[t] = c;
  }
}

// dz = up * row_coef * (onehot - softmax) from the saved log-sum-exp: one read, one write.
template <typename T>
__global__ void __launch_bounds__(256) preference_grad_kernel(const VocabLossArgs a, const float* __restrict__ row_coef,
                                                              int chunks, int chunk) {
  constexpr int N = Elem<T>::N;
  const int t = blockIdx.x / chunks, c = blockIdx.x % chunks;
  const RowVec<T> z(const_cast<T*>(reinterpret_cast<const T*>(a.z)) + (int64_t)t * a.z_stride, a.V);
  const RowVec<T> g(reinterpret_cast<T*>(a.grad) + (int64_t)t * a.grad_stride, a.V);
  const int j0 = c * chunk, j1 = min(j0 + chunk, z.nv);
  const int64_t label = load_id(a.labels, t, a.ids64);
  const float coef = row_coef[t];
  // rows outside the loss are not read: their logits may hold anything
  const bool on = label >= 0 && t >= a.offsets[0] && t < a.offsets[a.num_seq];
  const float A = on ? -coef * *a.up : 0.f;
  const float2 l = reinterpret_cast<const float2*>(a.lse)[t];
  for (int j = j0 + threadIdx.x; j < j1; j += blockDim.x) {
    float o[N];
    if (on) {
      Elem<T>::unpack(z.load(j), o);
      const int64_t e0 = z.first(j);
#pragma unroll
      for (int i = 0; i < N; ++i) o[i] = A * (ex2(fmaf(o[i] - l.x, a.c2, -l.y)) - (e0 + i == label ? 1.f : 0.f));
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) o[i] = 0.f;
    }
    g.store(z.first(j), o);
  }
}

template <typename T>
void launch_rows(const VocabLossArgs& a, int op, cudaStream_t st) {
  const size_t sm = entries_bytes(op, a.K);
  if (op == kOpDistill) vocab_row_kernel<T, kOpDistill><<<a.T, 512, sm, st>>>(a);
  else if (op == kOpPolicy) vocab_row_kernel<T, kOpPolicy><<<a.T, 512, sm, st>>>(a);
  else vocab_row_kernel<T, kOpLogp><<<a.T, 512, sm, st>>>(a);
  check_launch("vocab_loss");
}

}  // namespace

void vocab_count_rows(const VocabLossArgs& a, int op, int* count, cudaStream_t st) {
  if (a.T <= 0) return;
  if (op == kOpDistill)
    count_teacher_kernel<<<std::min((a.T + 7) / 8, 592), 256, 0, st>>>(a.ids, a.ids64, a.teacher, a.T, a.K, count);
  else
    count_labels_kernel<<<std::min((a.T + 255) / 256, 148), 256, 0, st>>>(a.labels, a.ids64, a.T, count);
  check_launch("vocab_count_rows");
}

void vocab_loss(const VocabLossArgs& a, int op, cudaStream_t st) {
  if (a.T <= 0) return;
  if (a.V < 1) throw std::runtime_error("vocab_loss: empty vocabulary");
  if (op == kOpDistill && (a.K < 1 || a.K > kMaxTeacher)) throw std::runtime_error("vocab_loss: teacher entries");
  if (a.dtype == kVocabBf16) launch_rows<__nv_bfloat16>(a, op, st);
  else if (a.dtype == kVocabF16) launch_rows<__half>(a, op, st);
  else launch_rows<float>(a, op, st);
}

void vocab_loss_sum(const VocabLossArgs& a, float* loss, cudaStream_t st) {
  rows_sum_kernel<<<1, 1024, 0, st>>>(a.row_loss, a.T, a.host_scale, a.count, loss);
  check_launch("vocab_loss_sum");
}

void vocab_scale_grad(void* grad, int dtype, int64_t n, const float* up, int num_sms, cudaStream_t st) {
  if (n <= 0) return;
  const int blocks = (int)std::min<int64_t>((n + 2047) / 2048, (int64_t)num_sms * 8);
  if (dtype == kVocabBf16) scale_grad_kernel<<<blocks, 256, 0, st>>>(reinterpret_cast<__nv_bfloat16*>(grad), n, up);
  else if (dtype == kVocabF16) scale_grad_kernel<<<blocks, 256, 0, st>>>(reinterpret_cast<__half*>(grad), n, up);
  else scale_grad_kernel<<<blocks, 256, 0, st>>>(reinterpret_cast<float*>(grad), n, up);
  check_launch("vocab_scale_grad");
}

void preference_pairs(const PreferenceArgs& a, cudaStream_t st) {
  if (a.pairs <= 0) return;
  preference_pairs_kernel<<<a.pairs, 256, 0, st>>>(a);
  check_launch("preference_pairs");
}

void preference_loss_sum(const float* pair_loss, int pairs, float* loss, cudaStream_t st) {
  rows_sum_kernel<<<1, 1024, 0, st>>>(pair_loss, pairs, 1.f / (float)std::max(pairs, 1), nullptr, loss);
  check_launch("preference_loss_sum");
}

void preference_grad(const VocabLossArgs& a, const float* row_coef, cudaStream_t st) {
  if (a.T <= 0) return;
  const int n = a.dtype == kVocabF32 ? 4 : 8;
  const int nv = (int)(((int64_t)a.V + 2 * n - 2) / n);  // vectors of a row at its worst phase
  const int chunk = 2048, chunks = (nv + chunk - 1) / chunk;
  const int64_t blocks = (int64_t)a.T * chunks;
  if (blocks > 0x7fffffff) throw std::runtime_error("preference_grad: too many rows");
  if (a.dtype == kVocabBf16)
    preference_grad_kernel<__nv_bfloat16><<<(int)blocks, 256, 0, st>>>(a, row_coef, chunks, chunk);
  else if (a.dtype == kVocabF16) preference_grad_kernel<__half><<<(int)blocks, 256, 0, st>>>(a, row_coef, chunks, chunk);
  else preference_grad_kernel<float><<<(int)blocks, 256, 0, st>>>(a, row_coef, chunks, chunk);
  check_launch("preference_grad");
}

}  // namespace sepx
