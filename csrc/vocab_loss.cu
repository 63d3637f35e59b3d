// Losses over a vocabulary's logits, each with its gradient:
//   distillation   p = softmax of the teacher's listed logits / tau, q = softmax(z / tau):
//                  loss_t = tau^2 sum_k p_k (ln p_k - ln q_k),  dz = tau (q - P)
//   policy         l = ln softmax(z / tau)[a], r = e^(l - old):
//                  loss_t = -min(r A, clip(r) A) + beta (e^(ref-l) - (ref-l) - 1)
//                  dz = -(1 / tau) dloss/dl (q - onehot(a))
//   log-prob       l = ln softmax(z)[y] for the preference loss
// All three need the row's log-sum-exp and one gradient form, A (q - P) with a P of few
// entries, so one kernel body serves them. Logits are read as they are (bf16, fp16 or fp32),
// everything is computed in fp32, and the gradient is rounded once, to the logits' type.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <array>
#include <map>
#include <mutex>
#include <stdexcept>
#include <string>
#include <type_traits>

#include "kernels.h"
#include "sm100.cuh"
#include "vocab_loss.h"

namespace sepx {
namespace {

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
__device__ __forceinline__ float warp_max(float v) {  // NaN gives way
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
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

// 2^x, hardware approximation (results below 2^-126 flush to 0: nothing beside a sum >= 1)
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two floats in one 64-bit register: sm_100 does one multiply-add for both.
struct F2 {
  unsigned long long v;
};
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void split(F2 a, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(a.v)); }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 ex2_2(F2 a) {
  float x, y;
  split(a, x, y);
  return f2(ex2(x), ex2(y));
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
// Exponentials of a row: 2^(z c2 - M2), c2 = log2(e) / tau in two parts (the rounding of one
// fp32 would show in log-probabilities: 1.3e-8 of a token's distance from the mean logit). The
// first part has 12 bits: its product with a 16-bit logit is exact, and the second part's
// product is not so small beside the first result that rounding always drops it, which left a
// mean error of 4e-8 per token. M2 = m c2 of a reference m (the row's maximum, or near it),
// rounded to a whole number: sums against different references are joined by powers of two,
// exactly. The fused products form z c2 - M2 to 2^-36 of |M2| (the second part's own rounding),
// which is 2^-19 where |M2| is 2^17; beyond that (rows of mask values such as -1e9 or the
// type's lowest, logits far from 0) the difference z - m comes first, and M2 is not used.
// ------------------------------------------------------------------------------------
constexpr float kFarM2 = 131072.f;
struct C2 {
  float all, hi, lo;  // all: one fp32, for references
};
// z c2 + R for two z, in sums and gradients alike: a gradient with the constant in one fp32
// would be off by 1.3e-8 of z against its row's sum.
__device__ __forceinline__ F2 arg2(F2 z, F2 hi, F2 lo, F2 R) { return fma2(z, lo, fma2(z, hi, R)); }
struct Expo {
  C2 c2;
  float m, M2;
  bool far;
  __device__ __forceinline__ Expo(C2 c2_, float m_) {
    c2 = c2_;
    m = m_;
    M2 = rintf(m_ * c2.all);
    far = !(fabsf(M2) <= kFarM2);
  }
  __device__ __forceinline__ float arg(float z) const {
    if (far) {
      const float d = z - m;
      return fmaf(d, c2.lo, d * c2.hi);
    }
    return fmaf(z, c2.lo, fmaf(z, c2.hi, -M2));
  }
  __device__ __forceinline__ float operator()(float z) const { return ex2(arg(z)); }
  // a sum against reference r, against this reference instead
  __device__ __forceinline__ float join(float r, float s) const {
    if (r == -INFINITY) return s;  // nothing yet: 0 (or NaN, which stays)
    const Expo w(c2, r);
    // how much of a power of two r lies above m; against a far reference no whole number
    const float up = w.far ? arg(r) : far ? -w.arg(m) : w.M2 - M2;
    return s * ex2(up);
  }
};

// Sets an element of a vector to -infinity: it adds nothing to a sum.
template <typename T>
__device__ __forceinline__ void blank(uint4& v, int element) {
  const uint32_t none = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00u : 0xff80u;
  const int at = element * (int)sizeof(T), shift = (at % 4) * 8;
  const uint32_t mask = sizeof(T) == 4 ? 0xffffffffu : 0xffffu << shift;
  auto put = [&](uint32_t& w, int i) { w = at / 4 == i ? (w & ~mask) | (none << shift) : w; };
  put(v.x, 0);
  put(v.y, 1);
  put(v.z, 2);
  put(v.w, 3);
}
// Largest element of a vector and ref; NaN gives way.
template <typename T>
__device__ __forceinline__ float max_of(const uint4& raw, float ref) {
  float o[Elem<T>::N];
  Elem<T>::unpack(raw, o);
#pragma unroll
  for (int i = 0; i < Elem<T>::N; ++i) ref = fmaxf(ref, o[i]);
  return ref;
}
// A row's sum leaves out the token that the outputs are about (the chosen token, the teacher's
// entry of largest logit): its own term joins in 64 bits, so that ln q = -log(1 + rest / own)
// and 1 - q = rest / (own + rest) keep their digits where q is near 1, and ln q is never above 0.
//
// The other terms are formed 2^kShift smaller, so that their arguments stay below 0 for values
// up to 20 tau above the reference (beyond, the reference moves): there the hardware
// exponential's mean error is one number (measured: -5.0e-8 relative over [-9, 0), -5.1e-8 down
// to -25; +3.3e-8 above 0), which is taken out of each row's sum in 64 bits. Left in, it adds up
// over a sequence's tokens while the other errors average out. It is a mean over arguments with
// spread fractions: in a row of equal logits (or at a temperature that makes them equal) it may
// itself be the error, below half a rounding of the row's log-probability. A shift of 10 moves
// the reference of rows with a few large logits: 576 instead of 493 us for 4096 x 151936 with 30
// logits of 8 to 20 in each row. An argument near -30 is rounded by 2^-20: where a few terms
// have a row's weight they lie above the reference, with smaller arguments; where many have it,
// their roundings average out.
constexpr float kShift = 30.f, kShiftUp = 1073741824.f;
// What a thread's sum of shifted terms may grow to before its reference moves: 512 terms (what a
// ring of kMaxSlots holds for a thread) near the reference are below 2^(9.5 - kShift); one with
// an argument above 0 is not below 1.
constexpr float kMostSum = 1.f;
constexpr double kExpMeanError = -5.05e-8;
// What the fast form z c2 + R adds for reference m: NaN (or infinity) where the sum has to
// take the careful form.
__device__ __forceinline__ float reference(float m, C2 c2) {
  const Expo w(c2, m);
  return m == -INFINITY ? INFINITY : w.far ? __int_as_float(0x7fffffff) : -w.M2 - kShift;
}

// The careful forms of the two passes over n vectors `step` apart in shared memory: a sum
// whose reference moves, and a vector of a gradient with another phase, at a row's ends, or of
// a row with a far reference. Out of line: they are rare, and inline they cost the usual path.
template <typename T>
__device__ __noinline__ float2 careful_sum(const uint4* v, int n, int step, C2 c2, float ref, float sum) {
  float m = ref;
  for (int k = 0; k < n; ++k) m = max_of<T>(v[k * step], m);
  const Expo w(c2, m == -INFINITY ? 0.f : m);
  sum = w.join(ref, sum);
  for (int k = 0; k < n; ++k) {
    float o[Elem<T>::N];
    Elem<T>::unpack(v[k * step], o);
#pragma unroll
    for (int i = 0; i < Elem<T>::N; ++i) sum += ex2(w.arg(o[i]) - kShift);
  }
  return make_float2(m, sum);
}
template <typename T>
__device__ __noinline__ void careful_store(const uint4* v, T* row, int V, int64_t e0, C2 c2, float m, float As) {
  constexpr int N = Elem<T>::N;
  const Expo w(c2, m);
  const RowVec<T> g(row, V);
  float o[N];
  Elem<T>::unpack(*v, o);
#pragma unroll
  for (int i = 0; i < N; ++i) o[i] = As * w(o[i]);
  g.store(e0, o);
}
// Bounded waits, out of line. The usual one sleeps in the barrier (polls of a waiting warp take
// issue slots from the working ones); the exchange of a row's sums, where every cycle
// counts, polls.
__device__ __noinline__ bool wait_asleep(uint64_t* bar, uint32_t parity, volatile int* abort, uint64_t limit_ns) {
  const uint64_t t0 = globaltimer_ns();
  for (;;) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(20000u)  // ns
        : "memory");
    if (ok) return true;
    if (*abort) return false;
    if (globaltimer_ns() - t0 > limit_ns) {
      *abort = 1;
      return false;
    }
  }
}
__device__ __noinline__ bool wait_awake(uint64_t* bar, uint32_t parity, volatile int* abort, uint64_t limit_ns) {
  return mbar_wait_bounded(bar, parity, abort, nullptr, limit_ns);
}

// ------------------------------------------------------------------------------------
// The sparse side of a row. One token per row (policy, log-probability) or K entries of a
// teacher in shared memory (distillation). What a row's outputs need is left in a RowRecord;
// a second kernel forms the outputs of all rows at once, in 64 bits.
// ------------------------------------------------------------------------------------
// A row's part in the loss. Bad: an id outside the vocabulary, which turns the row's
// outputs into NaN (and is never used as an index).
enum RowState : int { kRowOff = 0, kRowOn = 1, kRowBad = 2 };

struct RowRecord {
  double base;    // distillation: sum P (ln P - (z - zref) / tau)
  float m, rest;  // the row's reference, and its sum of exponentials without the token's
  float z;        // the token's logit; distillation: zref
  float weight;   // distillation: sum P
  int state;
  int id;         // the token; distillation: the first id with zref, -1 where no entry has a
                  // logit above -infinity (zref is 0 then, and the sum complete)
};
static_assert(sizeof(RowRecord) == kRowRecordBytes, "scratch size");

struct Entries {
  int* id;    // -1: not an entry
  float* p;   // weight, after the teacher's logit
  float* z;   // the row's logit at id
  int K4;     // entries, up to a multiple of 4 (those past K are none)
};
constexpr int kEntryBytes = 12;
__host__ __device__ inline int entries_padded(int K) { return (K + 3) / 4 * 4; }
__device__ __forceinline__ Entries entries_at(void* smem, int K) {
  const int K4 = entries_padded(K);
  float* f = reinterpret_cast<float*>(smem);
  return {reinterpret_cast<int*>(f), f + K4, f + 2 * K4, K4};
}
// The weight at an id: the sum over all entries with it, in their order (so equal ids get
// the same bits).
__device__ __forceinline__ float weight_of(const Entries& s, int id) {
  float P = 0.f;
  for (int j = 0; j < s.K4; j += 4) {
    const int4 i = *reinterpret_cast<const int4*>(s.id + j);
    const float4 p = *reinterpret_cast<const float4*>(s.p + j);
    P += i.x == id ? p.x : 0.f;
    P += i.y == id ? p.y : 0.f;
    P += i.z == id ? p.z : 0.f;
    P += i.w == id ? p.w : 0.f;
  }
  return P;
}

// What the sum and the gradient take from one token (distillation: the id and zref of the
// record).
struct Token {
  int state, id;
  float z, adv, old_logp, ref_logp;  // z: its logit
};

template <typename T, int OP>
__device__ __forceinline__ Token load_token(const VocabLossArgs& a, int t, const T* row) {
  const int64_t id = load_id(a.labels, t, a.ids64);
  bool on = id >= 0;
  if (OP == kOpLogp && a.offsets) on = on && t >= a.offsets[0] && t < a.offsets[a.num_seq];
  Token k = {!on ? kRowOff : id < a.V ? kRowOn : kRowBad, 0, 0.f, 0.f, 0.f, 0.f};
  if (on) {
    k.id = k.state == kRowOn ? (int)id : 0;
    k.z = Elem<T>::f(row[k.id]);
    if constexpr (OP == kOpPolicy) {
      k.adv = a.adv[t];
      k.old_logp = a.old_logp[t];
      k.ref_logp = a.ref_logp ? a.ref_logp[t] : 0.f;
    }
  }
  return k;
}

// Fills the teacher entries of row t from one warp and returns the row's state; lane 0 has
// the record's sparse half in *rec.
template <typename T>
__device__ __forceinline__ int load_entries(const VocabLossArgs& a, int t, const T* row, const Entries& s, int lane,
                                            RowRecord* rec) {
  const int K = a.K;
  float top = -INFINITY;
  bool any = false, bad = false;
  if (lane < s.K4 - K) {
    s.id[K + lane] = -1;
    s.p[K + lane] = 0.f;
  }
  for (int k = lane; k < K; k += 32) {
    const int64_t id = load_id(a.ids, (int64_t)t * K + k, a.ids64);
    const float v = a.teacher[(int64_t)t * K + k];
    const bool has = id >= 0 && v != -INFINITY;
    any |= has;
    bad |= has && id >= a.V;
    s.id[k] = has ? (int)(id < a.V ? id : 0) : -1;
    s.p[k] = v;
    if (has) top = fmaxf(top, v);
  }
  if (!__any_sync(0xffffffffu, any)) return rec->state = kRowOff;
  bad = __any_sync(0xffffffffu, bad);
  top = warp_max(top);
  float sum = 0.f, zref = -INFINITY;
  for (int k = lane; k < K; k += 32) {
    const int id = s.id[k];
    const float z = id >= 0 ? Elem<T>::f(row[id]) : 0.f;
    s.z[k] = z;
    if (id >= 0) {
      sum += expf((s.p[k] - top) / a.tau);
      zref = fmaxf(zref, z);
    }
  }
  const float lsum = logf(warp_sum(sum));
  zref = warp_max(zref);
  int first = 0x7fffffff;  // the lowest id with zref
  for (int k = lane; k < K; k += 32)
    if (s.id[k] >= 0 && s.z[k] == zref) first = min(first, s.id[k]);
  first = __reduce_min_sync(0xffffffffu, first);
  if (zref == -INFINITY) {
    zref = 0.f;
    first = -1;
  }
  double base = 0.0;
  float weight = 0.f;
  for (int k = lane; k < K; k += 32) {
    const bool has = s.id[k] >= 0;
    const float lp = has ? (s.p[k] - top) / a.tau - lsum : 0.f;
    const float P = has ? expf(lp) : 0.f;
    s.p[k] = P;
    if (P != 0.f) {  // P (ln P - (z - zref) / tau)
      base += (double)P * ((double)lp - ((double)s.z[k] - (double)zref) / a.tau64);
      weight += P;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) base += __shfl_xor_sync(0xffffffffu, base, o);
  rec->base = base;
  rec->weight = warp_sum(weight);
  rec->z = zref;
  rec->id = first;
  rec->state = bad ? kRowBad : kRowOn;
  __syncwarp();
  return rec->state;
}

// The policy loss of one token from r = pi / pi_old and d = ln (pi_ref / pi).
struct PolicyTerm {
  float loss, dl, kl;  // dl = d loss / d logp
};
__device__ __forceinline__ PolicyTerm policy_term(const VocabLossArgs& a, float A, float r, float d, bool has_ref) {
  // an advantage of 0 asks for nothing, also where the ratio overflows
  const float u = A == 0.f ? 0.f : r * A;
  const float v = A == 0.f ? 0.f : fminf(fmaxf(r, 1.f - a.clip_low), 1.f + a.clip_high) * A;
  PolicyTerm o;
  o.loss = -(u <= v ? u : v);
  o.dl = u <= v ? -u : 0.f;
  o.kl = 0.f;
  if (r != r) o.loss = o.dl = r;  // the clamp drops NaN
  if (has_ref) {
    const float em = expm1f(d);
    o.kl = em - d;
    if (a.kl_coef != 0.f) {
      o.loss += a.kl_coef * o.kl;
      o.dl -= a.kl_coef * em;
    }
  }
  return o;
}

// d (up * loss) / d (sum over rows)
__device__ __forceinline__ float loss_factor(const VocabLossArgs& a) {
  return (a.count ? 1.f / (float)max(*a.count, 1) : a.host_scale) * (a.up ? *a.up : 1.f);
}

// ln q of a token with logit z from the row's reference and the sum of the other terms (apart
// false: of all terms). Formed in 64 bits: in fp32 the rounding of ln(sum) near 12 alone is
// 5e-7, and a sequence's log-ratio sums hundreds.
__device__ __noinline__ double row_logp(C2 c2, float z, float m, float rest, bool apart) {
  const Expo x(c2, m);
  const double c = (double)c2.hi + (double)c2.lo;
  const double arg = x.far ? ((double)z - (double)m) * c : (double)z * c - (double)x.M2;  // the token's own term is 2^arg
  const double r = (double)rest * (1.0 - kExpMeanError), own = apart ? exp2(arg) : 0.0;
  return r < own ? -log1p(r / own) : arg * 0.69314718055994530942 - log(r + own);
}

// The same to fp32's accuracy (a 64-bit logarithm here would delay every row by 1000 cycles:
// 427 us instead of 397 us for 4096 x 151936). The policy loss and its gradient both take the
// ratio, and so their side of the clip, from these bits.
__device__ __forceinline__ double quick_logp(C2 c2, float z, float m, float rest) {
  const Expo x(c2, m);
  const float own = x(z);
  if (rest < own) return -log1pf(rest / own);
  const double c = (double)c2.hi + (double)c2.lo;
  const double arg = x.far ? ((double)z - (double)m) * c : (double)z * c - (double)x.M2;
  int e;
  const float f = frexpf(rest + own, &e);  // what is left is the logarithm of a number in [1/2, 1)
  return (arg - e) * 0.69314718055994530942 - logf(f);
}

// The factor A of the gradient A (q - P) of a row in the loss, from the row's reference and the
// sum of the other tokens' terms; g: loss_factor.
template <int OP>
__device__ __forceinline__ float row_factor(const VocabLossArgs& a, const Token& k, float m, float rest, float g) {
  if (k.state == kRowBad) return __int_as_float(0x7fffffff);
  if constexpr (OP == kOpLogp) return -1.f;
  if constexpr (OP == kOpDistill) return a.tau * g;
  const double lp = quick_logp(C2{a.c2, a.c2_hi, a.c2_lo}, k.z, m, rest);
  return -policy_term(a, k.adv, expf((float)(lp - (double)k.old_logp)), (float)((double)k.ref_logp - lp),
                      a.ref_logp != nullptr).dl / a.tau * g;
}

// Rows longer than a cluster's shared memory: one block per row, which reads the row for its
// maximum, and again (from L2 where it fits) for the sum and for the gradient.
template <typename T, int OP>
__global__ void __launch_bounds__(512) vocab_row_kernel(const VocabLossArgs a) {
  constexpr int N = Elem<T>::N;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float red[32];
  __shared__ Token s_token;
  const int t = blockIdx.x, lane = threadIdx.x & 31;
  const Entries s = entries_at(smem, a.K);
  const RowVec<T> z(const_cast<T*>(reinterpret_cast<const T*>(a.z)) + (int64_t)t * a.z_stride, a.V);
  const RowVec<T> g(reinterpret_cast<T*>(a.grad) + (a.grad ? (int64_t)t * a.grad_stride : 0), a.V);
  RowRecord* rec = reinterpret_cast<RowRecord*>(a.records) + t;
  if (threadIdx.x < 32) {
    RowRecord r = {};
    Token k = {};
    if constexpr (OP == kOpDistill) {
      k.state = load_entries(a, t, z.p, s, lane, &r);
      k.id = r.id;
      k.z = r.z;
    } else {
      k = load_token<T, OP>(a, t, z.p);
      r.z = k.z;
      r.state = k.state;
      r.id = k.id;
    }
    if (lane == 0) {
      s_token = k;
      *rec = r;
      if (t == 0) *a.ticket = 0;
    }
  }
  __syncthreads();
  const Token k = s_token;
  if (k.state == kRowOff) {
    if (a.grad) {
      const float o[N] = {};
      for (int j = threadIdx.x; j < z.nv; j += blockDim.x) g.store(z.first(j), o);
    }
    return;
  }
  float mx = -INFINITY, rest = 0.f;
  for (int j = threadIdx.x; j < z.nv; j += blockDim.x) {
    float o[N];
    Elem<T>::unpack(z.load(j), o);
#pragma unroll
    for (int i = 0; i < N; ++i) mx = fmaxf(mx, o[i]);
  }
  const Expo x(C2{a.c2, a.c2_hi, a.c2_lo}, block_max(mx, red));
  for (int j = threadIdx.x; j < z.nv; j += blockDim.x) {
    float o[N];
    Elem<T>::unpack(z.load(j), o);
    const int64_t own = (int64_t)k.id - z.first(j);
#pragma unroll
    for (int i = 0; i < N; ++i) rest += i == own ? 0.f : ex2(x.arg(o[i]) - kShift);
  }
  rest = block_sum(rest, red) * kShiftUp;
  if (x.m == -INFINITY) rest = __int_as_float(0x7fffffff);  // no finite logit: no softmax
  if (threadIdx.x == 0) {
    rec->m = x.m;
    rec->rest = rest;
  }
  if (!a.grad) return;
  const float A = row_factor<OP>(a, k, x.m, rest, loss_factor(a));
  const float As = A / (k.id >= 0 ? rest + x(k.z) : rest);
  for (int j = threadIdx.x; j < z.nv; j += blockDim.x) {
    float o[N];
    Elem<T>::unpack(z.load(j), o);
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = As * x(o[i]);
    g.store(z.first(j), o);
  }
  __syncthreads();
  if constexpr (OP == kOpDistill) {
    for (int i = threadIdx.x; i < a.K; i += blockDim.x)
      if (s.id[i] >= 0) g.p[s.id[i]] = Elem<T>::t(As * x(s.z[i]) - A * weight_of(s, s.id[i]));
  } else {
    if (threadIdx.x == 0) g.p[k.id] = Elem<T>::t(-As * rest);  // A (q - 1)
  }
}

// ------------------------------------------------------------------------------------
// Streaming kernel. A cluster of C blocks takes a row: each block streams its part of the row
// once from memory into a ring of pieces in shared memory, forms the partial sum as the
// pieces arrive, exchanges it with the other blocks, and writes the gradient from the pieces,
// which frees them for the next row. So every logit is read from memory once, and loads,
// arithmetic and stores of neighbouring rows overlap.
//   first CW warps  sum and gradient: thread i owns vectors i, i + 32 CW, .. of every piece
//   load warp       bulk copies of whole vectors; the partial vectors at a row's ends, and the
//                   token's without the token, come from the prepare warp
//   prepare warp    tokens (8 rows at a time) or teacher entries of the rows to come
//   join warp       the row's sum from all warps' parts and the factor of its gradient;
//                   distillation: the gradient at the entries' ids, once the block's dense part
//                   is written (a single token is set by the thread that owns its vector)
// Partial sums travel as (reference, sum) pairs of each warp, with asynchronous stores that
// complete on the receiver's mbarrier. Pair buffers alternate: a warp sends row r + 2 after it
// has row r + 1 of every warp, and each of those left after its block had all of row r.
// Every wait is bounded; one that runs out turns the outputs of all the cluster's rows,
// gradients among them, and with them the loss, into NaN.
//
// What bounds it: memory would take 380 us for 4096 x 151936 bf16 with gradients (2.5 GB at
// 6.55 TB/s); measured 490-516 us, 4.8-5.1 TB/s, with every byte moved once (a capture of 1024
// rows reads 313 MB and writes 311 MB, the last 58 MB of it still in L2). The two
// exponentials per logit keep the special-function unit 55% busy and the schedulers 49%: the
// consumers' own latencies (a wait costs ~120 cycles, a row's exchange of sums ~2500, hidden
// behind the next row's first pieces) set the pace, not memory. The forward alone: 270 us,
// 4.6 TB/s. Other shapes, measured when these rows took 484-502 us: 8 x 4 vectors 545 us, 24 or
// 28 warps 600-654 us (more waits for the same work), clusters of 4 blocks 990 us with one block
// and 569 us with two blocks per SM, pieces held in registers instead of the ring 575-641 us.
// ------------------------------------------------------------------------------------
constexpr int kMaxSlots = 32, kMaxCluster = 8, kMaxConsumers = 16;

// CW consumer warps, VPT vectors per thread and piece, B blocks per SM
template <int CW_, int VPT_, int B_>
struct StreamCfg {
  static constexpr int CW = CW_, VPT = VPT_, B = B_;
  static constexpr int Threads = (CW + 3) * 32;
  static constexpr int Lanes = CW * 32;  // vectors between a thread's own
  static constexpr int PieceVecs = Lanes * VPT, PieceBytes = PieceVecs * 16;
};

constexpr int kTokens = 16;  // rows between the prepare warp and the others (tokens)

struct StreamShared {
  uint64_t full[kMaxSlots], empty[kMaxSlots];
  uint64_t ent_full[kTokens], ent_done[kTokens], dense_done[kTokens];
  uint64_t pairs_full[2], factor_full[2];
  // a row's first and last vector, where they are partial, and the token's, where it is neither
  // of those; without the token
  uint4 edge[kTokens][3];
  Token token[kTokens];
  float factor[2][4];  // A, A / sum, reference, sum without the token
  float2 pairs[2][kMaxCluster * kMaxConsumers];
  int abort;
};

// The row's reference and the sum of all warps' pairs (one warp; the same bits in each). z: the
// logit of the token that the pairs leave out (none: -infinity).
__device__ __forceinline__ void join_pairs(const float2* pairs, int n, C2 c2, float z, int lane, float* m, float* rest) {
  float mx = z, v = 0.f;
  for (int i = lane; i < n; i += 32) mx = fmaxf(mx, pairs[i].x);
  mx = warp_max(mx);
  const Expo x(c2, mx);
  for (int i = lane; i < n; i += 32) v += x.join(pairs[i].x, pairs[i].y);
  v = warp_sum(v);
  // a row without a finite logit has no softmax
  *rest = mx == -INFINITY ? __int_as_float(0x7fffffff) : v;
  *m = mx;
}

template <typename T, int OP, typename Cfg>
__global__ void __launch_bounds__(Cfg::Threads, Cfg::B) vocab_stream_kernel(const VocabLossArgs a, int C, int slots,
                                                                            int rows_ahead) {
  constexpr int N = Elem<T>::N, CW = Cfg::CW, kPieceVecs = Cfg::PieceVecs, kPieceBytes = Cfg::PieceBytes;
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ StreamShared sh;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* ent_mem = ring + (size_t)slots * kPieceBytes;
  auto entries = [&](int e) { return entries_at(ent_mem + (size_t)e * entries_padded(a.K) * kEntryBytes, a.K); };
  const int rank = (int)(blockIdx.x % (unsigned)C);
  const int cluster = (int)(blockIdx.x / (unsigned)C), clusters = (int)(gridDim.x / (unsigned)C);
  volatile int* abort = &sh.abort;

  if (threadIdx.x == 0) {
    for (int i = 0; i < slots; ++i) {
      mbar_init(&sh.full[i], 1);
      mbar_init(&sh.empty[i], CW);
    }
    for (int i = 0; i < rows_ahead; ++i) {
      mbar_init(&sh.ent_full[i], 1);
      // the load and join warps, and the consumers (distillation: the join warp after them)
      mbar_init(&sh.ent_done[i], OP == kOpDistill ? 2 : CW + 2);
      mbar_init(&sh.dense_done[i], CW);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.pairs_full[i], C == 1 ? CW : 1);
      mbar_init(&sh.factor_full[i], 1);
    }
    sh.abort = 0;
    fence_barrier_init();
    if (blockIdx.x == 0) *a.ticket = 0;  // for the kernel that forms the outputs
  }
  __syncthreads();
  if (C > 1) cluster_sync();  // the other blocks' barriers are ready too
  // all lanes of a warp, with one answer
  auto wait = [&](uint64_t* bar, int phase) {
    const uint32_t parity = (uint32_t)phase & 1u;
    return __all_sync(0xffffffffu, mbar_try_wait(bar, parity)) ||
           __all_sync(0xffffffffu, wait_asleep(bar, parity, abort, a.wait_ns));
  };
  auto wait_exchange = [&](uint64_t* bar, int phase) {
    const uint32_t parity = (uint32_t)phase & 1u;
    return __all_sync(0xffffffffu, mbar_try_wait(bar, parity)) ||
           __all_sync(0xffffffffu, wait_awake(bar, parity, abort, a.wait_ns));
  };
  const int log2c = 31 - __clz(C);
  // this block's vectors of row t
  auto row_z = [&](int t) {
    return RowVec<T>(const_cast<T*>(reinterpret_cast<const T*>(a.z)) + (int64_t)t * a.z_stride, a.V);
  };
  auto part = [&](const RowVec<T>& z, int* j0, int* j1) {
    const int per = (z.nv + C - 1) >> log2c;  // C is a power of two
    *j0 = min(rank * per, z.nv);
    *j1 = min(*j0 + per, z.nv);
  };
  // the vector that an element is in
  auto vec_of = [](const RowVec<T>& z, int id) { return (int)(((int64_t)id + z.a) / N); };
  // edge i of entry e: a row's first or last vector, if partial, or the token's, without the token
  auto prepare_vec = [&](const RowVec<T>& z, int id, int e, int i) {
    const int own = id >= 0 ? vec_of(z, id) : -1;
    const int j = i == 0 ? 0 : i == 1 ? z.nv - 1 : own;
    if (j < 0 || z.full(j) != (i == 2)) return;
    uint4 v = z.load(j);
    if (j == own) blank<T>(v, (int)(((int64_t)id + z.a) % N));
    sh.edge[e][i] = v;
  };
  // position in the ring of rows: entry e, in its lap's phase
  auto next_entry = [&](int& e, int& lap) {
    if (++e == rows_ahead) {
      e = 0;
      lap ^= 1;
    }
  };

  if (warp == CW) {
    // ------------------------------- loads -------------------------------
    int slot = 0, turn = 0, e = 0, lap = 0;
    bool ok = true;
    for (int t = cluster; t < a.T && ok; t += clusters) {
      if (!wait(&sh.ent_full[e], lap)) break;
      if (sh.token[e].state != kRowOff) {
        const RowVec<T> z = row_z(t);
        int j0, j1;
        part(z, &j0, &j1);
        const int f0 = z.full(0) ? 0 : 1, f1 = z.full(z.nv - 1) ? z.nv : z.nv - 1;  // whole vectors
        const int id = sh.token[e].id, own = id >= 0 ? vec_of(z, id) : -1;
        for (int p = j0; p < j1; p += kPieceVecs) {
          const int q = min(p + kPieceVecs, j1);
          if (!wait(&sh.empty[slot], turn ^ 1)) { ok = false; break; }
          if (lane == 0) {
            uint4* dst = reinterpret_cast<uint4*>(ring + (size_t)slot * kPieceBytes);
            const bool head = p < f0, tail = q > f1;
            if (head) dst[0] = sh.edge[e][0];
            if (tail && z.nv - 1 >= f0) dst[z.nv - 1 - p] = sh.edge[e][1];
            const int b0 = max(p, f0), b1 = min(q, f1);
            const bool cut = own >= b0 && own < b1;
            if (cut) dst[own - p] = sh.edge[e][2];
            if (head || tail || cut) fence_proxy_async_smem();  // before a later bulk copy into the slot
            const int c0 = cut ? own : b1, c1 = cut ? own + 1 : b1;  // copied: b0 .. c0 and c1 .. b1
            const int n = b1 - b0 - (cut ? 1 : 0);
            if (n > 0) {
              mbar_arrive_expect_tx(&sh.full[slot], (uint32_t)n * 16u);
              if (c0 > b0) bulk_load(dst + (b0 - p), z.p + z.first(b0), (uint32_t)(c0 - b0) * 16u, &sh.full[slot]);
              if (b1 > c1) bulk_load(dst + (c1 - p), z.p + z.first(c1), (uint32_t)(b1 - c1) * 16u, &sh.full[slot]);
            } else {
              mbar_arrive(&sh.full[slot]);
            }
          }
          __syncwarp();
          if (++slot == slots) {
            slot = 0;
            turn ^= 1;
          }
        }
      }
      if (lane == 0) mbar_arrive(&sh.ent_done[e]);
      __syncwarp();
      next_entry(e, lap);
    }
  } else if (warp == CW + 1) {
    // ------------------------------ prepare ------------------------------
    RowRecord* recs = reinterpret_cast<RowRecord*>(a.records);
    if constexpr (OP == kOpDistill) {
      int e = 0, lap = 0;
      for (int t = cluster; t < a.T; t += clusters) {
        const RowVec<T> z = row_z(t);
        if (t == a.stall_row && rank == 0) break;
        if (!wait(&sh.ent_done[e], lap ^ 1)) break;
        RowRecord r = {};
        const int state = load_entries(a, t, z.p, entries(e), lane, &r);
        if (state != kRowOff && lane < 3) prepare_vec(z, r.id, e, lane);
        __syncwarp();
        if (lane == 0) {
          sh.token[e].state = state;
          sh.token[e].id = r.id;
          sh.token[e].z = r.z;
          if (rank == 0) {  // not the consumer's half
            recs[t].base = r.base;
            recs[t].z = r.z;
            recs[t].weight = r.weight;
            recs[t].state = state;
            recs[t].id = r.id;
          }
          mbar_arrive(&sh.ent_full[e]);
        }
        __syncwarp();
        next_entry(e, lap);
      }
    } else {
      // lane i takes row i of each group of 8; two groups alternate, so one is prepared
      // while the other is worked on
      for (int g0 = 0;; g0 += kTokens / 2) {
        const int64_t t = (int64_t)cluster + (int64_t)(g0 + lane) * clusters;
        const bool mine = lane < kTokens / 2 && t < a.T;
        if (!__any_sync(0xffffffffu, mine)) break;
        const int e = (g0 + lane) % kTokens;
        bool ok = true;
        if (mine) ok = wait_asleep(&sh.ent_done[e], (uint32_t)(((g0 + lane) / kTokens) & 1) ^ 1u, abort, a.wait_ns);
        if (!__all_sync(0xffffffffu, ok)) break;
        if (mine && !(t == a.stall_row && rank == 0)) {
          const RowVec<T> z = row_z((int)t);
          const Token k = load_token<T, OP>(a, (int)t, z.p);
          if (k.state != kRowOff)
#pragma unroll
            for (int i = 0; i < 3; ++i) prepare_vec(z, k.id, e, i);
          sh.token[e] = k;
          if (rank == 0) {
            recs[t].z = k.z;
            recs[t].state = k.state;
            recs[t].id = k.id;
          }
          mbar_arrive(&sh.ent_full[e]);
        }
        __syncwarp();
      }
    }
  } else if (warp == CW + 2) {
    // ---------------------------- join and fix ----------------------------
    const float factor = loss_factor(a);
    int e = 0, lap = 0, x = 0;
    for (int t = cluster; t < a.T; t += clusters) {
      if (!wait(&sh.ent_full[e], lap)) break;
      const Token token = sh.token[e];
      float m = 0.f, A = 0.f, As = 0.f;
      if (token.state != kRowOff) {
        if (C > 1 && lane == 0) mbar_arrive_expect_tx(&sh.pairs_full[x & 1], (uint32_t)(C * CW) * 8u);
        __syncwarp();
        if (!wait_exchange(&sh.pairs_full[x & 1], x >> 1)) break;
        const C2 c2 = {a.c2, a.c2_hi, a.c2_lo};
        const bool apart = token.id >= 0;
        float rest;
        join_pairs(sh.pairs[x & 1], C * CW, c2, apart ? token.z : -INFINITY, lane, &m, &rest);
        if (a.grad) {
          A = row_factor<OP>(a, token, m, rest, factor);
          As = A / (apart ? rest + Expo(c2, m)(token.z) : rest);
        }
        if (lane == 0) {
          sh.factor[x & 1][0] = A;
          sh.factor[x & 1][1] = As;
          sh.factor[x & 1][2] = m;
          sh.factor[x & 1][3] = rest;
          mbar_arrive(&sh.factor_full[x & 1]);
          if (rank == 0) {
            RowRecord* rec = reinterpret_cast<RowRecord*>(a.records) + t;
            rec->m = m;
            rec->rest = rest;
          }
        }
        ++x;
      }
      if constexpr (OP == kOpDistill) {
        if (!wait(&sh.dense_done[e], lap)) break;
        if (a.grad && token.state != kRowOff) {  // the entries' values replace the dense ones
          const Expo w(C2{a.c2, a.c2_hi, a.c2_lo}, m);
          const Entries s = entries(e);
          const RowVec<T> z = row_z(t);
          int j0, j1;
          part(z, &j0, &j1);
          const int64_t e0 = z.first(j0), e1 = z.first(j1);
          T* g = reinterpret_cast<T*>(a.grad) + (int64_t)t * a.grad_stride;
          for (int k = lane; k < a.K; k += 32)
            if (s.id[k] >= 0 && s.id[k] >= e0 && s.id[k] < e1)
              g[s.id[k]] = Elem<T>::t(As * w(s.z[k]) - A * weight_of(s, s.id[k]));
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.ent_done[e]);
      __syncwarp();
      next_entry(e, lap);
    }
  } else {
    // ---------------------------- sum and gradient ----------------------------
    // A row's sum is complete some 2500 cycles before its factor is back from the other
    // warps and blocks: meanwhile the sum of the next row begins, over the pieces that are
    // there already.
    constexpr int kAhead = 3;  // the first piece and a pair
    const int tid = threadIdx.x;
    uint4 none;  // a vector of -infinity
    {
      float o[N];
#pragma unroll
      for (int i = 0; i < N; ++i) o[i] = -INFINITY;
      none = Elem<T>::pack(o);
    }
    const C2 c2 = {a.c2, a.c2_hi, a.c2_lo};
    const F2 ch = f2(a.c2_hi, a.c2_hi), cl = f2(a.c2_lo, a.c2_lo);
    auto piece_at = [&](int sl) { return reinterpret_cast<const uint4*>(ring + (size_t)sl * kPieceBytes) + tid; };
    int slot = 0, turn = 0, grad_slot = 0, e = 0, lap = 0, x = 0;
    // the row that is summed: done of np pieces
    int t = cluster, np = 0, done = 0, part_n = 0;
    bool open = false;
    float ref = -INFINITY, sum = 0.f;
    F2 nR2 = f2(0.f, 0.f);
    // the row that waits for its factor
    int tg = -1, eg = 0;
    for (;;) {
      while (!open && t < a.T) {
        if (tg >= 0) {
          // a row's gradient is still owed, and the entries to come may wait for its own
          if (!__all_sync(0xffffffffu, mbar_test_wait(&sh.ent_full[e], (uint32_t)lap))) break;
        } else if (!wait(&sh.ent_full[e], lap)) {
          goto out;
        }
        const RowVec<T> z = row_z(t);
        int j0, j1;
        part(z, &j0, &j1);
        if (sh.token[e].state != kRowOff) {
          open = true;
          part_n = j1 - j0;
          np = (part_n + kPieceVecs - 1) / kPieceVecs;
          done = 0;
          ref = -INFINITY;
          sum = 0.f;
          break;
        }
        if (a.grad) {
          const RowVec<T> g(reinterpret_cast<T*>(a.grad) + (int64_t)t * a.grad_stride, a.V);
          const float o[N] = {};
          for (int j = j0 + tid; j < j1; j += Cfg::Lanes) g.store(z.first(j), o);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(OP == kOpDistill ? &sh.dense_done[e] : &sh.ent_done[e]);
        next_entry(e, lap);
        t += clusters;
      }
      if (open) {
        // Sum against a reference that is the maximum of the warp's first vectors: the usual
        // vector takes no maximum, and the reference rarely moves.
        const int stop = tg >= 0 ? min(np, done + kAhead) : np;
        auto there = [&](int sl, int tn) {  // a row's gradient is owed: do not wait
          return __all_sync(0xffffffffu, mbar_test_wait(&sh.full[sl], (uint32_t)tn)) != 0;
        };
        auto add_vec = [&](const uint4& raw, F2 (&acc)[2]) {
          float o[N];
          Elem<T>::unpack(raw, o);
#pragma unroll
          for (int i = 0; i < N; i += 2) {
            const F2 z2 = f2(o[i], o[i + 1]);
            acc[(i >> 1) & 1] = add2(acc[(i >> 1) & 1], ex2_2(arg2(z2, ch, cl, nR2)));
          }
        };
        auto total = [&](F2 (&acc)[2]) {
          float ax, ay;
          split(add2(acc[0], acc[1]), ax, ay);
          return sum + (ax + ay);
        };
        auto add_carefully = [&](const uint4* piece, int n, bool first) {
          const float2 r = careful_sum<T>(piece, n, Cfg::Lanes, c2, first ? -INFINITY : ref, sum);
          ref = r.x;
          sum = r.y;
          const float R = reference(ref, c2);
          nR2 = f2(R, R);
        };
        auto next_slot = [&] {
          if (!a.grad) {
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.empty[slot]);
          }
          if (++slot == slots) {
            slot = 0;
            turn ^= 1;
          }
        };
        while (done < stop) {
          if (tg >= 0) {
            if (!there(slot, turn)) break;
          } else if (!wait(&sh.full[slot], turn)) {
            goto out;
          }
          const int end = part_n - done * kPieceVecs;                // vectors left
          const uint4* piece = piece_at(slot);
          // After the first piece two whole ones at a time, for more arithmetic between the
          // waits. Where the sum is split depends on the place in the row alone, never on
          // what has arrived: the same bits on every run.
          if (done > 0 && end >= 2 * kPieceVecs) {
            const int slot1 = slot + 1 == slots ? 0 : slot + 1, turn1 = slot + 1 == slots ? turn ^ 1 : turn;
            if (tg >= 0) {
              if (!there(slot1, turn1)) break;
            } else if (!wait(&sh.full[slot1], turn1)) {
              goto out;
            }
            const uint4* piece1 = piece_at(slot1);
            uint4 raw[2 * Cfg::VPT];
#pragma unroll
            for (int v = 0; v < Cfg::VPT; ++v) {
              raw[v] = piece[v * Cfg::Lanes];
              raw[Cfg::VPT + v] = piece1[v * Cfg::Lanes];
            }
            F2 acc[2] = {f2(0.f, 0.f), f2(0.f, 0.f)};
#pragma unroll
            for (int v = 0; v < 2 * Cfg::VPT; ++v) add_vec(raw[v], acc);
            const float s1 = total(acc);
            if (s1 <= kMostSum) {
              sum = s1;
            } else {  // NaN too
              add_carefully(piece, Cfg::VPT, false);
              add_carefully(piece1, Cfg::VPT, false);
            }
            done += 2;
            next_slot();
            next_slot();
            continue;
          }
          const int left = (end - tid + Cfg::Lanes - 1) / Cfg::Lanes;  // this thread's vectors (or < 1)
          uint4 raw[Cfg::VPT];
          if (end >= kPieceVecs) {
#pragma unroll
            for (int v = 0; v < Cfg::VPT; ++v) raw[v] = piece[v * Cfg::Lanes];
          } else {  // the last piece, partly filled
#pragma unroll
            for (int v = 0; v < Cfg::VPT; ++v) raw[v] = v < left ? piece[v * Cfg::Lanes] : none;
          }
          if (done == 0) {
#pragma unroll
            for (int v = 0; v < Cfg::VPT; ++v) ref = max_of<T>(raw[v], ref);
            ref = warp_max(ref);
            const float R = reference(ref, c2);
            nR2 = f2(R, R);
          }
          F2 acc[2] = {f2(0.f, 0.f), f2(0.f, 0.f)};
#pragma unroll
          for (int v = 0; v < Cfg::VPT; ++v) {
            if (v > 0 && end <= v * Cfg::Lanes) break;  // nothing left for any thread
            add_vec(raw[v], acc);
          }
          const float s1 = total(acc);
          if (s1 <= kMostSum) sum = s1;
          else if (left > 0) add_carefully(piece, min(left, Cfg::VPT), done == 0);  // NaN too
          ++done;
          next_slot();
        }
      }
      if (tg >= 0) {
        const int xg = x - 1;
        if (!wait_exchange(&sh.factor_full[xg & 1], xg >> 1)) goto out;
        const float As = sh.factor[xg & 1][1], m = sh.factor[xg & 1][2];
        const Expo w(c2, m);
        const RowVec<T> z = row_z(tg);
        const RowVec<T> g(reinterpret_cast<T*>(a.grad) + (int64_t)tg * a.grad_stride, a.V);
        int j0, j1;
        part(z, &j0, &j1);
        const F2 nM2 = f2(-w.M2, -w.M2), As2 = f2(As, As);
        const bool plain = g.a == z.a && !w.far;
        // whole vectors of this part: pieces within them take the straight path
        const int lo = z.full(0) ? 0 : 1, hi = z.full(z.nv - 1) ? z.nv : z.nv - 1;
        T* gp = g.p + z.first(j0 + tid);
        auto grad_vec = [&](const uint4& raw, T* to) {
          float o[N];
          Elem<T>::unpack(raw, o);
#pragma unroll
          for (int i = 0; i < N; i += 2)
            split(mul2(As2, ex2_2(arg2(f2(o[i], o[i + 1]), ch, cl, nM2))), o[i], o[i + 1]);
          *reinterpret_cast<uint4*>(to) = Elem<T>::pack(o);
        };
        auto free_slot = [&] {
          if (lane == 0) mbar_arrive(&sh.empty[grad_slot]);
          if (++grad_slot == slots) grad_slot = 0;
        };
        const int inner = plain ? min(hi, j1) : 0;
        for (int base = j0; base < j1;) {
          const uint4* piece = piece_at(grad_slot);
          if (base >= lo && base + 2 * kPieceVecs <= inner) {
            const uint4* piece1 = piece_at(grad_slot + 1 == slots ? 0 : grad_slot + 1);
            uint4 raw[2 * Cfg::VPT];
#pragma unroll
            for (int v = 0; v < Cfg::VPT; ++v) {
              raw[v] = piece[v * Cfg::Lanes];
              raw[Cfg::VPT + v] = piece1[v * Cfg::Lanes];
            }
#pragma unroll
            for (int v = 0; v < 2 * Cfg::VPT; ++v) grad_vec(raw[v], gp + v * Cfg::Lanes * N);
            __syncwarp();
            free_slot();
            free_slot();
            base += 2 * kPieceVecs;
            gp += 2 * kPieceVecs * N;
            continue;
          }
          if (base >= lo && base + kPieceVecs <= inner) {
            uint4 raw[Cfg::VPT];
#pragma unroll
            for (int v = 0; v < Cfg::VPT; ++v) raw[v] = piece[v * Cfg::Lanes];
#pragma unroll
            for (int v = 0; v < Cfg::VPT; ++v) grad_vec(raw[v], gp + v * Cfg::Lanes * N);
          } else {  // a row's end in this piece, another phase, or a far reference
#pragma unroll 1
            for (int v = 0; v < Cfg::VPT; ++v) {
              const int j = base + tid + v * Cfg::Lanes;
              if (j >= j1) break;
              if (plain && j >= lo && j < hi) grad_vec(piece[v * Cfg::Lanes], gp + v * Cfg::Lanes * N);
              else careful_store<T>(piece + v * Cfg::Lanes, g.p, a.V, z.first(j), c2, m, As);
            }
          }
          __syncwarp();
          free_slot();
          base += kPieceVecs;
          gp += kPieceVecs * N;
        }
        if constexpr (OP != kOpDistill) {  // the token's element, from the thread that wrote its vector
          const Token token = sh.token[eg];
          const int own = (int)(((int64_t)token.id + z.a) / N) - j0;
          if (own >= 0 && own < j1 - j0 && own % Cfg::Lanes == tid)
            g.p[token.id] = Elem<T>::t(-As * sh.factor[xg & 1][3]);  // A (q - 1)
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(OP == kOpDistill ? &sh.dense_done[eg] : &sh.ent_done[eg]);
        tg = -1;
        continue;
      }
      if (!open) break;
      // Without a gradient nothing else makes a warp wait for the row before: a pair of row x
      // may only leave once this block has joined row x - 1.
      if (!a.grad && x > 0 && !wait(&sh.factor_full[(x - 1) & 1], (x - 1) >> 1)) goto out;
      const float mw = warp_max(ref);
      sum = warp_sum(Expo(c2, mw).join(ref, sum * kShiftUp));
      if (C == 1) {
        if (lane == 0) {
          sh.pairs[x & 1][warp] = make_float2(mw, sum);
          mbar_arrive(&sh.pairs_full[x & 1]);
        }
      } else if (lane < C) {
        const uint32_t to = mapa_shared(smem_u32(&sh.pairs[x & 1][rank * CW + warp]), (uint32_t)lane);
        const uint32_t bar = mapa_shared(smem_u32(&sh.pairs_full[x & 1]), (uint32_t)lane);
        st_async_f2(to, mw, sum, bar);
      }
      __syncwarp();
      if (a.grad) {
        tg = t;
        eg = e;
      } else if (lane == 0) {
        mbar_arrive(OP == kOpDistill ? &sh.dense_done[e] : &sh.ent_done[e]);
      }
      ++x;
      next_entry(e, lap);
      t += clusters;
      open = false;
    }
  out:;
  }
  __syncthreads();
  if (C > 1) {
    // a row is lost to all blocks of the cluster where one has given up
    if (*abort && threadIdx.x < (unsigned)C) st_cluster_u32(mapa_shared(smem_u32(&sh.abort), threadIdx.x), 1u);
    cluster_sync();  // no block leaves while another may still write to it
  }
  if (*abort) {
    const uint64_t t0 = globaltimer_ns();  // copies and pairs in flight land long before this
    while (globaltimer_ns() - t0 < 1000000) {
    }
    RowRecord* recs = reinterpret_cast<RowRecord*>(a.records);
    float o[N];
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = __int_as_float(0x7fffffff);
    for (int t = cluster; t < a.T; t += clusters) {
      if (threadIdx.x == 0) recs[t].state = kRowBad;
      if (a.grad) {  // what it holds may be the logits, or nothing yet
        const RowVec<T> z = row_z(t), g(reinterpret_cast<T*>(a.grad) + (int64_t)t * a.grad_stride, a.V);
        int j0, j1;
        part(z, &j0, &j1);
        for (int j = j0 + (int)threadIdx.x; j < j1; j += Cfg::Threads) g.store(z.first(j), o);
      }
    }
  }
}

// Outputs of all rows from their records, one thread per row, and the loss as the sum over
// rows in 64 bits: blocks leave partial sums, the last one adds them in their order, so the
// loss has the same bits on every run.
constexpr int kFinishThreads = 256;
template <int OP>
__global__ void __launch_bounds__(kFinishThreads) vocab_finish_kernel(const VocabLossArgs a) {
  __shared__ double red[32];
  __shared__ bool last;
  const int t = blockIdx.x * kFinishThreads + threadIdx.x;
  const float nan = __int_as_float(0x7fffffff);
  float loss = 0.f;
  if (t < a.T) {
    const RowRecord r = reinterpret_cast<const RowRecord*>(a.records)[t];
    const C2 c2 = {a.c2, a.c2_hi, a.c2_lo};
    double lp = 0.0;  // ln q of the token (of the entry that zref is from)
    if (r.state == kRowOn) lp = row_logp(c2, r.z, r.m, r.rest, r.id >= 0);
    if constexpr (OP == kOpDistill) {
      if (r.state == kRowOn) loss = (float)((double)a.tau * a.tau * (r.base - (double)r.weight * lp));
      else if (r.state == kRowBad) loss = nan;
    } else {
      const bool on = r.state != kRowOff;
      if (r.state == kRowBad) lp = (double)nan;
      a.logp[t] = (float)lp;
      if constexpr (OP == kOpLogp) {
        if (a.lse) {
          reinterpret_cast<float2*>(a.lse)[t] = on ? make_float2(r.m, r.rest + Expo(c2, r.m)(r.z)) : make_float2(0.f, 0.f);
          a.rest[t] = on ? r.rest : 0.f;
        }
        if (a.ratio) {
          a.ratio[t] = on ? (float)(lp - (double)a.ref_logp[t]) : 0.f;
          a.row_coef[t] = 0.f;  // rows of no pair keep it
        }
      } else {
        PolicyTerm o = {0.f, 0.f, 0.f};
        const double quick = r.state == kRowOn ? quick_logp(c2, r.z, r.m, r.rest) : lp;
        if (on)
          o = policy_term(a, a.adv[t], expf((float)(quick - (double)a.old_logp[t])),
                          a.ref_logp ? (float)((double)a.ref_logp[t] - lp) : 0.f, a.ref_logp != nullptr);
        loss = o.loss;
        a.kl[t] = o.kl;
      }
    }
  }
  if constexpr (OP != kOpLogp) {
    const double v = block_sum_d((double)loss, red);
    if (threadIdx.x == 0) {
      a.partial[blockIdx.x] = v;
      __threadfence();
      last = atomicAdd(a.ticket, 1u) == gridDim.x - 1;
    }
    __syncthreads();
    if (last) {
      __threadfence();
      double s = 0.0;
      for (int b = threadIdx.x; b < (int)gridDim.x; b += kFinishThreads) s += __ldcg(a.partial + b);
      s = block_sum_d(s, red);
      if (threadIdx.x == 0) *a.loss = (float)(a.count ? s / max(*a.count, 1) : s * (double)a.host_scale);
    }
  }
}

// ------------------------------------------------------------------------------------
// rows in the loss, sums over rows, scaling
// ------------------------------------------------------------------------------------
// One block: all labels, a load of several per thread in flight.
__global__ void __launch_bounds__(1024) count_labels_kernel(const void* labels, bool is64, int T, int* count) {
  __shared__ int red[32];
  int n = 0;
#pragma unroll 8
  for (int t = threadIdx.x; t < T; t += 1024) n += load_id(labels, t, is64) >= 0;
  n = __reduce_add_sync(0xffffffffu, n);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = n;
  __syncthreads();
  if (threadIdx.x < 32) {
    n = __reduce_add_sync(0xffffffffu, red[threadIdx.x]);
    if (threadIdx.x == 0) *count = n;
  }
}
// A warp per row. One block writes the count itself; several add to it (it is zeroed before;
// whole numbers, so their order does not matter).
__global__ void __launch_bounds__(1024) count_teacher_kernel(const void* ids, bool is64, const float* teacher, int T,
                                                             int K, int* count) {
  __shared__ int red[32];
  const int lane = threadIdx.x & 31;
  const int warps = gridDim.x * 32;
  int n = 0;
  for (int t = (blockIdx.x * 1024 + threadIdx.x) >> 5; t < T; t += warps) {
    bool any = false;
    for (int k = lane; k < K && !any; k += 32)
      any = load_id(ids, (int64_t)t * K + k, is64) >= 0 && teacher[(int64_t)t * K + k] != -INFINITY;
    n += __any_sync(0xffffffffu, any) ? 1 : 0;
  }
  if (lane == 0) red[threadIdx.x >> 5] = n;
  __syncthreads();
  if (threadIdx.x < 32) {
    n = __reduce_add_sync(0xffffffffu, red[threadIdx.x]);
    if (threadIdx.x == 0) {
      if (gridDim.x == 1) *count = n;
      else atomicAdd(count, n);
    }
  }
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
// One block per pair. Log-ratios, each rounded once from 64 bits, are summed in 64 bits: the margin is the difference of
// two sums over whole sequences.
__global__ void __launch_bounds__(256) preference_pairs_kernel(const PreferenceArgs a) {
  __shared__ double red[32];
  __shared__ bool last;
  const int i = blockIdx.x;
  int lo[2], hi[2];
  double R[2];
  for (int s = 0; s < 2; ++s) {  // offsets are clamped: a wrong one reads no other memory
    lo[s] = min(max(a.offsets[2 * i + s], 0), a.T);
    hi[s] = min(max(a.offsets[2 * i + s + 1], 0), a.T);
    double v = 0.0;
    for (int t = lo[s] + threadIdx.x; t < hi[s]; t += blockDim.x)
      v += (double)a.ratio[t];  // 0 where there is no label
    R[s] = (double)a.beta * block_sum_d(v, red);
  }
  const double m = R[0] - R[1], e = exp(-fabs(m));
  const double sp = log1p(e);  // softplus(-|m|)
  const double neg = m > 0 ? sp : sp - m, pos = m > 0 ? sp + m : sp;  // softplus(-m), softplus(m)
  const double sig_neg = m > 0 ? e / (1.0 + e) : 1.0 / (1.0 + e), sig_pos = 1.0 - sig_neg;
  const double dm = ((double)a.eps * sig_pos - (1.0 - (double)a.eps) * sig_neg) / a.pairs;
  for (int s = 0; s < 2; ++s) {
    const float c = (float)((s ? -dm : dm) * (double)a.beta);
    for (int t = lo[s] + threadIdx.x; t < hi[s]; t += blockDim.x)
      if (load_id(a.labels, t, a.ids64) >= 0) a.row_coef[t] = c;
  }
  // the mean over pairs: the last block adds them in their order
  if (threadIdx.x == 0) {
    a.rewards[2 * i] = (float)R[0];
    a.rewards[2 * i + 1] = (float)R[1];
    a.partial[i] = (1.0 - (double)a.eps) * neg + (double)a.eps * pos;
    __threadfence();
    last = atomicAdd(a.ticket, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  double v = 0.0;
  for (int p = threadIdx.x; p < a.pairs; p += blockDim.x) v += __ldcg(a.partial + p);
  v = block_sum_d(v, red);
  if (threadIdx.x == 0) *a.loss = (float)(v / a.pairs);
}

// dz = up * row_coef * (onehot - softmax) from the saved reference and sum: one read, one
// write. Rows go from the last to the first: the forward has just read the last ones, and
// what of them is still in L2 is not fetched again (the gradient is written around it).
// Bound by memory: 377 us for 4096 x 151936 bf16, 6.6 TB/s, as fast as a copy.
constexpr int kGradThreads = 256, kGradVecs = 4, kGradChunk = 2 * kGradThreads * kGradVecs;
template <typename T>
__global__ void __launch_bounds__(kGradThreads) preference_grad_kernel(const VocabLossArgs a,
                                                                       const float* __restrict__ row_coef, int chunks) {
  constexpr int N = Elem<T>::N;
  const int t = a.T - 1 - (int)(blockIdx.x / (unsigned)chunks), c = (int)(blockIdx.x % (unsigned)chunks);
  const int tid = threadIdx.x;
  const RowVec<T> z(const_cast<T*>(reinterpret_cast<const T*>(a.z)) + (int64_t)t * a.z_stride, a.V);
  const RowVec<T> g(reinterpret_cast<T*>(a.grad) + (int64_t)t * a.grad_stride, a.V);
  const int j0 = c * kGradChunk, j1 = min(j0 + kGradChunk, z.nv);
  const int64_t label = load_id(a.labels, t, a.ids64);
  const float coef = row_coef[t];
  const float2 l = reinterpret_cast<const float2*>(a.lse)[t];
  // rows outside the loss are not read: their logits may hold anything
  const bool on = label >= 0 && t >= a.offsets[0] && t < a.offsets[a.num_seq];
  // whole vectors at the same phase take the straight path
  const bool same = g.a == z.a;
  const int lo = z.full(0) ? 0 : 1, hi = z.full(z.nv - 1) ? z.nv : z.nv - 1;
  if (!on) {
    const float o[N] = {};
    for (int j = j0 + tid; j < j1; j += kGradThreads) {
      if (same && j >= lo && j < hi) __stcs(reinterpret_cast<uint4*>(g.p + z.first(j)), make_uint4(0, 0, 0, 0));
      else g.store(z.first(j), o);
    }
    return;
  }
  const float A = -coef * *a.up, As = A / l.y;
  const C2 c2 = {a.c2, a.c2_hi, a.c2_lo};
  const Expo x(c2, l.x);
  const bool plain = same && !x.far;
  const F2 ch = f2(a.c2_hi, a.c2_hi), cl = f2(a.c2_lo, a.c2_lo), nM2 = f2(-x.M2, -x.M2), As2 = f2(As, As);
  for (int base = j0; base < j1; base += kGradThreads * kGradVecs) {
    uint4 raw[kGradVecs];
#pragma unroll
    for (int v = 0; v < kGradVecs; ++v) {
      const int j = base + v * kGradThreads + tid;
      if (j >= lo && j < min(hi, j1)) raw[v] = __ldg(reinterpret_cast<const uint4*>(z.p + z.first(j)));
    }
#pragma unroll
    for (int v = 0; v < kGradVecs; ++v) {
      const int j = base + v * kGradThreads + tid;
      if (j >= j1) break;
      if (plain && j >= lo && j < hi) {
        float o[N];
        Elem<T>::unpack(raw[v], o);
#pragma unroll
        for (int i = 0; i < N; i += 2)
          split(mul2(As2, ex2_2(arg2(f2(o[i], o[i + 1]), ch, cl, nM2))), o[i], o[i + 1]);
        __stcs(reinterpret_cast<uint4*>(g.p + z.first(j)), Elem<T>::pack(o));
      } else {
        const uint4 r = z.load(j);
        careful_store<T>(&r, g.p, a.V, z.first(j), c2, l.x, As);
      }
    }
  }
  // the label's element, from the thread that wrote its vector
  if (label < a.V) {
    const int own = (int)((label + z.a) / N) - j0;
    if (own >= 0 && own < j1 - j0 && own % kGradThreads == tid)
      g.p[label] = Elem<T>::t(-As * a.rest[t]);  // A (q - 1)
  }
}

// Dynamic shared memory of a block, beside its static part and the system's 1 KB.
template <typename Cfg>
constexpr int stream_smem() {
  return (228 * 1024 / Cfg::B - 1024 - (int)sizeof(StreamShared) - 256) & ~127;
}

template <typename Cfg>
void stream_config(cudaLaunchConfig_t* cfg, cudaLaunchAttribute* at, int blocks, int C, int smem, cudaStream_t st) {
  cfg->gridDim = dim3((unsigned)blocks);
  cfg->blockDim = dim3(Cfg::Threads);
  cfg->dynamicSmemBytes = (size_t)smem;
  cfg->stream = st;
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)C;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg->attrs = at;
  cfg->numAttrs = 1;
}

// Clusters of C blocks that fit on the device at once, per kernel and device.
template <typename T, int OP, typename Cfg>
int resident_clusters(int C, int smem) {
  static std::mutex mu;
  static std::map<std::array<int, 3>, int> known;
  int dev = 0;
  cudaGetDevice(&dev);
  const std::lock_guard<std::mutex> lock(mu);
  int& n = known[{dev, C, smem}];
  if (!n) {
    auto kernel = vocab_stream_kernel<T, OP, Cfg>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, stream_smem<Cfg>());
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at[1];
    stream_config<Cfg>(&cfg, at, C, C, smem, nullptr);
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveClusters(&n, kernel, &cfg);
    if (e != cudaSuccess || n < 1) {
      n = 0;
      throw std::runtime_error(std::string("vocab_loss: ") + (e != cudaSuccess ? cudaGetErrorString(e) : "no room for a cluster"));
    }
  }
  return n;
}

template <typename Cfg>
int stream_slots(int ent) { return std::min(kMaxSlots, (stream_smem<Cfg>() - ent) / Cfg::PieceBytes); }
template <typename Cfg>
int stream_pieces(int nv, int C) { return ((nv + C - 1) / C + Cfg::PieceVecs - 1) / Cfg::PieceVecs; }

template <typename T, int OP, typename Cfg>
void launch_stream(const VocabLossArgs& a, int C, int rows_ahead, int ent, cudaStream_t st) {
  const int slots = stream_slots<Cfg>(ent);
  const int smem = slots * Cfg::PieceBytes + ent;
  const int clusters = std::min(a.T, resident_clusters<T, OP, Cfg>(C, smem));
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[1];
  stream_config<Cfg>(&cfg, at, clusters * C, C, smem, st);
  cudaError_t e = cudaLaunchKernelEx(&cfg, vocab_stream_kernel<T, OP, Cfg>, a, C, slots, rows_ahead);
  if (e != cudaSuccess) throw std::runtime_error(std::string("vocab_loss: ") + cudaGetErrorString(e));
  check_launch("vocab_loss");
}

// One block of 16 warps per SM, or more and smaller blocks. What a row costs beside its
// vectors (waits, the exchange of sums: some 3000 cycles) overlaps between the blocks of an
// SM, so short rows want many small blocks and long ones the whole ring. Policy loss with its
// gradient, us on a B200, for 1 / 2 / 4 / 8 blocks per SM: 4096 x 32001 bf16 156 / 137 / - / -;
// 16384 x 8000 301 / 214 / 167 / -; 16384 x 4096 273 / 161 / 115 / 115; 60000 x 1000
// 874 / 500 / 295 / 245 (-: the row does not fit).
using CfgBig = StreamCfg<16, 2, 1>;
using CfgMid = StreamCfg<8, 2, 2>;
using CfgSmall = StreamCfg<4, 2, 4>;
using CfgTiny = StreamCfg<2, 2, 8>;

// Whether rows of nv vectors take Cfg: one block holds a row and a part of the next one, and
// there are more rows than blocks of the next larger kind.
template <typename Cfg>
bool stream_fits(int nv, int T, int ent, int num_sms) {
  const int slots = stream_slots<Cfg>(ent);
  return (int64_t)T > (int64_t)num_sms * (Cfg::B / 2) && stream_pieces<Cfg>(nv, 1) <= slots - slots / 4;
}

template <typename T, int OP>
void launch_op(const VocabLossArgs& a, int num_sms, cudaStream_t st) {
  constexpr int N = Elem<T>::N;
  const int nv = (int)(((int64_t)a.V + 2 * N - 2) / N);  // vectors of a row at its worst phase
  // distillation: entries of 4 rows, of 2 where they would take the ring's room
  const int rows_ahead = OP != kOpDistill ? kTokens : a.K <= 256 ? 4 : 2;
  const int ent = OP == kOpDistill ? rows_ahead * entries_padded(a.K) * kEntryBytes : 0;
  if (stream_fits<CfgTiny>(nv, a.T, ent, num_sms)) return launch_stream<T, OP, CfgTiny>(a, 1, rows_ahead, ent, st);
  if (stream_fits<CfgSmall>(nv, a.T, ent, num_sms)) return launch_stream<T, OP, CfgSmall>(a, 1, rows_ahead, ent, st);
  if (stream_fits<CfgMid>(nv, a.T, ent, num_sms)) return launch_stream<T, OP, CfgMid>(a, 1, rows_ahead, ent, st);
  // Blocks per row: as many as it takes for the row to stay in shared memory, and more
  // while that leaves SMs without a row.
  int C = 1;
  const int slots = stream_slots<CfgBig>(ent);
  while (C < kMaxCluster && (stream_pieces<CfgBig>(nv, C) > slots ||
                             (stream_pieces<CfgBig>(nv, C) > 1 && (int64_t)a.T * C * 2 <= num_sms)))
    C *= 2;
  if (stream_pieces<CfgBig>(nv, C) <= slots) return launch_stream<T, OP, CfgBig>(a, C, rows_ahead, ent, st);
  vocab_row_kernel<T, OP><<<a.T, 512, OP == kOpDistill ? entries_padded(a.K) * kEntryBytes : 16, st>>>(a);
  check_launch("vocab_loss");
}

template <typename T>
void launch_rows(const VocabLossArgs& a, int op, int num_sms, cudaStream_t st) {
  const int blocks = vocab_finish_blocks(a.T);
  if (op == kOpDistill) {
    launch_op<T, kOpDistill>(a, num_sms, st);
    vocab_finish_kernel<kOpDistill><<<blocks, kFinishThreads, 0, st>>>(a);
  } else if (op == kOpPolicy) {
    launch_op<T, kOpPolicy>(a, num_sms, st);
    vocab_finish_kernel<kOpPolicy><<<blocks, kFinishThreads, 0, st>>>(a);
  } else {
    launch_op<T, kOpLogp>(a, num_sms, st);
    vocab_finish_kernel<kOpLogp><<<blocks, kFinishThreads, 0, st>>>(a);
  }
  check_launch("vocab_finish");
}

}  // namespace

void vocab_count_rows(const VocabLossArgs& a, int op, int* count, cudaStream_t st) {
  if (a.T <= 0) return;
  if (op == kOpDistill) {
    // a block of 32 rows at a time costs about 1.5 us per turn: more than 4 turns are split
    const int blocks = a.T <= 128 ? 1 : std::min((a.T + 31) / 32, 148);
    if (blocks > 1) cudaMemsetAsync(count, 0, sizeof(int), st);
    count_teacher_kernel<<<blocks, 1024, 0, st>>>(a.ids, a.ids64, a.teacher, a.T, a.K, count);
  } else {
    count_labels_kernel<<<1, 1024, 0, st>>>(a.labels, a.ids64, a.T, count);
  }
  check_launch("vocab_count_rows");
}

int vocab_finish_blocks(int T) { return (T + kFinishThreads - 1) / kFinishThreads; }

void vocab_loss(const VocabLossArgs& a, int op, int num_sms, cudaStream_t st) {
  if (a.T <= 0) {  // a loss over nothing
    if (a.loss) cudaMemsetAsync(a.loss, 0, sizeof(float), st);
    return;
  }
  if (a.V < 1) throw std::runtime_error("vocab_loss: empty vocabulary");
  if (op == kOpDistill && (a.K < 1 || a.K > kMaxTeacher)) throw std::runtime_error("vocab_loss: teacher entries");
  if (a.dtype == kVocabBf16) launch_rows<__nv_bfloat16>(a, op, num_sms, st);
  else if (a.dtype == kVocabF16) launch_rows<__half>(a, op, num_sms, st);
  else launch_rows<float>(a, op, num_sms, st);
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
  if (a.pairs <= 0) {  // a loss over nothing
    cudaMemsetAsync(a.loss, 0, sizeof(float), st);
    return;
  }
  preference_pairs_kernel<<<a.pairs, 256, 0, st>>>(a);
  check_launch("preference_pairs");
}

void preference_grad(const VocabLossArgs& a, const float* row_coef, cudaStream_t st) {
  if (a.T <= 0) return;
  const int n = a.dtype == kVocabF32 ? 4 : 8;
  const int nv = (int)(((int64_t)a.V + 2 * n - 2) / n);  // vectors of a row at its worst phase
  const int chunks = (nv + kGradChunk - 1) / kGradChunk;
  const int64_t blocks = (int64_t)a.T * chunks;
  if (blocks > 0x7fffffff) throw std::runtime_error("preference_grad: too many rows");
  if (a.dtype == kVocabBf16)
    preference_grad_kernel<__nv_bfloat16><<<(int)blocks, kGradThreads, 0, st>>>(a, row_coef, chunks);
  else if (a.dtype == kVocabF16)
    preference_grad_kernel<__half><<<(int)blocks, kGradThreads, 0, st>>>(a, row_coef, chunks);
  else preference_grad_kernel<float><<<(int)blocks, kGradThreads, 0, st>>>(a, row_coef, chunks);
  check_launch("preference_grad");
}

}  // namespace sepx
