// Losses on logits and their gradients (sm_100a): log-probabilities of given labels, a preference loss over pairs of
// sequences, a clipped policy loss with a KL term.
//
//   S = sum_v exp(x_v - M), M the row's maximum     logp = (x[label] - M) - log S (0 where the label is the ignored one)
//   dx_v = w (onehot_v - exp(x_v - M) / S)          with w = dloss / dlogp of the row
//   preference: L_i = sum_t logp_it, reward_i = beta (L_i - ref_i), h = reward_chosen - reward_rejected,
//               loss = mean over pairs of -(1 - s) logsigmoid(h) - s logsigmoid(-h);
//               w_chosen = beta / P (s sigmoid(h) - (1 - s) sigmoid(-h)) = -w_rejected
//   policy:     rho = exp(logp - old), q = clamp(rho, 1 - low, 1 + high) A, d = ref - logp, n = rows with a label,
//               loss = 1/n sum(-min(rho A, q) + k (exp(d) - d - 1)); w = (-[rho A <= q] rho A + k (1 - exp(d))) / n
//
// A row of logits is read once with a running maximum and sum per thread, the group's are joined at the end: fp32, base
// 2, the maximum subtracted before the product with log2 e, so that rows of the type's lowest value give no infinity.
// The maximum starts at the lowest finite number, not at -inf: a row of -inf then ends with a sum of 0, and is NaN.
// M and log2 S go from the forward to the backward pass apart: added up, log S would be lost beside a maximum of 1e9 (a row of
// one mask value) and off by 5e-4 beside one of 1e4, and with it all of the row's gradient.
// A row belongs to a warp or to a CTA of 128 to 512 threads, by its length and the number of rows (group_of).
// The policy loss's w depends on its own row alone, so its kernel writes the row's gradient right behind the sum, while
// the row is in L2: HBM sees each row once, up to the length that policy_rows tells.  The preference loss has to see both sequences first; its backward takes the
// rows in the opposite order, so that the last ones read are still in L2.
#include <cfloat>
#include <type_traits>

#include "common.cuh"
#include "nvfp4_b200.h"

namespace nvfp4 {
namespace logprob {

constexpr int kThreads = 256;                     // of the CTAs whose rows belong to warps, and of those that add up
// log2 e in two parts: alone, the first is off by 1.3e-8 of itself, which moves every term of a row the same way, and the sum
// of a sequence's thousand log-probabilities shows it.  ex2.approx falls short by 5e-8 on average (torch.exp is 6e-9 too large); of a
// log-probability of 13 to 150000 normal logits with a spread of 1 to 4 this leaves 2e-8 or less, in 4096 to 16384 rows, where fp32 torch
// operations are off by 1e-8 to 4e-8.
constexpr float kLog2e = 1.4426950408889634f, kLog2eRest = 1.925963e-8f;

struct Rows {
  const void* x;
  int64_t stride_b, stride_t;     // in elements; the logits of a row are contiguous
  int64_t rows;                   // batch * seq
  uint32_t seq, vocab;
  const int64_t* labels;          // [rows]
  int64_t ignore;
};
// Running maximum and sum of exp(x - maximum), s + c.  A row of 150000 logits whose spread is 4 has most of its terms under 2^-24 of
// its sum.  Added to that one by one they round away: 4e-7 of the sum, in one direction, for every row of a sequence.  So 16 or 32 terms
// are added up by themselves, and c takes what their sum loses beside s, exactly (Dekker 1971, the larger of the two first): 5e-9.  16384
// rows of 50257 bf16 take the 290 us that they took without it; with s in 64 bits 298.
struct Stat {
  float m, s, c;
};
using Norm = nvfp4_row_stat;                      // what a row's probabilities take: its maximum and the base-2 logarithm of that sum

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float exp_of(float d) { return ex2(fmaf(d, kLog2e, d * kLog2eRest)); }
__device__ __forceinline__ float2 both(float a) { return make_float2(a, a); }
// the same of two, in packed instructions
__device__ __forceinline__ float2 exp_of(float2 d) {
  const float2 t = __ffma2_rn(d, both(kLog2e), __fmul2_rn(d, both(kLog2eRest)));
  return make_float2(ex2(t.x), ex2(t.y));
}
// exp(d) / S within 1.3e-8 d of itself: enough for a gradient.  less: -log2 S
__device__ __forceinline__ float exp_near(float d, float less) { return ex2(fmaf(d, kLog2e, less)); }
__device__ __forceinline__ float2 exp_near(float2 d, float2 less) {
  const float2 t = __ffma2_rn(d, both(kLog2e), less);
  return make_float2(ex2(t.x), ex2(t.y));
}
// max(m, a, b) as one three-input instruction (a NaN does not count; it shows in the sum)
__device__ __forceinline__ float max3(float m, float a, float b) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(m), "f"(a), "f"(b));
  return r;
}
// log s.  The sum's exponent is taken off in front of the logarithm, whose own rounding is then far below that of an fp32
// result.  (Beside a coarse maximum, logf(s) would leave every other result halfway between two fp32 numbers.)
__device__ __forceinline__ double log_of(float s) {
  const int k = min(max((int)(__float_as_uint(s) >> 23) - 127, 0), 63);          // s is 1 to 2^31, or 0, or no number
  const float f = s * __uint_as_float((uint32_t)(127 - k) << 23);
  return k * 0.69314718055994531 + (double)logf(f);
}
__device__ __forceinline__ Norm norm_of(Stat st, double log_s) { return Norm{st.m, (float)(log_s * 1.4426950408889634)}; }

// A 16-byte vector of logits as pairs of fp32, and back.
template <class T> struct Vec;
template <> struct Vec<float> {
  static constexpr int n = 4;
  static __device__ __forceinline__ void open(const uint4& q, float2* v) {
    v[0] = make_float2(__uint_as_float(q.x), __uint_as_float(q.y));
    v[1] = make_float2(__uint_as_float(q.z), __uint_as_float(q.w));
  }
  static __device__ __forceinline__ uint4 close(const float2* v) {
    return make_uint4(__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x), __float_as_uint(v[1].y));
  }
};
__device__ __forceinline__ uint32_t pack(float2 a) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a.x, a.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <> struct Vec<__nv_bfloat16> {
  static constexpr int n = 8;
  static __device__ __forceinline__ void open(const uint4& q, float2* v) {
    v[0] = make_float2(bf16_lo(q.x), bf16_hi(q.x));
    v[1] = make_float2(bf16_lo(q.y), bf16_hi(q.y));
    v[2] = make_float2(bf16_lo(q.z), bf16_hi(q.z));
    v[3] = make_float2(bf16_lo(q.w), bf16_hi(q.w));
  }
  static __device__ __forceinline__ uint4 close(const float2* v) { return make_uint4(pack(v[0]), pack(v[1]), pack(v[2]), pack(v[3])); }
};
__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// elements in front of the first 16-byte boundary
template <class T> __device__ __forceinline__ uint32_t lead(const T* p, uint32_t n) {
  const uint32_t h = (uint32_t)((16u - (reinterpret_cast<uintptr_t>(p) & 15u)) & 15u) / sizeof(T);
  return h < n ? h : n;
}

// ---- reading a row -----------------------------------------------------------------------------------------------------
__device__ __forceinline__ void take(Stat& st, float m, float sum) {         // sum: of exp(x - m), m not below st.m
  if (m > st.m) {
    const float by = expf(st.m - m);
    st.s *= by;
    st.c *= by;
  }
  const float big = fmaxf(st.s, sum), t = st.s + sum;
  st = Stat{m, t, st.c + (fminf(st.s, sum) - (t - big))};
}
__device__ __forceinline__ void take(Stat& st, float x) {
  const float m = fmaxf(st.m, x);
  take(st, m, exp_of(x - m));
}
template <int N> __device__ __forceinline__ void take(Stat& st, const float2 (&v)[N]) {
  float m = st.m, m1 = -FLT_MAX;
#pragma unroll
  for (int j = 0; j < N; j += 2) {
    m = max3(m, v[j].x, v[j].y);
    m1 = max3(m1, v[j + 1].x, v[j + 1].y);
  }
  m = fmaxf(m, m1);
  const float2 below = both(-m);
  float2 s = exp_of(__fadd2_rn(v[0], below)), s1 = exp_of(__fadd2_rn(v[1], below));
#pragma unroll
  for (int j = 2; j < N; j += 2) {
    s = __fadd2_rn(s, exp_of(__fadd2_rn(v[j], below)));
    s1 = __fadd2_rn(s1, exp_of(__fadd2_rn(v[j + 1], below)));
  }
  s = __fadd2_rn(s, s1);
  take(st, m, s.x + s.y);
}

// Maximum and sum of this thread's part of a row; GROUP threads share the row.  Four vectors of a thread are in flight while
// it works on the four before.
template <class T, int GROUP> __device__ __forceinline__ Stat scan(const T* x, uint32_t n, uint32_t tid) {
  constexpr int V = Vec<T>::n, UNROLL = 4;
  Stat st{-FLT_MAX, 0.0f, 0.0f};
  const uint32_t head = lead(x, n), vecs = (n - head) / V, tail = head + vecs * V;
  const uint4* q = reinterpret_cast<const uint4*>(x + head) + tid;
  // (vectors behind the row's last are not loaded; they count as -inf)
  uint4 ahead[UNROLL];
  auto load = [&](uint32_t i) {
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
      if (i + u * GROUP < vecs) ahead[u] = __ldg(q + (i - tid) + u * GROUP);
  };
  load(tid);
  if (tid < head) take(st, as_float(x[tid]));
  if (tail + tid < n) take(st, as_float(x[tail + tid]));
  for (uint32_t i = tid; i < vecs; i += UNROLL * GROUP) {
    uint4 w[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) w[u] = ahead[u];
    load(i + UNROLL * GROUP);
    if (i + (UNROLL - 1) * GROUP < vecs) {
      float2 v[UNROLL * V / 2];
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) Vec<T>::open(w[u], v + u * (V / 2));
      take(st, v);
    } else {
#pragma unroll
      for (int u = 0; u < UNROLL; ++u)
        if (i + u * GROUP < vecs) {
          float2 v[V / 2];
          Vec<T>::open(w[u], v);
          take(st, v);
        }
    }
  }
  return st;
}
// The group's maximum and sum, the same bits in every thread (a butterfly of plain sums is symmetric).
template <int GROUP> __device__ __forceinline__ Stat join_group(Stat st) {
  float m = st.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  float s = (st.s + st.c) * expf(st.m - m);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (GROUP > 32) {
    __shared__ Stat part[GROUP / 32];
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = Stat{m, s, 0.0f};
    __syncthreads();
#pragma unroll
    for (int w = 0; w < GROUP / 32; ++w) m = fmaxf(m, part[w].m);
    s = 0.0f;
#pragma unroll
    for (int w = 0; w < GROUP / 32; ++w) s += part[w].s * expf(part[w].m - m);
  }
  return Stat{m, s, 0.0f};
}

// ---- writing a row of the gradient --------------------------------------------------------------------------------------
template <class T, int GROUP> __device__ __forceinline__ void clear_row(T* out, uint32_t n, uint32_t tid) {
  constexpr int V = Vec<T>::n;
  const uint32_t head = lead(out, n), vecs = (n - head) / V, tail = head + vecs * V;
  for (uint32_t i = tid; i < head; i += GROUP) out[i] = from_float<T>(0.0f);
  uint4* q = reinterpret_cast<uint4*>(out + head);
  for (uint32_t i = tid; i < vecs; i += GROUP) q[i] = make_uint4(0u, 0u, 0u, 0u);
  for (uint32_t j = tail + tid; j < n; j += GROUP) out[j] = from_float<T>(0.0f);
}
// out = w (onehot - exp(x - M) / S); w = 0 gives zeros unless the row holds something that is no number
template <class T> struct GradRow {
  static constexpr int V = Vec<T>::n;
  Norm norm;
  float w;
  uint32_t label;
  __device__ __forceinline__ GradRow(Norm norm_, float w_, uint32_t label_) : norm(norm_), w(w_), label(label_) {}
  __device__ __forceinline__ void one(const T* x, T* out, uint32_t i) const {
    const float p = exp_near(as_float(x[i]) - norm.max, -norm.log2_sum);
    out[i] = from_float<T>(i == label ? __fmaf_rn(-w, p, w) : __fmul_rn(-w, p));
  }
  __device__ __forceinline__ uint4 cold(const uint4& q) const {      // a vector that does not hold the label
    const float2 below = both(-norm.max), less = both(-norm.log2_sum), minus = both(-w);
    float2 v[V / 2];
    Vec<T>::open(q, v);
#pragma unroll
    for (int j = 0; j < V / 2; ++j) v[j] = __fmul2_rn(minus, exp_near(__fadd2_rn(v[j], below), less));
    return Vec<T>::close(v);
  }
  __device__ __forceinline__ uint4 hot(const uint4& q, uint32_t at) const {      // one that holds it, as element `at`
    const float2 below = both(-norm.max), less = both(-norm.log2_sum), minus = both(-w);
    float2 v[V / 2];
    Vec<T>::open(q, v);
#pragma unroll
    for (int j = 0; j < V / 2; ++j)
      v[j] = __ffma2_rn(minus, exp_near(__fadd2_rn(v[j], below), less), make_float2(at == 2 * j ? w : 0.0f, at == 2 * j + 1 ? w : 0.0f));
    return Vec<T>::close(v);
  }
};
template <class T, int GROUP, int UNROLL>
__device__ __forceinline__ void grad_row(const T* x, T* out, uint32_t n, uint32_t label, Norm norm, float w, uint32_t tid) {
  const GradRow<T> g(norm, w, label);
  const uint32_t head = lead(x, n), vecs = (n - head) / Vec<T>::n, tail = head + vecs * Vec<T>::n;
  if (lead(out, n) != head) {                     // the two rows lie differently: element by element
    for (uint32_t i = tid; i < n; i += GROUP) g.one(x, out, i);
    return;
  }
  if (tid < head) g.one(x, out, tid);
  if (tail + tid < n) g.one(x, out, tail + tid);
  const uint4* q = reinterpret_cast<const uint4*>(x + head);
  uint4* o = reinterpret_cast<uint4*>(out + head);
  const uint32_t hot = (label - head) / Vec<T>::n, at = (label - head) % Vec<T>::n;     // (a label in front wraps: no vector's)
  for (uint32_t i = tid; i < vecs; i += UNROLL * GROUP) {
    uint4 v[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
      if (i + u * GROUP < vecs) v[u] = __ldg(q + i + u * GROUP);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
      if (i + u * GROUP < vecs) o[i + u * GROUP] = i + u * GROUP == hot ? g.hot(v[u], at) : g.cold(v[u]);
  }
}

template <class T> __device__ __forceinline__ const T* row_of(const Rows& r, int64_t row) {
  const int64_t b = row / r.seq, t = row - b * r.seq;
  return static_cast<const T*>(r.x) + b * r.stride_b + t * r.stride_t;
}
template <class T> struct Out {                   // where the gradient's rows lie
  T* x;
  int64_t stride_b, stride_t;
  __device__ __forceinline__ T* row(int64_t i, uint32_t seq) const {
    const int64_t b = i / seq, t = i - b * seq;
    return x + b * stride_b + t * stride_t;
  }
};
// the label's logit; NaN for a label that is no index
template <class T> __device__ __forceinline__ float at_label(const T* x, int64_t label, uint32_t vocab) {
  return label >= 0 && label < (int64_t)vocab ? as_float(x[label]) : __uint_as_float(0x7fc00000u);
}
template <int GROUP> struct Group {               // a row's threads: a warp of a CTA of kThreads, or a CTA; one group for each row
  static constexpr int threads = GROUP == 32 ? kThreads : GROUP, per_cta = threads / GROUP;
  static __device__ __forceinline__ uint32_t tid() { return GROUP == 32 ? threadIdx.x & 31 : threadIdx.x; }
  static __device__ __forceinline__ int64_t row() {
    return GROUP == 32 ? (int64_t)blockIdx.x * per_cta + (threadIdx.x >> 5) : (int64_t)blockIdx.x;
  }
};

// L: fp32 for the caller, fp64 for the preference loss, whose rewards are small differences of long sums
template <class T, int GROUP, class L>
__global__ void __launch_bounds__(Group<GROUP>::threads, 1024 / Group<GROUP>::threads)
forward_kernel(const Rows r, L* __restrict__ logp, Norm* __restrict__ norms, unsigned int* __restrict__ ticket) {
  using G = Group<GROUP>;
  if (ticket != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *ticket = 0;      // for the kernel behind this one
  const int64_t row = G::row();
  if (row >= r.rows) return;
  const int64_t label = r.labels[row];
  if (label == r.ignore) {
    if (G::tid() == 0) { logp[row] = (L)0; norms[row] = Norm{0.0f, 0.0f}; }
    return;
  }
  const T* x = row_of<T>(r, row);
  const Stat st = join_group<GROUP>(scan<T, GROUP>(x, r.vocab, G::tid()));
  if (G::tid() == 0) {
    const double log_s = log_of(st.s);
    norms[row] = norm_of(st, log_s);
    logp[row] = (L)(((double)at_label(x, label, r.vocab) - (double)st.m) - log_s);
  }
}

// 8192 rows of 50257 bf16, half masked: 208 to 216 us, 6.1 TB/s.
// w of row i: weight[i / per] (* *scale).  UNLESS_ONE: nothing is left to do when *scale is 1, which is most often so: then few
// CTAs are launched, which go through the rows in turn where they have to.
template <class T, int GROUP, bool UNLESS_ONE>
__global__ void __launch_bounds__(Group<GROUP>::threads) backward_kernel(const Rows r, const Norm* __restrict__ norms,
                                                                         const float* __restrict__ weight, uint32_t per,
                                                                         const float* __restrict__ scale, const Out<T> out) {
  using G = Group<GROUP>;
  const float by = scale != nullptr ? *scale : 1.0f;
  auto one = [&](int64_t i) {
    const int64_t row = r.rows - 1 - i, label = r.labels[row];
    T* o = out.row(row, r.seq);
    float w = label == r.ignore ? 0.0f : weight[row / per] * by;
    const Norm norm = norms[row];
    if (label == r.ignore || (w == 0.0f && fabsf(norm.max) <= FLT_MAX && fabsf(norm.log2_sum) <= FLT_MAX)) {
      clear_row<T, GROUP>(o, r.vocab, G::tid());
      return;
    }
    if (label < 0 || label >= (int64_t)r.vocab) w = __uint_as_float(0x7fc00000u);
    grad_row<T, GROUP, 2>(row_of<T>(r, row), o, r.vocab, (uint32_t)label, norm, w, G::tid());
  };
  if constexpr (UNLESS_ONE) {
    if (by == 1.0f) return;
    for (int64_t i = G::row(); i < r.rows; i += (int64_t)gridDim.x * G::per_cta) one(i);
  } else if (G::row() < r.rows) {
    one(G::row());
  }
}

// ---- sums over the CTAs of a grid in a fixed order ----------------------------------------------------------------------
template <int N> __device__ __forceinline__ void cta_sum(double (&v)[N]) {
  __shared__ double part[N][kThreads / 32];
#pragma unroll
  for (int k = 0; k < N; ++k) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) {
#pragma unroll
    for (int k = 0; k < N; ++k) part[k][threadIdx.x >> 5] = v[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; ++k) {
    v[k] = 0.0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) v[k] += part[k][w];
  }
}
// Every CTA leaves its sums in parts[blockIdx.x]; true in all threads of the last one to do so, with the totals in v.
template <int N> __device__ __forceinline__ bool grid_sum(double (&v)[N], double* parts, unsigned int* ticket) {
  __shared__ bool last;
  cta_sum(v);
  if (threadIdx.x == 0) {
#pragma unroll
    for (int k = 0; k < N; ++k) parts[(int64_t)blockIdx.x * N + k] = v[k];
    __threadfence();
    last = atomicAdd(ticket, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return false;
  __threadfence();
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = 0.0;
  for (unsigned int i = threadIdx.x; i < gridDim.x; i += kThreads)
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] += __ldcg(parts + (int64_t)i * N + k);
  cta_sum(v);
  return true;
}

// ---- preference loss ----------------------------------------------------------------------------------------------------
// One CTA per pair in turn: sums of both sequences in 64 bits (they differ little and are long), rewards, loss, weights.  The reference
// comes as it was given, fp32 or fp64: a cast in front would be a launch of its own (78 us instead of 72 for pairs of 12 rows of 13).
template <class Ref>
__global__ void __launch_bounds__(kThreads) preference_kernel(const double* __restrict__ logp, const Ref* __restrict__ ref, int64_t pairs,
                                                              uint32_t seq, double beta, double smooth, double* __restrict__ parts,
                                                              unsigned int* __restrict__ ticket, float* __restrict__ loss,
                                                              float* __restrict__ rewards, float* __restrict__ weight) {
  double sum[1] = {0.0};
  for (int64_t p = blockIdx.x; p < pairs; p += gridDim.x) {
    double s[2] = {0.0, 0.0};
    for (uint32_t t = threadIdx.x; t < seq; t += kThreads) {
      s[0] += logp[p * seq + t];
      s[1] += logp[(pairs + p) * seq + t];
    }
    cta_sum(s);
    if (threadIdx.x == 0) {
      const double chosen = beta * (s[0] - ref[p]), rejected = beta * (s[1] - ref[pairs + p]), h = chosen - rejected;
      const double tail = log1p(exp(-fabs(h)));             // -logsigmoid(h) = max(-h, 0) + log(1 + exp(-|h|))
      // (h is infinite where a label's logit is -inf; a term whose factor is 0 is left out then, not 0 times infinity)
      if (smooth < 1.0) sum[0] += (1.0 - smooth) * (fmax(-h, 0.0) + tail);
      if (smooth > 0.0) sum[0] += smooth * (fmax(h, 0.0) + tail);
      if (h != h) sum[0] = h;
      const double w = beta / (double)pairs * (smooth / (1.0 + exp(-h)) - (1.0 - smooth) / (1.0 + exp(h)));
      rewards[p] = (float)chosen;
      rewards[pairs + p] = (float)rejected;
      weight[p] = (float)w;                                  // of dloss / dlogp, constant along the sequence
      weight[pairs + p] = (float)-w;
    }
  }
  if (grid_sum(sum, parts, ticket) && threadIdx.x == 0) *loss = (float)(sum[0] / (double)pairs);
}

// ---- policy loss --------------------------------------------------------------------------------------------------------
struct Policy {
  const float* old;         // [rows]
  const float* ref;         // [rows] or null
  const float* advantage;   // [rows / per]
  uint32_t per;
  float low, high, kl;      // 1 - clip, 1 + clip_high, coefficient of the KL term
};
// Rows that have a label: one count per CTA, which those who need it add up.  Also readies the words of the kernels behind it.
constexpr int kCountParts = 148;
struct Words {
  unsigned int ticket;
  unsigned int count[kCountParts];
};
__global__ void __launch_bounds__(kThreads) count_kernel(const int64_t* __restrict__ labels, int64_t rows, int64_t ignore,
                                                         Words* __restrict__ words) {
  unsigned int n = 0;
#pragma unroll 8
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < rows; i += (int64_t)gridDim.x * kThreads)
    n += labels[i] != ignore;
  __shared__ unsigned int part[kThreads / 32];
  n = __reduce_add_sync(0xffffffffu, n);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = n;
  __syncthreads();
  if (threadIdx.x == 0) {
    n = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) n += part[w];
    words->count[blockIdx.x] = n;
    if (blockIdx.x == 0) words->ticket = 0;
  }
}
// (the counts are loaded by the lanes of a warp, long before their sum is needed)
__device__ __forceinline__ unsigned int my_counts(const Words* words, int parts) {
  unsigned int n = 0;
  for (int i = threadIdx.x & 31; i < parts; i += 32) n += words->count[i];
  return n;
}
__device__ __forceinline__ float share_of(unsigned int counts) {
  const unsigned int live = __reduce_add_sync(0xffffffffu, counts);
  return 1.0f / (float)(live > 0 ? live : 1);
}

struct PolicyOut {
  float* logp;              // [rows]
  Norm* norm;               // [rows]
  float* weight;            // [rows]: dloss / dlogp
  float* term;              // [2, rows]: the row's loss; its KL term, with the sign set where the clamp cut the gradient
};
// What the loss needs of a row beside its sum, loaded while that is found.
struct RowIn {
  float advantage, old, ref, x;
};
template <class T> __device__ __forceinline__ RowIn row_in(const Policy& p, int64_t row, const T* x, int64_t label, uint32_t vocab) {
  return RowIn{p.advantage[row / p.per], p.old[row], p.ref != nullptr ? p.ref[row] : 0.0f, at_label(x, label, vocab)};
}
// The row's results, stored by its first thread, and its weight.
__device__ __forceinline__ float policy_row(const Policy& p, const PolicyOut& o, int64_t rows, int64_t row, const RowIn& in, float logp,
                                            Norm norm, float share, bool store) {
  const float a = in.advantage, rho = expf(logp - in.old);
  const float s = rho * a, q = fminf(fmaxf(rho, p.low), p.high) * a;
  const bool clipped = s > q;                                // (not when it is no number: that has to show)
  float w = clipped ? 0.0f : -s, kl = 0.0f, term = -(clipped ? q : s);
  if (p.ref != nullptr) {
    const float d = in.ref - logp, e = expm1f(d);
    kl = e <= FLT_MAX ? fabsf(e - d) : e;                    // (never negative but for the last rounding; inf - inf is inf here)
    if (p.kl != 0.0f) {                                      // (the term may be infinite where it is only looked at)
      w = fmaf(-p.kl, e, w);
      term = fmaf(p.kl, kl, term);
    }
  }
  w *= share;
  if (store) {
    o.logp[row] = logp;
    o.norm[row] = norm;
    o.weight[row] = w;
    o.term[row] = term;
    o.term[rows + row] = clipped ? -kl : kl;
  }
  return w;
}
__device__ __forceinline__ void no_row(const PolicyOut& o, int64_t rows, int64_t row) {
  o.logp[row] = o.weight[row] = o.term[row] = o.term[rows + row] = 0.0f;
  o.norm[row] = Norm{0.0f, 0.0f};
}

// One group for each row, which it reads twice when it writes the gradient: the second time from L2 unless the rows are very long.
template <class T, int GROUP>
__global__ void __launch_bounds__(Group<GROUP>::threads) policy_kernel(const Rows r, const Policy p, const Words* __restrict__ words, int parts,
                                                                       const PolicyOut o, const Out<T> grad) {
  using G = Group<GROUP>;
  const int64_t row = G::row();
  if (row >= r.rows) return;
  const unsigned int counts = my_counts(words, parts);
  const int64_t label = r.labels[row];
  if (label == r.ignore) {
    if (G::tid() == 0) no_row(o, r.rows, row);
    if (grad.x != nullptr) clear_row<T, GROUP>(grad.row(row, r.seq), r.vocab, G::tid());
    return;
  }
  const T* x = row_of<T>(r, row);
  const RowIn in = row_in(p, row, x, label, r.vocab);
  const Stat st = join_group<GROUP>(scan<T, GROUP>(x, r.vocab, G::tid()));
  const double log_s = log_of(st.s);
  const Norm norm = norm_of(st, log_s);
  const float logp = (float)(((double)in.x - (double)st.m) - log_s);
  const float w = policy_row(p, o, r.rows, row, in, logp, norm, share_of(counts), G::tid() == 0);
  if (grad.x != nullptr) grad_row<T, GROUP, 8>(x, grad.row(row, r.seq), r.vocab, (uint32_t)label, norm, w, G::tid());
}

// Means over the rows with a label, in 64 bits and in a fixed order.
__global__ void __launch_bounds__(kThreads) policy_sum_kernel(const float* __restrict__ term, const int64_t* __restrict__ labels, int64_t ignore,
                                                              int64_t rows, Words* __restrict__ words, double* __restrict__ parts,
                                                              float* __restrict__ loss, float* __restrict__ stats) {
  double sum[4] = {0.0, 0.0, 0.0, 0.0};
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < rows; i += (int64_t)gridDim.x * kThreads) {
    const float kl = term[rows + i];
    sum[0] += (double)term[i];
    sum[1] += fabs((double)kl);
    sum[2] += (__float_as_uint(kl) >> 31) != 0u ? 1.0 : 0.0;
    sum[3] += labels[i] != ignore ? 1.0 : 0.0;
  }
  if (grid_sum(sum, parts, &words->ticket) && threadIdx.x == 0) {
    const double n = fmax(sum[3], 1.0);
    *loss = (float)(sum[0] / n);
    stats[0] = (float)(sum[1] / n);
    stats[1] = (float)(sum[2] / n);
  }
}

// ---- launches -----------------------------------------------------------------------------------------------------------
inline bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

int check_rows(const nvfp4_logit_rows* in, Rows& r) {
  if (in == nullptr || !in->logits || !in->labels) return NVFP4_E_NULL;
  if (in->batch <= 0 || in->seq <= 0 || in->vocab <= 0) return NVFP4_E_SHAPE;
  if (in->seq > 0x7fffffffLL || in->vocab > 0x7fffffffLL || in->batch > INT64_MAX / in->seq / in->vocab / 4 ||
      in->batch > 0x7fffffffLL / in->seq)
    return NVFP4_E_LIMIT;
  if (!aligned(in->logits, in->is_f32 ? 4 : 2) || !aligned(in->labels, 8)) return NVFP4_E_ALIGN;
  r = Rows{in->logits, in->stride_b, in->stride_t, in->batch * in->seq, (uint32_t)in->seq, (uint32_t)in->vocab, in->labels,
           in->ignore_index};
  return NVFP4_OK;
}
int launched() { return cudaGetLastError() == cudaSuccess ? NVFP4_OK : NVFP4_E_LAUNCH; }

// Threads for a row of `vecs` 16-byte vectors.  Many short rows go to warps (16384 rows of 512 vectors, bf16, forward 34 us; 42 with
// CTAs of 128, 167 with 512), long ones to as few threads as still have many loads in flight: the fewer, the more rows an SM has
// under way, whose ends do not meet (16384 rows of 8192 vectors, forward 327 us with 128 threads, 415 with 512).  Kernels that
// write read a row again behind its sum and want few of them, so that it is still in L2: more threads for long rows
// (4096 vectors 392 us with 256 threads, 438 with 128, 478 with 512; fp32, 8192 vectors 697 with 512, 904 with 256).  Where there are few rows,
// latency counts, and they are spread wider (16 rows of 16384 vectors, gradient: 100 us with a warp, 28 with 128 threads, 10.7 with 512).
// Over 16 to 16384 rows of 64 to 32768 vectors no choice takes 1.35 times the best of the four.
int group_of(int64_t rows, int64_t vecs, bool writes) {
  if (rows >= 148 * 4) {
    if (vecs <= 256 || (rows >= 4096 && vecs <= 1024)) return 32;
    if (!writes || vecs <= 2048) return 128;
    return vecs < 8192 ? 256 : 512;
  }
  if (vecs <= 128) return 32;
  if (vecs <= 512) return 128;
  return vecs <= (writes ? 2048 : 8192) ? 256 : 512;
}
// f(type tag, group size tag, grid)
template <class F> void by_rows(bool f32, const Rows& r, bool writes, F f) {
  const int group = group_of(r.rows, ((int64_t)r.vocab * (f32 ? 4 : 2) + 15) / 16, writes);
  auto sized = [&](auto t) {
    if (group == 32) f(t, std::integral_constant<int, 32>(), (unsigned)((r.rows + kThreads / 32 - 1) / (kThreads / 32)));
    else if (group == 128) f(t, std::integral_constant<int, 128>(), (unsigned)r.rows);
    else if (group == 256) f(t, std::integral_constant<int, 256>(), (unsigned)r.rows);
    else f(t, std::integral_constant<int, 512>(), (unsigned)r.rows);
  };
  if (f32) sized(float());
  else sized(__nv_bfloat16());
}
// (16384 rows of 50257 bf16: 246 us, 6.7 TB/s, with eight CTAs of 128 threads an SM; 262 with four of 256)
template <class L> void forward(const Rows& r, bool f32, L* logp, Norm* norms, unsigned int* ticket, cudaStream_t stream) {
  by_rows(f32, r, false, [&](auto t, auto g, unsigned grid) {
    constexpr int G = decltype(g)::value;
    forward_kernel<decltype(t), G, L><<<grid, Group<G>::threads, 0, stream>>>(r, logp, norms, ticket);
  });
}

constexpr int kWordsBytes = 1024;
static_assert(sizeof(Words) <= kWordsBytes && kWordsBytes + 4 * 8 * NVFP4_LOSS_PARTS <= NVFP4_LOSS_WORKSPACE, "");

// The row is read again right behind its sum, from L2, with eight vectors of a thread in flight to hide its latency (8192 rows of
// 50257 bf16, a quarter masked: 276 us, 5.1 TB/s; 317 with two vectors, 285 with four; 309 with the row kept in shared memory and
// the next one copied in behind it).  The rows in flight, two an SM for long ones, and their gradients have to fit in L2: of 1.6 GB of logits
// 1.6 GB are read from HBM in rows of up to 131 KB, 2.0 to 2.3 in rows of 200 KB, 2.9 to 3.0 in rows of 262 KB (65536 fp32 logits,
// 131072 of bf16) and 3.2 beyond: 541, 599, 693 and 725 to 763 us in fp32.  The same kernel with and without a gradient: the loss has the same bits.
void policy_rows(const Rows& r, bool f32, const Policy& p, Words* words, int counts, const PolicyOut& o, void* dlogits, int64_t dstride_b,
                 int64_t dstride_t, cudaStream_t stream) {
  by_rows(f32, r, true, [&](auto t, auto g, unsigned grid) {
    using T = decltype(t);
    constexpr int G = decltype(g)::value;
    policy_kernel<T, G><<<grid, Group<G>::threads, 0, stream>>>(r, p, words, counts, o, Out<T>{static_cast<T*>(dlogits), dstride_b, dstride_t});
  });
}

}  // namespace logprob
}  // namespace nvfp4

using namespace nvfp4::logprob;

extern "C" int nvfp4_logprob_fwd(const nvfp4_logit_rows* in, float* logp, nvfp4_row_stat* stat, void* stream_) {
  Rows r;
  if (const int code = check_rows(in, r); code != NVFP4_OK) return code;
  if (!logp || !stat) return NVFP4_E_NULL;
  if (!aligned(logp, 4) || !aligned(stat, 8)) return NVFP4_E_ALIGN;
  forward(r, in->is_f32 != 0, logp, stat, nullptr, static_cast<cudaStream_t>(stream_));
  return launched();
}

extern "C" int nvfp4_logprob_bwd(const nvfp4_logit_rows* in, const nvfp4_row_stat* stat, const float* weight, int64_t rows_per_weight,
                                 const float* scale, int unless_one, void* dlogits, int64_t dstride_b, int64_t dstride_t,
                                 void* stream_) {
  Rows r;
  if (const int code = check_rows(in, r); code != NVFP4_OK) return code;
  if (!stat || !weight || !dlogits || (unless_one && !scale)) return NVFP4_E_NULL;
  if (rows_per_weight <= 0 || rows_per_weight > 0x7fffffffLL) return NVFP4_E_SHAPE;
  if (!aligned(stat, 8) || !aligned(weight, 4) || !aligned(scale, 4) || !aligned(dlogits, in->is_f32 ? 4 : 2)) return NVFP4_E_ALIGN;
  by_rows(in->is_f32 != 0, r, true, [&](auto t, auto g, unsigned grid) {
    using T = decltype(t);
    constexpr int G = decltype(g)::value;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    const Out<T> out{static_cast<T*>(dlogits), dstride_b, dstride_t};
    const uint32_t per = (uint32_t)rows_per_weight;
    if (unless_one) backward_kernel<T, G, true><<<grid < 148 * 4 ? grid : 148 * 4, Group<G>::threads, 0, stream>>>(r, stat, weight, per, scale, out);
    else backward_kernel<T, G, false><<<grid, Group<G>::threads, 0, stream>>>(r, stat, weight, per, scale, out);
  });
  return launched();
}

template <class Ref>
static int preference_fwd(const nvfp4_logit_rows* in, const Ref* ref, double beta, double label_smoothing, double* logp, nvfp4_row_stat* stat,
                          float* loss, float* rewards, float* weight, void* workspace, size_t workspace_bytes, void* stream_) {
  Rows r;
  if (const int code = check_rows(in, r); code != NVFP4_OK) return code;
  if (in->batch % 2 != 0) return NVFP4_E_SHAPE;
  if (!ref || !logp || !stat || !loss || !rewards || !weight || !workspace) return NVFP4_E_NULL;
  if (workspace_bytes < NVFP4_LOSS_WORKSPACE) return NVFP4_E_WORKSPACE;
  if (!aligned(ref, sizeof(Ref)) || !aligned(logp, 8) || !aligned(stat, 8) || !aligned(loss, 4) || !aligned(rewards, 4) || !aligned(weight, 4) ||
      !aligned(workspace, 16))
    return NVFP4_E_ALIGN;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  unsigned int* ticket = static_cast<unsigned int*>(workspace);
  double* parts = reinterpret_cast<double*>(static_cast<char*>(workspace) + 16);
  forward(r, in->is_f32 != 0, logp, stat, ticket, stream);
  if (const int code = launched(); code != NVFP4_OK) return code;
  const int64_t pairs = in->batch / 2;
  preference_kernel<Ref><<<(unsigned)(pairs < NVFP4_LOSS_PARTS ? pairs : NVFP4_LOSS_PARTS), kThreads, 0, stream>>>(
      logp, ref, pairs, r.seq, beta, label_smoothing, parts, ticket, loss, rewards, weight);
  return launched();
}

extern "C" int nvfp4_preference_fwd(const nvfp4_logit_rows* in, const float* ref, double beta, double label_smoothing, double* logp,
                                    nvfp4_row_stat* stat, float* loss, float* rewards, float* weight, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  return preference_fwd(in, ref, beta, label_smoothing, logp, stat, loss, rewards, weight, workspace, workspace_bytes, stream);
}
extern "C" int nvfp4_preference_fwd_ref64(const nvfp4_logit_rows* in, const double* ref, double beta, double label_smoothing, double* logp,
                                          nvfp4_row_stat* stat, float* loss, float* rewards, float* weight, void* workspace,
                                          size_t workspace_bytes, void* stream) {
  return preference_fwd(in, ref, beta, label_smoothing, logp, stat, loss, rewards, weight, workspace, workspace_bytes, stream);
}

extern "C" int nvfp4_policy_fwd(const nvfp4_logit_rows* in, const float* old_logp, const float* advantage,
                                int64_t rows_per_advantage, const float* ref_logp, double clip_low, double clip_high, double kl,
                                float* logp, nvfp4_row_stat* stat, float* weight, float* terms, float* loss, float* stats2, void* dlogits,
                                int64_t dstride_b, int64_t dstride_t, void* workspace, size_t workspace_bytes, void* stream_) {
  Rows r;
  if (const int code = check_rows(in, r); code != NVFP4_OK) return code;
  if (!old_logp || !advantage || !logp || !stat || !weight || !terms || !loss || !stats2 || !workspace) return NVFP4_E_NULL;
  if (rows_per_advantage <= 0 || rows_per_advantage > 0x7fffffffLL) return NVFP4_E_SHAPE;
  if (workspace_bytes < NVFP4_LOSS_WORKSPACE) return NVFP4_E_WORKSPACE;
  if (!aligned(old_logp, 4) || !aligned(advantage, 4) || !aligned(ref_logp, 4) || !aligned(logp, 4) || !aligned(stat, 8) ||
      !aligned(weight, 4) || !aligned(terms, 4) || !aligned(loss, 4) || !aligned(stats2, 4) || !aligned(dlogits, in->is_f32 ? 4 : 2) || !aligned(workspace, 16))
    return NVFP4_E_ALIGN;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  char* ws = static_cast<char*>(workspace);
  Words* words = reinterpret_cast<Words*>(ws);
  double* parts = reinterpret_cast<double*>(ws + kWordsBytes);
  const int64_t ctas = (r.rows + kThreads * 8 - 1) / (kThreads * 8);
  const int counts = (int)(ctas < kCountParts ? ctas : kCountParts);
  count_kernel<<<counts, kThreads, 0, stream>>>(r.labels, r.rows, r.ignore, words);
  if (const int code = launched(); code != NVFP4_OK) return code;
  const Policy p{old_logp, ref_logp, advantage, (uint32_t)rows_per_advantage, (float)(1.0 - clip_low),
                 (float)(1.0 + clip_high), (float)kl};
  const PolicyOut o{logp, stat, weight, terms};
  policy_rows(r, in->is_f32 != 0, p, words, counts, o, dlogits, dstride_b, dstride_t, stream);
  if (const int code = launched(); code != NVFP4_OK) return code;
  const int64_t sums = (r.rows + kThreads * 8 - 1) / (kThreads * 8);
  policy_sum_kernel<<<(unsigned)(sums < NVFP4_LOSS_PARTS ? sums : NVFP4_LOSS_PARTS), kThreads, 0, stream>>>(
      terms, r.labels, r.ignore, r.rows, words, parts, loss, stats2);
  return launched();
}
