// Losses on logits and their gradients (sm_100a): log-probabilities of given labels, a preference loss over pairs of
// sequences, a clipped policy loss with a KL term.
//
//   lse = M + log sum_v exp(x_v - M)        logp = x[label] - lse (0 where the label is the ignored one)
//   dx_v = w (onehot_v - exp(x_v - lse))    with w = dloss / dlogp of the row
//   preference: L_i = sum_t logp_it, reward_i = beta (L_i - ref_i), h = reward_chosen - reward_rejected,
//               loss = mean over pairs of -(1 - s) logsigmoid(h) - s logsigmoid(-h);
//               w_chosen = beta / P (s sigmoid(h) - (1 - s) sigmoid(-h)) = -w_rejected
//   policy:     rho = exp(logp - old), q = clamp(rho, 1 - low, 1 + high) A, d = ref - logp, n = rows with a label,
//               loss = 1/n sum(-min(rho A, q) + k (exp(d) - d - 1)); w = (-[rho A <= q] rho A + k (1 - exp(d))) / n
//
// A row of logits is read once with a running maximum and sum per thread, the group's are joined at the end: fp32, base
// 2, the maximum subtracted before the product with log2 e, so that rows of the type's lowest value give no infinity.
// The maximum starts at the lowest finite number, not at -inf: a row of -inf then ends with a sum of 0 and lse = -inf.
// A row of more than kWarpRow logits belongs to a CTA, a shorter one to a warp.
// The policy loss's w depends on its own row alone, so its kernel writes the row's gradient right behind the sum, while
// the row is in L2: HBM sees each row once.  The preference loss has to see both sequences first; its backward takes the
// rows in the opposite order, so that the last ones read are still in L2.
#include <cfloat>
#include <type_traits>

#include "common.cuh"
#include "nvfp4_b200.h"

namespace nvfp4 {
namespace logprob {

constexpr int kThreads = 256;
constexpr int kWarpRow = 2048;
// log2 e in two parts: alone, the first is off by 1.3e-8 of itself, which moves every term of a row the same way, and the sum
// of a sequence's thousand log-probabilities shows it.  (The mean error of a row's logsumexp, measured over 2048 rows of 13
// to 50257 logits, is 1e-8; the 5e-8 by which ex2.approx falls short on average reaches the small terms only.)
constexpr float kLog2e = 1.4426950408889634f, kLog2eRest = 1.925963e-8f;

struct Rows {
  const void* x;
  int64_t stride_b, stride_t;     // in elements; the logits of a row are contiguous
  int64_t rows;                   // batch * seq
  uint32_t seq, vocab;
  const int64_t* labels;          // [rows]
  int64_t ignore;
};
// running maximum and sum of exp(x - maximum)
struct Stat {
  float m, s;
};

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float exp_of(float d) { return ex2(fmaf(d, kLog2e, d * kLog2eRest)); }
// M + log s.  The sum's exponent is taken off in front of the logarithm, whose own rounding is then far below that of an fp32
// result.  (Beside a coarse maximum, logf(s) would leave every other result halfway between two fp32 numbers.)
__device__ __forceinline__ double lse_of(Stat st) {
  const int k = min(max((int)(__float_as_uint(st.s) >> 23) - 127, 0), 63);       // s is 1 to 2^31, or 0, or no number
  const float f = st.s * __uint_as_float((uint32_t)(127 - k) << 23);
  return (double)st.m + (k * 0.69314718055994531 + (double)logf(f));
}

template <class T> struct Vec;
template <> struct Vec<float> {
  static constexpr int n = 4;
  static __device__ __forceinline__ void open(const uint4& q, float (&v)[4]) {
    v[0] = __uint_as_float(q.x); v[1] = __uint_as_float(q.y); v[2] = __uint_as_float(q.z); v[3] = __uint_as_float(q.w);
  }
  static __device__ __forceinline__ uint4 close(const float (&v)[4]) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  }
};
__device__ __forceinline__ uint32_t pack(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <> struct Vec<__nv_bfloat16> {
  static constexpr int n = 8;
  static __device__ __forceinline__ void open(const uint4& q, float (&v)[8]) {
    v[0] = bf16_lo(q.x); v[1] = bf16_hi(q.x); v[2] = bf16_lo(q.y); v[3] = bf16_hi(q.y);
    v[4] = bf16_lo(q.z); v[5] = bf16_hi(q.z); v[6] = bf16_lo(q.w); v[7] = bf16_hi(q.w);
  }
  static __device__ __forceinline__ uint4 close(const float (&v)[8]) {
    return make_uint4(pack(v[0], v[1]), pack(v[2], v[3]), pack(v[4], v[5]), pack(v[6], v[7]));
  }
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
template <int N> __device__ __forceinline__ void take(Stat& st, const float (&v)[N]) {
  float m = st.m;
#pragma unroll
  for (int j = 0; j < N; ++j) m = fmaxf(m, v[j]);
  float s = m > st.m ? st.s * expf(st.m - m) : st.s, s1 = 0.0f;
#pragma unroll
  for (int j = 0; j < N; j += 2) {
    s += exp_of(v[j] - m);
    if (j + 1 < N) s1 += exp_of(v[j + 1] - m);
  }
  st = Stat{m, s + s1};
}

// maximum and sum of this thread's part of a row; GROUP threads share the row
template <class T, int GROUP> __device__ __forceinline__ Stat scan(const T* x, uint32_t n, uint32_t tid) {
  constexpr int V = Vec<T>::n, UNROLL = 4;
  Stat st{-FLT_MAX, 0.0f};
  const uint32_t head = lead(x, n), vecs = (n - head) / V, tail = head + vecs * V;
  for (uint32_t i = tid; i < head; i += GROUP) { const float one[1] = {as_float(x[i])}; take(st, one); }
  const uint4* q = reinterpret_cast<const uint4*>(x + head);
  uint32_t i = tid;
  for (; i + (UNROLL - 1) * GROUP < vecs; i += UNROLL * GROUP) {
    uint4 w[UNROLL];
    float v[UNROLL * V];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) w[u] = __ldg(q + i + u * GROUP);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) Vec<T>::open(w[u], reinterpret_cast<float(&)[V]>(v[u * V]));
    take(st, v);
  }
  for (; i < vecs; i += GROUP) {
    float v[V];
    Vec<T>::open(__ldg(q + i), v);
    take(st, v);
  }
  for (uint32_t j = tail + tid; j < n; j += GROUP) { const float one[1] = {as_float(x[j])}; take(st, one); }
  return st;
}
// The group's maximum and sum, the same bits in every thread (a butterfly of plain sums is symmetric).
template <int GROUP> __device__ __forceinline__ Stat join_group(Stat st) {
  float m = st.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  float s = st.s * expf(st.m - m);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (GROUP > 32) {
    __shared__ Stat part[kThreads / 32];
    __syncthreads();                              // the last row's have been read
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = Stat{m, s};
    __syncthreads();
#pragma unroll
    for (int w = 0; w < GROUP / 32; ++w) m = fmaxf(m, part[w].m);
    s = 0.0f;
#pragma unroll
    for (int w = 0; w < GROUP / 32; ++w) s += part[w].s * expf(part[w].m - m);
  }
  return Stat{m, s};
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
// out = w (onehot - exp(x - lse)); w = 0 gives zeros unless the row holds something that is no number
template <class T, int GROUP>
__device__ __forceinline__ void grad_row(const T* x, T* out, uint32_t n, uint32_t label, float lse, float w, uint32_t tid) {
  constexpr int V = Vec<T>::n;
  auto one = [&](uint32_t i) {
    const float p = exp_of(as_float(x[i]) - lse);
    out[i] = from_float<T>(i == label ? __fmaf_rn(-w, p, w) : __fmul_rn(-w, p));
  };
  const uint32_t head = lead(x, n), vecs = (n - head) / V, tail = head + vecs * V;
  if (lead(out, n) != head) {                     // the two rows lie differently: element by element
    for (uint32_t i = tid; i < n; i += GROUP) one(i);
    return;
  }
  for (uint32_t i = tid; i < head; i += GROUP) one(i);
  const uint4* q = reinterpret_cast<const uint4*>(x + head);
  uint4* o = reinterpret_cast<uint4*>(out + head);
  const uint32_t hot = label - head;              // (wraps when the label lies in front: then no vector holds it)
#pragma unroll 2
  for (uint32_t i = tid; i < vecs; i += GROUP) {
    float v[V];
    Vec<T>::open(__ldg(q + i), v);
    const uint32_t at = hot / V == i ? hot % V : V;
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = __fmaf_rn(-w, exp_of(v[j] - lse), at == j ? w : 0.0f);
    o[i] = Vec<T>::close(v);
  }
  for (uint32_t j = tail + tid; j < n; j += GROUP) one(j);
}

template <class T> __device__ __forceinline__ const T* row_of(const Rows& r, int64_t row) {
  const int64_t b = row / r.seq, t = row - b * r.seq;
  return static_cast<const T*>(r.x) + b * r.stride_b + t * r.stride_t;
}
// log-probability of a label; NaN for a label that is no index
template <class T> __device__ __forceinline__ double logp_of(const T* x, int64_t label, uint32_t vocab, double lse) {
  return label >= 0 && label < (int64_t)vocab ? (double)as_float(x[label]) - lse : (double)__uint_as_float(0x7fc00000u);
}
template <int GROUP> struct Group {               // rows are dealt to the groups of the grid in turn
  static constexpr int per_cta = kThreads / GROUP;
  static __device__ __forceinline__ uint32_t tid() { return GROUP == kThreads ? threadIdx.x : threadIdx.x & 31; }
  static __device__ __forceinline__ int64_t first() {
    return GROUP == kThreads ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * per_cta + (threadIdx.x >> 5);
  }
  static __device__ __forceinline__ int64_t step() { return (int64_t)gridDim.x * per_cta; }
};

// L: fp32 for the caller, fp64 for the preference loss, whose rewards are small differences of long sums
template <class T, int GROUP, class L>
__global__ void __launch_bounds__(kThreads) forward_kernel(const Rows r, L* __restrict__ logp, float* __restrict__ lse_out,
                                                           unsigned int* __restrict__ ticket) {
  using G = Group<GROUP>;
  if (ticket != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *ticket = 0;      // for the kernel behind this one
  for (int64_t row = G::first(); row < r.rows; row += G::step()) {
    const int64_t label = r.labels[row];
    if (label == r.ignore) {
      if (G::tid() == 0) { logp[row] = (L)0; lse_out[row] = 0.0f; }
      continue;
    }
    const T* x = row_of<T>(r, row);
    const Stat st = join_group<GROUP>(scan<T, GROUP>(x, r.vocab, G::tid()));
    if (G::tid() == 0) {
      const double lse = lse_of(st);
      lse_out[row] = (float)lse;
      logp[row] = (L)logp_of(x, label, r.vocab, lse);
    }
  }
}

// w of row i: weight[i / per] (* *scale).  unless_one: nothing is left to do when *scale is 1.
template <class T, int GROUP>
__global__ void __launch_bounds__(kThreads) backward_kernel(const Rows r, const float* __restrict__ lse, const float* __restrict__ weight,
                                                            uint32_t per, const float* __restrict__ scale, bool unless_one,
                                                            T* __restrict__ out) {
  using G = Group<GROUP>;
  const float by = scale != nullptr ? *scale : 1.0f;
  if (unless_one && by == 1.0f) return;
  for (int64_t i = G::first(); i < r.rows; i += G::step()) {
    const int64_t row = r.rows - 1 - i, label = r.labels[row];
    T* o = out + row * r.vocab;
    float w = label == r.ignore ? 0.0f : weight[row / per] * by;
    const float l = lse[row];
    if (label == r.ignore || (w == 0.0f && fabsf(l) <= FLT_MAX)) {
      clear_row<T, GROUP>(o, r.vocab, G::tid());
      continue;
    }
    if (label < 0 || label >= (int64_t)r.vocab) w = __uint_as_float(0x7fc00000u);
    grad_row<T, GROUP>(row_of<T>(r, row), o, r.vocab, (uint32_t)label, l, w, G::tid());
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
// One CTA per pair in turn: sums of both sequences in 64 bits (they differ little and are long), rewards, loss, weights.
__global__ void __launch_bounds__(kThreads) preference_kernel(const double* __restrict__ logp, const float* __restrict__ ref, int64_t pairs,
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
      sum[0] += (1.0 - smooth) * (fmax(-h, 0.0) + tail) + smooth * (fmax(h, 0.0) + tail);
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
__global__ void __launch_bounds__(kThreads) count_kernel(const int64_t* __restrict__ labels, int64_t rows, int64_t ignore,
                                                         unsigned long long* __restrict__ count) {
  unsigned int n = 0;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < rows; i += (int64_t)gridDim.x * kThreads)
    n += labels[i] != ignore;
  n = __reduce_add_sync(0xffffffffu, n);
  if ((threadIdx.x & 31) == 0 && n != 0) atomicAdd(count, (unsigned long long)n);
}

struct PolicyOut {
  float* logp;              // [rows]
  float* lse;               // [rows]
  float* weight;            // [rows]: dloss / dlogp
  float* loss;
  float* stats;             // mean of the KL term, share of clipped rows
  double* parts;
  unsigned int* ticket;
};
template <class T, int GROUP>
__global__ void __launch_bounds__(kThreads) policy_kernel(const Rows r, const Policy p, const unsigned long long* __restrict__ count,
                                                          const PolicyOut o, T* __restrict__ grad) {
  using G = Group<GROUP>;
  const unsigned long long live = *count;
  const float share = 1.0f / (float)(live > 0 ? live : 1);
  double sum[3] = {0.0, 0.0, 0.0};
  for (int64_t row = G::first(); row < r.rows; row += G::step()) {
    const int64_t label = r.labels[row];
    if (label == r.ignore) {
      if (G::tid() == 0) { o.logp[row] = 0.0f; o.lse[row] = 0.0f; o.weight[row] = 0.0f; }
      if (grad != nullptr) clear_row<T, GROUP>(grad + row * r.vocab, r.vocab, G::tid());
      continue;
    }
    const T* x = row_of<T>(r, row);
    const Stat st = join_group<GROUP>(scan<T, GROUP>(x, r.vocab, G::tid()));
    const double lse64 = lse_of(st);
    const float lse = (float)lse64, logp = (float)logp_of(x, label, r.vocab, lse64);
    const float a = p.advantage[row / p.per], rho = expf(logp - p.old[row]);
    const float s = rho * a, q = fminf(fmaxf(rho, p.low), p.high) * a;
    const bool clipped = s > q;                              // (not when it is no number: that has to show)
    float w = clipped ? 0.0f : -s, kl = 0.0f;
    if (p.ref != nullptr) {
      const float d = p.ref[row] - logp, e = expm1f(d);
      kl = e - d;
      w -= p.kl * e;
    }
    w *= share;
    if (G::tid() == 0) {
      o.logp[row] = logp;
      o.lse[row] = lse;
      o.weight[row] = w;
      sum[0] += (double)(p.kl * kl) - (double)(clipped ? q : s);
      sum[1] += (double)kl;
      sum[2] += clipped ? 1.0 : 0.0;
    }
    if (grad != nullptr) grad_row<T, GROUP>(x, grad + row * r.vocab, r.vocab, (uint32_t)label, lse, w, G::tid());
  }
  if (grid_sum(sum, o.parts, o.ticket) && threadIdx.x == 0) {
    const double n = (double)(live > 0 ? live : 1);
    *o.loss = (float)(sum[0] / n);
    o.stats[0] = (float)(sum[1] / n);
    o.stats[1] = (float)(sum[2] / n);
  }
}

// ---- launches -----------------------------------------------------------------------------------------------------------
inline bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

int check_rows(const nvfp4_logit_rows* in, Rows& r) {
  if (in == nullptr || !in->logits || !in->labels) return NVFP4_E_NULL;
  if (in->batch <= 0 || in->seq <= 0 || in->vocab <= 0) return NVFP4_E_SHAPE;
  if (in->seq > 0x7fffffffLL || in->vocab > 0x7fffffffLL || in->batch > INT64_MAX / in->seq / in->vocab / 4) return NVFP4_E_LIMIT;
  if (!aligned(in->logits, in->is_f32 ? 4 : 2) || !aligned(in->labels, 8)) return NVFP4_E_ALIGN;
  r = Rows{in->logits, in->stride_b, in->stride_t, in->batch * in->seq, (uint32_t)in->seq, (uint32_t)in->vocab, in->labels,
           in->ignore_index};
  return NVFP4_OK;
}
// CTAs for `rows` rows in groups of a warp or a CTA: enough to fill the machine, few enough to sum their parts quickly
unsigned grid_of(const Rows& r) {
  const int64_t ctas = r.vocab <= kWarpRow ? (r.rows + kThreads / 32 - 1) / (kThreads / 32) : r.rows;
  return (unsigned)(ctas < NVFP4_LOSS_PARTS ? ctas : NVFP4_LOSS_PARTS);
}
int launched() { return cudaGetLastError() == cudaSuccess ? NVFP4_OK : NVFP4_E_LAUNCH; }

// f(type tag, group size tag)
template <class F> void by_kind(bool f32, const Rows& r, F f) {
  using Warp = std::integral_constant<int, 32>;
  using Cta = std::integral_constant<int, kThreads>;
  if (f32) {
    if (r.vocab <= kWarpRow) f(float(), Warp());
    else f(float(), Cta());
  } else {
    if (r.vocab <= kWarpRow) f(__nv_bfloat16(), Warp());
    else f(__nv_bfloat16(), Cta());
  }
}
template <class L> void forward(const Rows& r, bool f32, L* logp, float* lse, unsigned int* ticket, cudaStream_t stream) {
  by_kind(f32, r, [&](auto t, auto g) {
    forward_kernel<decltype(t), decltype(g)::value, L><<<grid_of(r), kThreads, 0, stream>>>(r, logp, lse, ticket);
  });
}

}  // namespace logprob
}  // namespace nvfp4

using namespace nvfp4::logprob;

extern "C" int nvfp4_logprob_fwd(const nvfp4_logit_rows* in, float* logp, float* lse, void* stream_) {
  Rows r;
  if (const int code = check_rows(in, r); code != NVFP4_OK) return code;
  if (!logp || !lse) return NVFP4_E_NULL;
  if (!aligned(logp, 4) || !aligned(lse, 4)) return NVFP4_E_ALIGN;
  forward(r, in->is_f32 != 0, logp, lse, nullptr, static_cast<cudaStream_t>(stream_));
  return launched();
}

extern "C" int nvfp4_logprob_bwd(const nvfp4_logit_rows* in, const float* lse, const float* weight, int64_t rows_per_weight,
                                 const float* scale, int unless_one, void* dlogits, void* stream_) {
  Rows r;
  if (const int code = check_rows(in, r); code != NVFP4_OK) return code;
  if (!lse || !weight || !dlogits || (unless_one && !scale)) return NVFP4_E_NULL;
  if (rows_per_weight <= 0 || rows_per_weight > 0x7fffffffLL) return NVFP4_E_SHAPE;
  if (!aligned(lse, 4) || !aligned(weight, 4) || !aligned(scale, 4) || !aligned(dlogits, in->is_f32 ? 4 : 2)) return NVFP4_E_ALIGN;
  by_kind(in->is_f32 != 0, r, [&](auto t, auto g) {
    using T = decltype(t);
    backward_kernel<T, decltype(g)::value><<<grid_of(r), kThreads, 0, static_cast<cudaStream_t>(stream_)>>>(
        r, lse, weight, (uint32_t)rows_per_weight, scale, unless_one != 0, static_cast<T*>(dlogits));
  });
  return launched();
}

extern "C" int nvfp4_preference_fwd(const nvfp4_logit_rows* in, const float* ref, double beta, double label_smoothing, double* logp,
                                    float* lse, float* loss, float* rewards, float* weight, void* workspace,
                                    size_t workspace_bytes, void* stream_) {
  Rows r;
  if (const int code = check_rows(in, r); code != NVFP4_OK) return code;
  if (in->batch % 2 != 0) return NVFP4_E_SHAPE;
  if (!ref || !logp || !lse || !loss || !rewards || !weight || !workspace) return NVFP4_E_NULL;
  if (workspace_bytes < NVFP4_LOSS_WORKSPACE) return NVFP4_E_WORKSPACE;
  if (!aligned(ref, 4) || !aligned(logp, 8) || !aligned(lse, 4) || !aligned(loss, 4) || !aligned(rewards, 4) || !aligned(weight, 4) ||
      !aligned(workspace, 16))
    return NVFP4_E_ALIGN;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  unsigned int* ticket = static_cast<unsigned int*>(workspace);
  double* parts = reinterpret_cast<double*>(static_cast<char*>(workspace) + 16);
  forward(r, in->is_f32 != 0, logp, lse, ticket, stream);
  if (const int code = launched(); code != NVFP4_OK) return code;
  const int64_t pairs = in->batch / 2;
  preference_kernel<<<(unsigned)(pairs < NVFP4_LOSS_PARTS ? pairs : NVFP4_LOSS_PARTS), kThreads, 0, stream>>>(
      logp, ref, pairs, r.seq, beta, label_smoothing, parts, ticket, loss, rewards, weight);
  return launched();
}

extern "C" int nvfp4_policy_fwd(const nvfp4_logit_rows* in, const float* old_logp, const float* advantage,
                                int64_t rows_per_advantage, const float* ref_logp, double clip_low, double clip_high, double kl,
                                float* logp, float* lse, float* weight, float* loss, float* stats2, void* dlogits,
                                void* workspace, size_t workspace_bytes, void* stream_) {
  Rows r;
  if (const int code = check_rows(in, r); code != NVFP4_OK) return code;
  if (!old_logp || !advantage || !logp || !lse || !weight || !loss || !stats2 || !workspace) return NVFP4_E_NULL;
  if (rows_per_advantage <= 0 || rows_per_advantage > 0x7fffffffLL) return NVFP4_E_SHAPE;
  if (workspace_bytes < NVFP4_LOSS_WORKSPACE) return NVFP4_E_WORKSPACE;
  if (!aligned(old_logp, 4) || !aligned(advantage, 4) || !aligned(ref_logp, 4) || !aligned(logp, 4) || !aligned(lse, 4) ||
      !aligned(weight, 4) || !aligned(loss, 4) || !aligned(stats2, 4) || !aligned(dlogits, in->is_f32 ? 4 : 2) || !aligned(workspace, 16))
    return NVFP4_E_ALIGN;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (cudaMemsetAsync(workspace, 0, 16, stream) != cudaSuccess) return NVFP4_E_LAUNCH;
  unsigned int* ticket = static_cast<unsigned int*>(workspace);
  unsigned long long* count = static_cast<unsigned long long*>(workspace) + 1;
  const int64_t ctas = (r.rows + kThreads * 4 - 1) / (kThreads * 4);
  count_kernel<<<(unsigned)(ctas < 148 ? ctas : 148), kThreads, 0, stream>>>(r.labels, r.rows, r.ignore, count);
  if (const int code = launched(); code != NVFP4_OK) return code;
  const Policy p{old_logp, ref_logp, advantage, (uint32_t)rows_per_advantage, (float)(1.0 - clip_low),
                 (float)(1.0 + clip_high), (float)kl};
  const PolicyOut o{logp, lse, weight, loss, stats2, reinterpret_cast<double*>(static_cast<char*>(workspace) + 16), ticket};
  by_kind(in->is_f32 != 0, r, [&](auto t, auto g) {
    using T = decltype(t);
    policy_kernel<T, decltype(g)::value><<<grid_of(r), kThreads, 0, stream>>>(r, p, count, o, static_cast<T*>(dlogits));
  });
  return launched();
}
