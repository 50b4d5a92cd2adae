// AdamW step over many tensors in one launch, moments in 32 bits or in 8, and the norm of all gradients (sm_100a).
//
//   g' = c g (c = min(1, max_norm / (norm + 1e-6)) when the gradients are clipped)
//   m' = b1 m + (1 - b1) g'      v' = b2 v + ((1 - b2) g') g'      r = sqrt(v')
//   p' = p (1 - lr wd) - (lr / (1 - b1^t)) m' / (r / sqrt(1 - b2^t) + eps)
// in fp32, every product, sum, quotient and root rounded by itself, so that the same operations of torch give the same
// bits.
//
// Moments in 8 bits: m and r (the root: it spans half the octaves of v) are E4M3 codes under one power of two per 256
// elements, S = 2^(e - 7) for a block whose largest magnitude lies in [2^e, 2^(e + 1)).  Powers of two, because another
// scale would move every value of the block off the grid and round it again each time the maximum changes.  Codes are
// rounded stochastically: a step moves the root by (1 - b2) / 2 of itself, 5e-4, and a code step is 2^-3 to 2^-4 of the
// value, so rounding to nearest would hold the first root for ever.  |x| times a power of two that puts its exponent on
// E4M3's leaves the code in bits 20 and up of the fp32 word, subnormal codes as fp32 denormals: one integer addition of
// 16 random bits below bit 20 and a shift round it.  Philox runs once per eight elements; the root takes the bits of the
// first moment reversed.
//
// The tensors come as a table in the kernel's parameters (32 KB of constant memory: nothing to allocate, nothing to copy
// beforehand, and a captured launch keeps its own).  A CTA takes one chunk of one tensor, 2048 elements, or with 8-bit
// moments four or five blocks for each warp, eight consecutive ones a thread: 32-byte accesses, and the maximum of a block is
// one redux per moment.
#include <type_traits>

#include <cuda_fp16.h>

#include "quantize_common.cuh"

namespace nvfp4 {
namespace adamw {

using fused::PhiloxKeys;

constexpr int kThreads = 256, kChunk = kThreads * 8, kBlock = 256;
constexpr int kHypers = 8;

struct Entry {
  void* param;
  const void* grad;
  void* first;               // fp32 [n], or E4M3 codes [ceil(n / 256) * 256]
  void* second;
  uint8_t* first_scale;      // E8M0 [ceil(n / 256)]
  uint8_t* second_scale;
  int64_t n;
  uint64_t group;            // counter of its first eight elements
  int32_t hyper;
  int32_t wide;              // every pointer takes 32-byte (16-byte for bf16) accesses
};
struct Hyper {               // each twice, as the packed instructions take them: one load from constant memory, no copies
  float2 decay, beta1, rest1, beta2, rest2, step, inv_root, eps, one;       // step: with its sign
  uint64_t offset;
};
template <int CAP> struct Table {
  Entry e[CAP];
  uint32_t start[CAP + 1];   // first chunk of each tensor, and the chunks in all
  int32_t count;
  Hyper h[kHypers];
};
struct Clip {
  const double* parts;       // sums of squares to add up, or null
  const float* norm;         // the norm itself, or null
  int32_t n_parts;
  float max_norm;
  float* norm_out;           // the norm that was used
};

// The tensor that chunk c belongs to.
template <class Table> __device__ __forceinline__ int find(const Table& t, uint32_t c) {
  int lo = 0, hi = t.count;                      // start[lo] <= c < start[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.start[mid] <= c) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Pairs of fp32 in the two lanes of sm_100's packed instructions.
struct Eight {
  float2 v[4];
  __device__ __forceinline__ float& operator[](int j) { return j & 1 ? v[j >> 1].y : v[j >> 1].x; }
};
// Eight elements as they lie in memory.  They are opened where they are used: a conversion behind the load would wait for
// that load in front of the next one.
template <class T> struct Raw;
template <> struct Raw<float> {
  float w[8];
  __device__ __forceinline__ void load(const float* p) {
    asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
        : "=f"(w[0]), "=f"(w[1]), "=f"(w[2]), "=f"(w[3]), "=f"(w[4]), "=f"(w[5]), "=f"(w[6]), "=f"(w[7]) : "l"(p) : "memory");
  }
  __device__ __forceinline__ void gather(const float* p, int64_t left) {
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = j < left ? p[j] : 0.0f;
  }
  __device__ __forceinline__ Eight open() const {
    return Eight{{make_float2(w[0], w[1]), make_float2(w[2], w[3]), make_float2(w[4], w[5]), make_float2(w[6], w[7])}};
  }
};
template <> struct Raw<__nv_bfloat16> {
  uint32_t w[4];
  __device__ __forceinline__ void load(const __nv_bfloat16* p) {
    asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "l"(p) : "memory");
  }
  __device__ __forceinline__ void gather(const __nv_bfloat16* p, int64_t left) {
    const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      w[j] = (2 * j < left ? (uint32_t)h[2 * j] : 0u) | (2 * j + 1 < left ? (uint32_t)h[2 * j + 1] << 16 : 0u);
  }
  __device__ __forceinline__ Eight open() const {
    Eight x;
#pragma unroll
    for (int j = 0; j < 4; ++j) x.v[j] = make_float2(bf16_lo(w[j]), bf16_hi(w[j]));
    return x;
  }
};
// eight elements from `at` on, those behind the end as zeros
template <class T> __device__ __forceinline__ void fetch(const T* p, int64_t at, int64_t n, bool whole, Raw<T>& x) {
  if (whole) x.load(p + at);
  else x.gather(p + at, n - at);
}

__device__ __forceinline__ void store8(float* p, const Eight& x) {
  asm volatile("st.global.v8.f32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};"
      :: "f"(x.v[0].x), "f"(x.v[0].y), "f"(x.v[1].x), "f"(x.v[1].y), "f"(x.v[2].x), "f"(x.v[2].y), "f"(x.v[3].x),
         "f"(x.v[3].y), "l"(p) : "memory");
}
__device__ __forceinline__ uint32_t pack(float2 a) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a.x, a.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const Eight& x) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack(x.v[0]), pack(x.v[1]), pack(x.v[2]), pack(x.v[3]));
}
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
template <class T> __device__ __forceinline__ void keep(T* p, int64_t at, int64_t n, bool whole, Eight& x) {
  if (whole) {
    store8(p + at, x);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (at + j < n) put(p + at + j, x[j]);
  }
}

// ---- sums of squares -------------------------------------------------------------------------------------------------
// One double per CTA, summed in a fixed order by whoever reads them.  Squares of fp32 are exact in 64 bits and neither
// overflow nor underflow there; at the memory's rate the conversions are a third of what the SM can do.  490 MB of fp32 in
// a training loop, where the L2 is still full of the last step's writes: 88 us with up to 148 * 16 CTAs, 95 with 148 * 4,
// 86 with 148 * 24; every CTA of the step adds their sums up again.
template <int R> __device__ __forceinline__ double cta_sum(double (&s)[R]) {
  __shared__ double part[kThreads / 32];
#pragma unroll
  for (int r = 0; r < R; ++r) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s[r] += __shfl_xor_sync(0xffffffffu, s[r], o);
    if ((threadIdx.x & 31) == 0) part[(threadIdx.x >> 5) + r * (kThreads / R / 32)] = s[r];
  }
  __syncthreads();
  double sum = 0.0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) sum += part[w];
  return sum;
}

constexpr int kNormSmall = 64, kNormLarge = 512, kNormGrid = 148 * 16;
template <int CAP> struct NormTable {
  const void* grad[CAP];
  int64_t n[CAP];
  uint32_t start[CAP + 1];
  uint8_t wide[CAP];
  int32_t count;
};

constexpr int kNormChunk = 4 * kChunk;             // four loads of eight elements in flight in each thread
template <class T, int CAP>
__global__ void __launch_bounds__(kThreads) sumsq_kernel(const __grid_constant__ NormTable<CAP> t, double* __restrict__ parts) {
  double sum[1] = {0.0};
  const uint32_t total = t.start[t.count];
  uint32_t c = blockIdx.x;
  int k = c < total ? find(t, c) : 0;
  for (; c < total; c += gridDim.x) {
    while (t.start[k + 1] <= c) ++k;
    const T* g = static_cast<const T*>(t.grad[k]);
    const int64_t n = t.n[k], at = (int64_t)(c - t.start[k]) * kNormChunk + threadIdx.x * 8;
    const bool wide = t.wide[k];
    Raw<T> x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (at + u * kChunk < n) fetch(g, at + u * kChunk, n, wide && at + u * kChunk + 8 <= n, x[u]);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (at + u * kChunk < n) {
        Eight v = x[u].open();
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[0] = fma((double)v[j], (double)v[j], sum[0]);
      }
  }
  const double all = cta_sum<1>(sum);
  if (threadIdx.x == 0) parts[blockIdx.x] = all;
}

// In the order of kThreads threads, however many there are: the norm has the same bits wherever it is found.
template <int THREADS> __device__ __forceinline__ float norm_of(const double* parts, int n) {
  constexpr int R = kThreads / THREADS;
  double s[R] = {};
  for (int i = threadIdx.x; i < n; i += 5 * kThreads) {      // (half of what one launch leaves is in flight at once)
    double v[5 * R];
#pragma unroll
    for (int u = 0; u < 5 * R; ++u) v[u] = i + u * THREADS < n ? parts[i + u * THREADS] : 0.0;
#pragma unroll
    for (int r = 0; r < R; ++r) s[r] += (v[r] + v[R + r]) + (v[2 * R + r] + v[3 * R + r]) + v[4 * R + r];
  }
  return (float)sqrt(cta_sum<R>(s));
}
__global__ void __launch_bounds__(kThreads) norm_kernel(const double* __restrict__ parts, int n, float* __restrict__ out) {
  const float v = norm_of<kThreads>(parts, n);
  if (threadIdx.x == 0) *out = v;
}

// ---- the step --------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float2 both(float a) { return make_float2(a, a); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
// a + b as a * 1 + b with a 1 that the compiler does not see: nvcc 12.9 and its assembler make one fused multiply-add of a
// packed product and a packed sum, roundings asked for or not
__device__ __forceinline__ float2 add2(float2 a, float2 b, float2 one) { return __ffma2_rn(a, one, b); }
// max(|a|, |b|, |c|), a NaN if one of them is
__device__ __forceinline__ float max3_abs_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(fabsf(a)), "f"(fabsf(b)), "f"(fabsf(c)));
  return r;
}

__device__ __forceinline__ float scale_of(uint32_t e8m0) {
  return __uint_as_float(e8m0 == 255u ? 0x7fc00000u : e8m0 == 0u ? 0x00400000u : e8m0 << 23);
}
// Eight E4M3 codes -> fp32.
__device__ __forceinline__ void decode8(uint2 q, Eight& x) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint16_t two = (uint16_t)((j < 2 ? q.x : q.y) >> (16 * (j & 1)));
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(two));
    x.v[j] = __half22float2(*reinterpret_cast<const __half2*>(&h));
  }
}

// Codes of eight elements under the block's scale, which lane 0 stores.  d: a word for two elements, 16 random bits each; the
// first takes the low ones, or the high ones when the word has been turned round.
template <bool SIGNED, bool TURNED> __device__ __forceinline__ uint2 encode8(Eight x, const uint32_t (&d)[4], uint8_t* scale) {
  constexpr uint32_t kLow = 0x0010u, kHigh = 0x1000u;        // 16 bits times 16 and the others times 0: one dot product
  const float top_f = max3_abs_nan(max3_abs_nan(x[0], x[1], x[2]), x[3], x[4]);
  const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(max3_abs_nan(max3_abs_nan(top_f, x[5], x[6]), x[7], x[7])));
  const uint32_t e = min(max(top >> 23, 27u), 177u);
  // a block with an element of 2^51 or more, an infinity or a NaN is held as NaN
  if ((threadIdx.x & 31) == 0) *scale = (top >> 23) > 177u ? 255 : (uint8_t)(e - 7);
  float2 h = both(__uint_as_float((141u - e) << 23));       // 2^-(113 + its exponent)
  if (e > 140u) {                                            // below fp32's normal numbers: in two steps
    h = both(__uint_as_float((205u - e) << 23));
#pragma unroll
    for (int j = 0; j < 4; ++j) x.v[j] = mul2(x.v[j], both(0x1p-64f));
  }
  uint32_t u[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 y = mul2(x.v[j], h);
    u[2 * j] = __dp2a_lo(d[j], TURNED ? kHigh : kLow, __float_as_uint(y.x));         // (the sign bit stays: the
    u[2 * j + 1] = __dp2a_lo(d[j], TURNED ? kLow : kHigh, __float_as_uint(y.y));     // magnitude ends at bit 26)
  }
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t tops = __byte_perm(u[2 * j], u[2 * j + 1], 0x7632);       // sign, four zeros, code, four bits below it; twice
    w[j] = tops >> 4;
    if (SIGNED) w[j] = (w[j] & 0x007f007fu) | ((tops >> 8) & 0xff80ff80u);
  }
  return make_uint2(__byte_perm(w[0], w[1], 0x6420), __byte_perm(w[2], w[3], 0x6420));
}

// The norm to clip by, 0 without clipping; the first CTA leaves it for the caller.  Loads of the step may stand between this and
// its use: then they do not wait for it.
template <int THREADS> __device__ __forceinline__ float norm_to_clip(const Clip& clip) {
  if (clip.parts == nullptr && clip.norm == nullptr) return 0.0f;
  const float norm = clip.parts != nullptr ? norm_of<THREADS>(clip.parts, clip.n_parts) : *clip.norm;
  if (blockIdx.x == 0 && threadIdx.x == 0 && clip.norm_out != nullptr) *clip.norm_out = norm;
  return norm;
}
// c = min(1, max_norm / (norm + 1e-6)), 1 without clipping
__device__ __forceinline__ float clip_factor(const Clip& clip, float norm) {
  if (clip.parts == nullptr && clip.norm == nullptr) return 1.0f;
  const float c = __fdiv_rn(clip.max_norm, __fadd_rn(norm, 1e-6f));
  return c > 1.0f ? 1.0f : c;                    // (a NaN stays one)
}

// Both kernels go through the chunks last one first: the norm's pass has just read the gradients in their order, and the last
// of them are still in L2.
// 32-bit moments, 124M fp32 parameters: 491 us, 28 bytes each at 7.1 TB/s.  A CTA for each chunk: with four on an SM that go
// through the chunks in turn some SMs are done early, 545 us; with 8, 16, 64 times as many CTAs 511, 504, 496.
template <class T, int CAP>
__global__ void __launch_bounds__(kThreads, 4) adamw_kernel(const __grid_constant__ Table<CAP> t, const Clip clip) {
  const float norm = norm_to_clip<kThreads>(clip);
  const uint32_t chunk = t.start[t.count] - 1 - blockIdx.x;
  const int k = find(t, chunk);
  const Entry& e = t.e[k];
  const Hyper& h = t.h[e.hyper];
  const int64_t n = e.n, at = (int64_t)(chunk - t.start[k]) * kChunk + threadIdx.x * 8;
  if (at >= n) return;
  const bool whole = e.wide && at + 8 <= n;
  Raw<T> param, grad;
  Raw<float> first, second;
  fetch(static_cast<const T*>(e.param), at, n, whole, param);
  fetch(static_cast<const T*>(e.grad), at, n, whole, grad);
  fetch(static_cast<const float*>(e.first), at, n, whole, first);
  fetch(static_cast<const float*>(e.second), at, n, whole, second);
  const float c = clip_factor(clip, norm);
  Eight p = param.open(), g = grad.open(), m = first.open(), v = second.open();
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 gg = mul2(g.v[j], both(c));                 // (by 1 when nothing is clipped)
    m.v[j] = add2(mul2(m.v[j], h.beta1), mul2(gg, h.rest1), h.one);
    v.v[j] = add2(mul2(v.v[j], h.beta2), mul2(mul2(gg, h.rest2), gg), h.one);
  }
  keep(static_cast<float*>(e.first), at, n, whole, m);
  keep(static_cast<float*>(e.second), at, n, whole, v);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 root = make_float2(__fsqrt_rn(v.v[j].x), __fsqrt_rn(v.v[j].y));
    const float2 below = add2(mul2(root, h.inv_root), h.eps, h.one);
    const float2 ratio = make_float2(__fdiv_rn(m.v[j].x, below.x), __fdiv_rn(m.v[j].y, below.y));
    p.v[j] = add2(mul2(p.v[j], h.decay), mul2(ratio, h.step), h.one);
  }
  keep(static_cast<T*>(e.param), at, n, whole, p);
}

// Roots of two numbers: the approximate reciprocal root and one Newton step with the exact residual (Markstein 1990), which gives
// the correctly rounded root but for cases too close to call in 44 bits.  The smallest normal number is added for zero's sake,
// whose root is zero; from 2^-100 on that changes nothing, and a root under 2^-50 is nothing beside any eps.
__device__ __forceinline__ float2 roots(float2 x) {
  float2 y;
  const float2 z = __fadd2_rn(x, both(0x1p-126f));
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y.x) : "f"(z.x));
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y.y) : "f"(z.y));
  const float2 r = __fmul2_rn(x, y), minus_half = __fmul2_rn(y, both(-0.5f));
  return __ffma2_rn(__ffma2_rn(r, r, __fmul2_rn(x, both(-1.0f))), minus_half, r);
}
__device__ __forceinline__ float reciprocal_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// The same step on 8-bit moments.  It is bound by instructions as much as by memory (75 for an element with the arithmetic
// above, 16 or 10 bytes).  The moments keep that arithmetic, so that the codes are those of its definition; in the update the
// quotient is a product with the approximate reciprocal, and products are fused with their sums: 2^-21 of an update.  The scale
// of the first moment goes into beta1, and a dot product of 16-bit halves adds an element's share of a random word.
// 124M fp32 parameters 281 us (7.0 TB/s), 222M bf16 ones 421 (5.3).
//
// A warp takes four blocks in a row of fp32 parameters, five of bf16, as many as fit in 128 registers, with the loads of all
// of them in flight before the first is worked on; the table, the constants and the addresses are worked out once for them.  A
// CTA takes one such chunk and goes, so that its registers go to the loads of the next one while its neighbours compute: eight
// CTAs of two warps on an SM.  (CTAs that stay and go from chunk to chunk: 364 and 474.  CTAs of 128 threads 285 and 441, of 32
// 280 and 431; two fp32 blocks 348, three 304, five 308 with spills; four bf16 blocks 432, six 435 with spills; nine CTAs of 96
// registers 337 and 427, six of 160 294 and 459.)
template <class T> constexpr int kRun = sizeof(T) == 4 ? 4 : 5;
constexpr int kThreads8 = 64;
template <class T> constexpr int kChunk8 = kRun<T> * kThreads8 * 8;
template <class T> struct Item8 {
  Raw<T> param, grad;
  uint2 first, second;
  uint32_t first_scale, second_scale;
};
// The step of one block: x in; p, the codes and the scales (at `first_scale` and `second_scale`) out.  left: elements from this
// thread's first to the end of the tensor.
template <class T>
__device__ __forceinline__ void step8(const Item8<T>& x, const Hyper& h, float c, const PhiloxKeys& keys, uint64_t group, int64_t left,
                                      Eight& p, uint8_t* first, uint8_t* second, uint8_t* first_scale, uint8_t* second_scale) {
  Eight m, r;
  p = x.param.open();
  const Eight g8 = x.grad.open();
  decode8(x.first, m);
  decode8(x.second, r);
  const float scale_r = scale_of(x.second_scale);
  const float2 scaled_beta1 = __fmul2_rn(both(scale_of(x.first_scale)), h.beta1);      // (exact: encode8 makes powers of two of 2^-107 and more)
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 g = __fmul2_rn(g8.v[j], both(c));
    m.v[j] = add2(mul2(m.v[j], scaled_beta1), mul2(g, h.rest1), h.one);
    r.v[j] = mul2(r.v[j], both(scale_r));
    r.v[j] = roots(add2(mul2(mul2(r.v[j], r.v[j]), h.beta2), mul2(mul2(g, h.rest2), g), h.one));
    const float2 below = __ffma2_rn(r.v[j], h.inv_root, h.eps);
    const float2 ratio = __fmul2_rn(m.v[j], make_float2(reciprocal_approx(below.x), reciprocal_approx(below.y)));
    p.v[j] = __ffma2_rn(ratio, h.step, __fmul2_rn(p.v[j], h.decay));
  }
  if (left < 8) {                                            // (eps 0 or a NaN factor must not reach the block's scale from there)
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j >= left) m[j] = r[j] = 0.0f;
  }
  const Philox4 y = fused::philox_rounds((uint32_t)group, (uint32_t)(group >> 32), (uint32_t)h.offset,
                                         (uint32_t)(h.offset >> 32), keys);
  const uint32_t d[4] = {y.x, y.y, y.z, y.w}, b[4] = {__brev(y.x), __brev(y.y), __brev(y.z), __brev(y.w)};
  *reinterpret_cast<uint2*>(first) = encode8<true, false>(m, d, first_scale);
  *reinterpret_cast<uint2*>(second) = encode8<false, true>(r, b, second_scale);
}

template <class T, int CAP>
__global__ void __launch_bounds__(kThreads8, 8) adamw8_kernel(const __grid_constant__ Table<CAP> t, const Clip clip,
                                                               const PhiloxKeys keys) {
  const float norm = norm_to_clip<kThreads8>(clip);
  const uint32_t chunk = t.start[t.count] - 1 - blockIdx.x;
  const int k = find(t, chunk);
  const Entry& e = t.e[k];
  const Hyper& h = t.h[e.hyper];
  const int64_t n = e.n, run = (int64_t)(chunk - t.start[k]) * kChunk8<T> + (threadIdx.x >> 5) * (kRun<T> * kBlock);
  const int64_t at = run + (threadIdx.x & 31) * 8;
  if (run >= n) return;
  T* param = static_cast<T*>(e.param) + at;
  const T* grad = static_cast<const T*>(e.grad) + at;
  uint8_t *first = static_cast<uint8_t*>(e.first) + at, *second = static_cast<uint8_t*>(e.second) + at;
  uint8_t *first_scale = e.first_scale + run / kBlock, *second_scale = e.second_scale + run / kBlock;
  const uint64_t group = e.group + (uint64_t)at / 8;
  Eight p;
  if (e.wide && run + kRun<T> * kBlock <= n) {
    Item8<T> x[kRun<T>];
#pragma unroll
    for (int u = 0; u < kRun<T>; ++u) {
      x[u].first = *reinterpret_cast<const uint2*>(first + u * kBlock);
      x[u].second = *reinterpret_cast<const uint2*>(second + u * kBlock);
      x[u].first_scale = first_scale[u];
      x[u].second_scale = second_scale[u];
      x[u].param.load(param + u * kBlock);
      x[u].grad.load(grad + u * kBlock);
    }
    const float c = clip_factor(clip, norm);
#pragma unroll
    for (int u = 0; u < kRun<T>; ++u) {
      step8<T>(x[u], h, c, keys, group + u * (kBlock / 8), 8, p, first + u * kBlock, second + u * kBlock, first_scale + u,
               second_scale + u);
      store8(param + u * kBlock, p);
    }
  } else {                                                   // a run that ends in it, or one that lies off the vectors' boundaries
    const float c = clip_factor(clip, norm);
#pragma unroll 1
    for (int u = 0; u < kRun<T> && run + u * kBlock < n; ++u) {
      const int64_t left = n - at - u * kBlock;              // lanes behind the end but inside the block carry zeros
      const bool whole = e.wide && left >= 8;
      Item8<T> x;
      fetch(param + u * kBlock, 0, left, whole, x.param);
      fetch(grad + u * kBlock, 0, left, whole, x.grad);
      x.first = *reinterpret_cast<const uint2*>(first + u * kBlock);
      x.second = *reinterpret_cast<const uint2*>(second + u * kBlock);
      x.first_scale = first_scale[u];
      x.second_scale = second_scale[u];
      step8<T>(x, h, c, keys, group + u * (kBlock / 8), left, p, first + u * kBlock, second + u * kBlock, first_scale + u,
               second_scale + u);
      keep(param + u * kBlock, 0, left, whole, p);
    }
  }
}

template <int CAP> constexpr bool fits() { return sizeof(Table<CAP>) + sizeof(Clip) + sizeof(PhiloxKeys) <= 32764; }
constexpr int kSmall = 64, kLarge = 400;
// Parameters from which the norm is found in front of the step on 8-bit moments, by one launch for all its many CTAs (16M 59 us
// instead of 60, 124M 3 + 281 instead of 318; below, the launch costs more than it saves: 8M 33 instead of 32, 4M 23, not 21).
// The step on 32-bit moments has twice the warps on an SM to hide the sum behind (124M 495 us, 493 with it in front).
constexpr double kNormFirst = 12e6;
static_assert(fits<kLarge>() && sizeof(NormTable<kNormLarge>) + 8 <= 32764, "kernel parameters are 32764 bytes at most");

inline bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

template <class T, bool EIGHT, int CAP>
int launch_step(const nvfp4_adamw_tensor* ts, int count, const nvfp4_adamw_hyper* hs, int n_hypers, const Clip& clip,
           const PhiloxKeys& keys, cudaStream_t stream) {
  constexpr int chunk = EIGHT ? kChunk8<T> : kChunk;
  Table<CAP> t;
  uint64_t chunks = 0;
  for (int i = 0; i < count; ++i) {
    const nvfp4_adamw_tensor& s = ts[i];
    const uintptr_t a = sizeof(T) * 8;
    const bool wide = aligned(s.param, a) && aligned(s.grad, a) && (EIGHT || (aligned(s.first, 32) && aligned(s.second, 32)));
    t.e[i] = Entry{s.param, s.grad, s.first, s.second, static_cast<uint8_t*>(s.first_scale),
                   static_cast<uint8_t*>(s.second_scale), s.n, s.counter_base, s.hyper, wide};
    t.start[i] = (uint32_t)chunks;
    chunks += (uint64_t)((s.n + chunk - 1) / chunk);
    if (chunks > 0x7fffffffu) return NVFP4_E_LIMIT;
  }
  t.start[count] = (uint32_t)chunks;
  t.count = count;
  for (int i = 0; i < n_hypers; ++i) {
    const nvfp4_adamw_hyper& s = hs[i];
    auto two = [](float a) { return make_float2(a, a); };
    t.h[i] = Hyper{two(s.decay), two(s.beta1), two(s.rest1), two(s.beta2), two(s.rest2), two(-s.step_size),
                   two(s.inv_root_correction), two(s.eps), two(1.0f), s.philox_offset};
  }
  if constexpr (EIGHT) adamw8_kernel<T, CAP><<<(unsigned)chunks, kThreads8, 0, stream>>>(t, clip, keys);
  else adamw_kernel<T, CAP><<<(unsigned)chunks, kThreads, 0, stream>>>(t, clip);
  return cudaGetLastError() == cudaSuccess ? NVFP4_OK : NVFP4_E_LAUNCH;
}

// The CTAs that were launched, which is how many parts they leave.
template <int CAP>
int launch_sumsq(const void* const* grads, const int64_t* counts, int m, bool f32, double* parts, cudaStream_t stream) {
  NormTable<CAP> t;
  uint32_t chunks = 0;
  for (int j = 0; j < m; ++j) {
    t.grad[j] = grads[j];
    t.n[j] = counts[j];
    t.wide[j] = aligned(grads[j], f32 ? 32 : 16);
    t.start[j] = chunks;
    chunks += (uint32_t)((counts[j] + kNormChunk - 1) / kNormChunk);
  }
  t.start[m] = chunks;
  t.count = m;
  const int grid = chunks < kNormGrid ? (int)chunks : kNormGrid;
  if (f32) sumsq_kernel<float, CAP><<<grid, kThreads, 0, stream>>>(t, parts);
  else sumsq_kernel<__nv_bfloat16, CAP><<<grid, kThreads, 0, stream>>>(t, parts);
  return grid;
}

}  // namespace adamw
}  // namespace nvfp4

using namespace nvfp4::adamw;

extern "C" int nvfp4_sumsq_parts(int count, const int64_t* counts) {
  if (count < 0 || (count > 0 && counts == nullptr)) return NVFP4_E_NULL;
  int parts = 0;
  for (int i = 0; i < count; i += kNormLarge) {
    uint64_t chunks = 0;
    for (int j = i; j < count && j < i + kNormLarge; ++j) {
      if (counts[j] <= 0) return NVFP4_E_SHAPE;
      chunks += (uint64_t)((counts[j] + kNormChunk - 1) / kNormChunk);
    }
    if (chunks > 0x7fffffffu) return NVFP4_E_LIMIT;
    parts += (int)(chunks < kNormGrid ? chunks : kNormGrid);
  }
  return parts;
}

extern "C" int nvfp4_sumsq(const void* const* grads, const int64_t* counts, int count, int is_f32, double* parts,
                           void* stream_) {
  if (count <= 0) return NVFP4_E_SHAPE;
  if (!grads || !counts || !parts) return NVFP4_E_NULL;
  if (!aligned(parts, 8)) return NVFP4_E_ALIGN;
  if (const int all = nvfp4_sumsq_parts(count, counts); all < 0) return all;
  for (int i = 0; i < count; ++i) {
    if (!grads[i]) return NVFP4_E_NULL;
    if (!aligned(grads[i], is_f32 ? 4 : 2)) return NVFP4_E_ALIGN;
  }
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  for (int i = 0; i < count; i += kNormLarge) {
    const int m = count - i < kNormLarge ? count - i : kNormLarge;
    const int grid = m <= kNormSmall ? launch_sumsq<kNormSmall>(grads + i, counts + i, m, is_f32 != 0, parts, stream)
                                     : launch_sumsq<kNormLarge>(grads + i, counts + i, m, is_f32 != 0, parts, stream);
    if (cudaGetLastError() != cudaSuccess) return NVFP4_E_LAUNCH;
    parts += grid;
  }
  return NVFP4_OK;
}

extern "C" int nvfp4_norm_of_sumsq(const double* parts, int n_parts, float* norm, void* stream_) {
  if (!parts || !norm) return NVFP4_E_NULL;
  if (n_parts <= 0) return NVFP4_E_SHAPE;
  if (!aligned(parts, 8) || !aligned(norm, 4)) return NVFP4_E_ALIGN;
  norm_kernel<<<1, kThreads, 0, static_cast<cudaStream_t>(stream_)>>>(parts, n_parts, norm);
  return cudaGetLastError() == cudaSuccess ? NVFP4_OK : NVFP4_E_LAUNCH;
}

extern "C" int nvfp4_adamw(const nvfp4_adamw_tensor* tensors, int count, const nvfp4_adamw_hyper* hypers, int n_hypers,
                           int is_f32, int state_bits, uint64_t philox_seed, const double* sumsq_parts, int n_parts,
                           const float* norm, float max_norm, float* norm_out, void* stream_) {
  if (count <= 0 || n_hypers <= 0) return NVFP4_E_SHAPE;
  if (!tensors || !hypers) return NVFP4_E_NULL;
  if (state_bits != 8 && state_bits != 32) return NVFP4_E_MODE;
  if (n_hypers > kHypers) return NVFP4_E_LIMIT;
  if (sumsq_parts != nullptr && (norm != nullptr || n_parts <= 0)) return NVFP4_E_MODE;
  if (!aligned(sumsq_parts, 8) || !aligned(norm, 4) || !aligned(norm_out, 4)) return NVFP4_E_ALIGN;
  const bool eight = state_bits == 8;
  double elements = 0.0;
  for (int i = 0; i < count; ++i) {
    const nvfp4_adamw_tensor& s = tensors[i];
    if (s.n <= 0) return NVFP4_E_SHAPE;
    elements += (double)s.n;
    if (!s.param || !s.grad || !s.first || !s.second || (eight && (!s.first_scale || !s.second_scale))) return NVFP4_E_NULL;
    if (s.hyper < 0 || s.hyper >= n_hypers) return NVFP4_E_MODE;
    const uintptr_t a = is_f32 ? 4 : 2;
    if (!aligned(s.param, a) || !aligned(s.grad, a) || !aligned(s.first, eight ? 8 : 4) || !aligned(s.second, eight ? 8 : 4))
      return NVFP4_E_ALIGN;
  }
  PhiloxKeys keys;
  for (int r = 0; r < 10; ++r) {
    keys.k[r][0] = (uint32_t)philox_seed + (uint32_t)r * 0x9E3779B9u;
    keys.k[r][1] = (uint32_t)(philox_seed >> 32) + (uint32_t)r * 0xBB67AE85u;
  }
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (eight && sumsq_parts != nullptr && norm_out != nullptr && elements > kNormFirst) {
    norm_kernel<<<1, kThreads, 0, stream>>>(sumsq_parts, n_parts, norm_out);
    if (cudaGetLastError() != cudaSuccess) return NVFP4_E_LAUNCH;
    norm = norm_out;
    sumsq_parts = nullptr;
  }
  for (int i = 0; i < count; i += kLarge) {
    const int m = count - i < kLarge ? count - i : kLarge;
    const Clip clip{sumsq_parts, norm, n_parts, max_norm, i == 0 && norm_out != norm ? norm_out : nullptr};
    auto go = [&](auto small) -> int {
      constexpr int cap = decltype(small)::value;
      const nvfp4_adamw_tensor* ts = tensors + i;
      if (is_f32)
        return eight ? launch_step<float, true, cap>(ts, m, hypers, n_hypers, clip, keys, stream)
                     : launch_step<float, false, cap>(ts, m, hypers, n_hypers, clip, keys, stream);
      return eight ? launch_step<__nv_bfloat16, true, cap>(ts, m, hypers, n_hypers, clip, keys, stream)
                   : launch_step<__nv_bfloat16, false, cap>(ts, m, hypers, n_hypers, clip, keys, stream);
    };
    const int code = m <= kSmall ? go(std::integral_constant<int, kSmall>()) : go(std::integral_constant<int, kLarge>());
    if (code != NVFP4_OK) return code;
  }
  return NVFP4_OK;
}
