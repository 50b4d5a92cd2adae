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
// beforehand, and a captured launch keeps its own).  A CTA takes 2048 elements of one tensor at a time, eight consecutive
// ones a thread: 32-byte accesses, and one warp is one 256-element block, whose maximum is one redux per moment.
#include <type_traits>

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
struct Hyper {
  float decay, beta1, rest1, beta2, rest2, step, inv_root, eps;
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

// the tensor that chunk c belongs to
template <int CAP> __device__ __forceinline__ int find(const Table<CAP>& t, uint32_t c) {
  int lo = 0, hi = t.count;                      // start[lo] <= c < start[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.start[mid] <= c) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  asm("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]) : "l"(p) : "memory");
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 q = *reinterpret_cast<const uint4*>(p);
  v[0] = bf16_lo(q.x); v[1] = bf16_hi(q.x); v[2] = bf16_lo(q.y); v[3] = bf16_hi(q.y);
  v[4] = bf16_lo(q.z); v[5] = bf16_hi(q.z); v[6] = bf16_lo(q.w); v[7] = bf16_hi(q.w);
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  asm volatile("st.global.v8.f32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};"
      :: "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "l"(p) : "memory");
}
__device__ __forceinline__ uint32_t pack(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack(v[0], v[1]), pack(v[2], v[3]), pack(v[4], v[5]), pack(v[6], v[7]));
}
__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// eight elements from `at` on, those behind the end as zeros
template <class T> __device__ __forceinline__ void fetch(const T* p, int64_t at, int64_t n, bool whole, float (&v)[8]) {
  if (whole) {
    load8(p + at, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = at + j < n ? as_float(p[at + j]) : 0.0f;
  }
}
template <class T> __device__ __forceinline__ void keep(T* p, int64_t at, int64_t n, bool whole, const float (&v)[8]) {
  if (whole) {
    store8(p + at, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (at + j < n) put(p + at + j, v[j]);
  }
}

// ---- sums of squares -------------------------------------------------------------------------------------------------
// One double per CTA, summed in a fixed order by whoever reads them.  Squares of fp32 are exact in 64 bits and neither
// overflow nor underflow there; at the memory's rate the conversions are a third of what the SM can do.
__device__ __forceinline__ double cta_sum(double s) {
  __shared__ double part[kThreads / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
  __syncthreads();
  s = 0.0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) s += part[w];
  return s;
}

constexpr int kNormCap = 512;
struct NormTable {
  const void* grad[kNormCap];
  int64_t n[kNormCap];
  uint32_t start[kNormCap + 1];
  uint8_t wide[kNormCap];
  int32_t count;
};

template <class T>
__global__ void __launch_bounds__(kThreads) sumsq_kernel(const __grid_constant__ NormTable t, double* __restrict__ parts) {
  double sum = 0.0;
  const uint32_t total = t.start[t.count];
  for (uint32_t c = blockIdx.x; c < total; c += gridDim.x) {
    int lo = 0, hi = t.count;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (t.start[mid] <= c) lo = mid;
      else hi = mid;
    }
    const T* g = static_cast<const T*>(t.grad[lo]);
    const int64_t n = t.n[lo], at = (int64_t)(c - t.start[lo]) * kChunk + threadIdx.x * 8;
    if (at >= n) continue;
    float v[8];
    fetch(g, at, n, t.wide[lo] && at + 8 <= n, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) sum = fma((double)v[j], (double)v[j], sum);
  }
  sum = cta_sum(sum);
  if (threadIdx.x == 0) parts[blockIdx.x] = sum;
}

__device__ __forceinline__ float norm_of(const double* parts, int n) {
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += kThreads) s += parts[i];
  return (float)sqrt(cta_sum(s));
}
__global__ void __launch_bounds__(kThreads) norm_kernel(const double* __restrict__ parts, int n, float* __restrict__ out) {
  const float v = norm_of(parts, n);
  if (threadIdx.x == 0) *out = v;
}

// ---- the step --------------------------------------------------------------------------------------------------------
// E4M3 codes of eight elements -> fp32; f = 2^(e + 49).  The code's exponent and mantissa in bits 20 to 26 make an fp32
// (or a denormal) 2^120 too small; both products are exact.
__device__ __forceinline__ void decode8(uint2 q, uint8_t scale, float (&v)[8]) {
  const float f = scale == 255 ? __uint_as_float(0x7fc00000u) : __uint_as_float(min((uint32_t)scale + 56u, 254u) << 23);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t b = (j < 4 ? q.x : q.y) >> (8 * (j & 3));
    v[j] = (__uint_as_float(((b & 0x80u) << 24) | ((b & 0x7fu) << 20)) * 0x1p64f) * f;
  }
}

// Codes of eight elements under the block's scale, which lane 0 stores; d: 16 random bits each.
__device__ __forceinline__ uint2 encode8(const float (&v)[8], const uint32_t (&d)[8], uint8_t* scale, bool live) {
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
  top = __reduce_max_sync(0xffffffffu, top);
  const uint32_t e = min(max(top >> 23, 27u), 177u);
  // a block with an element of 2^51 or more, an infinity or a NaN is held as NaN
  if (live && (threadIdx.x & 31) == 0) *scale = (top >> 23) > 177u ? 255 : (uint8_t)(e - 7);
  const float h = __uint_as_float((205u - e) << 23);
  uint32_t w[2] = {0u, 0u};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float y = (fabsf(v[j]) * h) * 0x1p-64f;
    const uint32_t code = ((__float_as_uint(y) + (d[j] << 4)) >> 20) & 0x7fu;
    w[j >> 2] |= (code | ((__float_as_uint(v[j]) >> 24) & 0x80u)) << (8 * (j & 3));
  }
  return make_uint2(w[0], w[1]);
}

template <class T, bool EIGHT, int CAP>
__global__ void __launch_bounds__(kThreads) adamw_kernel(const __grid_constant__ Table<CAP> t, const Clip clip,
                                                         const PhiloxKeys keys) {
  float c = 1.0f;
  const bool clipped = clip.parts != nullptr || clip.norm != nullptr;
  if (clipped) {
    const float norm = clip.parts != nullptr ? norm_of(clip.parts, clip.n_parts) : *clip.norm;
    if (blockIdx.x == 0 && threadIdx.x == 0 && clip.norm_out != nullptr) *clip.norm_out = norm;
    c = __fdiv_rn(clip.max_norm, __fadd_rn(norm, 1e-6f));
    c = c > 1.0f ? 1.0f : c;                     // (a NaN stays one)
  }
  const int64_t total = t.start[t.count];
  for (int64_t chunk = total - 1 - blockIdx.x; chunk >= 0; chunk -= gridDim.x) {
    const int k = find(t, (uint32_t)chunk);
    const Entry& e = t.e[k];
    const Hyper& h = t.h[e.hyper];
    const int64_t n = e.n, at = (chunk - t.start[k]) * kChunk + threadIdx.x * 8;
    const bool whole = e.wide && at + 8 <= n;
    T* param = static_cast<T*>(e.param);
    float p[8], g[8], m[8], r[8];
    if (EIGHT) {
      // the warp's block; lanes behind the end of the tensor but inside the block carry zeros, other warps nothing
      if ((at & ~(int64_t)(kBlock - 1)) >= n) continue;
      decode8(*reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(e.first) + at), e.first_scale[at / kBlock], m);
      decode8(*reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(e.second) + at), e.second_scale[at / kBlock], r);
      fetch(param, at, n, whole, p);
      fetch(static_cast<const T*>(e.grad), at, n, whole, g);
#pragma unroll
      for (int j = 0; j < 8; ++j) r[j] = __fmul_rn(r[j], r[j]);
    } else {
      if (at >= n) continue;
      fetch(param, at, n, whole, p);
      fetch(static_cast<const T*>(e.grad), at, n, whole, g);
      fetch(static_cast<const float*>(e.first), at, n, whole, m);
      fetch(static_cast<const float*>(e.second), at, n, whole, r);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (clipped) g[j] = __fmul_rn(g[j], c);
      m[j] = __fadd_rn(__fmul_rn(m[j], h.beta1), __fmul_rn(g[j], h.rest1));
      r[j] = __fadd_rn(__fmul_rn(r[j], h.beta2), __fmul_rn(__fmul_rn(g[j], h.rest2), g[j]));
    }
    if (!EIGHT) {
      keep(static_cast<float*>(e.first), at, n, whole, m);
      keep(static_cast<float*>(e.second), at, n, whole, r);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      r[j] = __fsqrt_rn(r[j]);
      const float ratio = __fdiv_rn(m[j], __fadd_rn(__fmul_rn(r[j], h.inv_root), h.eps));
      p[j] = __fsub_rn(__fmul_rn(p[j], h.decay), __fmul_rn(ratio, h.step));
    }
    keep(param, at, n, whole, p);
    if (EIGHT) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (at + j >= n) m[j] = r[j] = 0.0f;     // (eps 0 or a NaN factor must not reach the block's scale from there)
      const uint64_t group = e.group + (uint64_t)at / 8;
      const Philox4 x = fused::philox_rounds((uint32_t)group, (uint32_t)(group >> 32), (uint32_t)h.offset,
                                             (uint32_t)(h.offset >> 32), keys);
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
      uint32_t d[8], b[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t turned = __brev(w[j]);
        d[2 * j] = w[j] & 0xffffu; d[2 * j + 1] = w[j] >> 16;
        b[2 * j] = turned >> 16; b[2 * j + 1] = turned & 0xffffu;
      }
      const uint2 qm = encode8(m, d, e.first_scale + at / kBlock, true);
      const uint2 qr = encode8(r, b, e.second_scale + at / kBlock, true);
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(e.first) + at) = qm;
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(e.second) + at) = qr;
    }
  }
}

template <int CAP> constexpr bool fits() { return sizeof(Table<CAP>) + sizeof(Clip) + sizeof(PhiloxKeys) <= 32764; }
constexpr int kSmall = 48, kLarge = 400;
static_assert(fits<kLarge>() && sizeof(NormTable) + 8 <= 32764, "kernel parameters are 32764 bytes at most");

inline bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

template <class T, bool EIGHT, int CAP>
int launch(const nvfp4_adamw_tensor* ts, int count, const nvfp4_adamw_hyper* hs, int n_hypers, const Clip& clip,
           const PhiloxKeys& keys, cudaStream_t stream) {
  static_assert(sizeof(T) == 2 || sizeof(T) == 4, "");
  Table<CAP> t;
  uint64_t chunks = 0;
  for (int i = 0; i < count; ++i) {
    const nvfp4_adamw_tensor& s = ts[i];
    const uintptr_t a = sizeof(T) * 8;
    const bool wide = aligned(s.param, a) && aligned(s.grad, a) && (EIGHT || (aligned(s.first, 32) && aligned(s.second, 32)));
    t.e[i] = Entry{s.param, s.grad, s.first, s.second, static_cast<uint8_t*>(s.first_scale),
                   static_cast<uint8_t*>(s.second_scale), s.n, s.counter_base, s.hyper, wide};
    t.start[i] = (uint32_t)chunks;
    chunks += (uint64_t)((s.n + kChunk - 1) / kChunk);
    if (chunks > 0x7fffffffu) return NVFP4_E_LIMIT;
  }
  t.start[count] = (uint32_t)chunks;
  t.count = count;
  for (int i = 0; i < n_hypers; ++i) {
    const nvfp4_adamw_hyper& s = hs[i];
    t.h[i] = Hyper{s.decay, s.beta1, s.rest1, s.beta2, s.rest2, s.step_size, s.inv_root_correction, s.eps, s.philox_offset};
  }
  const unsigned grid = (unsigned)(chunks < 148 * 4 ? chunks : 148 * 4);
  adamw_kernel<T, EIGHT, CAP><<<grid, kThreads, 0, stream>>>(t, clip, keys);
  return cudaGetLastError() == cudaSuccess ? NVFP4_OK : NVFP4_E_LAUNCH;
}

}  // namespace adamw
}  // namespace nvfp4

using namespace nvfp4::adamw;

extern "C" int nvfp4_sumsq_parts(int count, const int64_t* counts) {
  if (count < 0 || (count > 0 && counts == nullptr)) return NVFP4_E_NULL;
  int parts = 0;
  for (int i = 0; i < count; i += kNormCap) {
    uint64_t chunks = 0;
    for (int j = i; j < count && j < i + kNormCap; ++j) {
      if (counts[j] <= 0) return NVFP4_E_SHAPE;
      chunks += (uint64_t)((counts[j] + kChunk - 1) / kChunk);
    }
    if (chunks > 0x7fffffffu) return NVFP4_E_LIMIT;
    parts += (int)(chunks < 148 * 4 ? chunks : 148 * 4);
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
  for (int i = 0; i < count; i += kNormCap) {
    const int m = count - i < kNormCap ? count - i : kNormCap;
    NormTable t;
    uint32_t chunks = 0;
    for (int j = 0; j < m; ++j) {
      t.grad[j] = grads[i + j];
      t.n[j] = counts[i + j];
      t.wide[j] = aligned(grads[i + j], is_f32 ? 32 : 16);
      t.start[j] = chunks;
      chunks += (uint32_t)((counts[i + j] + kChunk - 1) / kChunk);
    }
    t.start[m] = chunks;
    t.count = m;
    const unsigned grid = chunks < 148 * 4 ? chunks : 148 * 4;
    if (is_f32) sumsq_kernel<float><<<grid, kThreads, 0, stream>>>(t, parts);
    else sumsq_kernel<__nv_bfloat16><<<grid, kThreads, 0, stream>>>(t, parts);
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
  for (int i = 0; i < count; ++i) {
    const nvfp4_adamw_tensor& s = tensors[i];
    if (s.n <= 0) return NVFP4_E_SHAPE;
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
  for (int i = 0; i < count; i += kLarge) {
    const int m = count - i < kLarge ? count - i : kLarge;
    const Clip clip{sumsq_parts, norm, n_parts, max_norm, i == 0 ? norm_out : nullptr};
    auto go = [&](auto small) -> int {
      constexpr int cap = decltype(small)::value;
      const nvfp4_adamw_tensor* ts = tensors + i;
      if (is_f32)
        return eight ? launch<float, true, cap>(ts, m, hypers, n_hypers, clip, keys, stream)
                     : launch<float, false, cap>(ts, m, hypers, n_hypers, clip, keys, stream);
      return eight ? launch<__nv_bfloat16, true, cap>(ts, m, hypers, n_hypers, clip, keys, stream)
                   : launch<__nv_bfloat16, false, cap>(ts, m, hypers, n_hypers, clip, keys, stream);
    };
    const int code = m <= kSmall ? go(std::integral_constant<int, kSmall>()) : go(std::integral_constant<int, kLarge>());
    if (code != NVFP4_OK) return code;
  }
  return NVFP4_OK;
}
