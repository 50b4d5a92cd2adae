// Host side of the quantizer, GEMM and optimizer entry points: argument handling, output allocation, stream lookup and
// the calls into libnvfp4_b200.so, in C++.  quant.py, gemm.py and optim.py keep the public functions, their defaults and
// the seed counter and call in here.
//
// Why native: the small calls of this path are bound by the host.  One quantization took 25 us through Python (a
// device context manager, three torch.empty, a ctypes call with sixteen arguments) for 6 us of kernel, an FP4Linear
// step of 512 tokens 484 us for 74 us of kernels.
#include <dlfcn.h>

#include <cmath>
#include <mutex>
#include <unordered_map>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/utils/pybind.h>

#include "nvfp4_b200.h"

namespace py = pybind11;

namespace {

#define NVFP4_FOR_EACH(F)                                                                                              \
  F(nvfp4_amax_bf16) F(nvfp4_amax_both_bf16) F(nvfp4_quantize_fused_bf16) F(nvfp4_quantize_shard_bf16)                 \
  F(nvfp4_quantize_weight_bf16) F(nvfp4_quantize_dual_bf16) F(nvfp4_round_amax_f32) F(nvfp4_gemm) F(nvfp4_gemm_amax) \
  F(nvfp4_gemm_bf16_as_f32) F(nvfp4_adamw) F(nvfp4_sumsq) F(nvfp4_sumsq_parts) F(nvfp4_norm_of_sumsq)       \
  F(nvfp4_logprob_fwd) F(nvfp4_logprob_bwd) F(nvfp4_preference_fwd) F(nvfp4_preference_fwd_ref64)               \
  F(nvfp4_policy_fwd) F(nvfp4_status_string)

struct Library {
#define F(name) decltype(&::name) name = nullptr;
  NVFP4_FOR_EACH(F)
#undef F
} lib;

// Python callables of _lib.py: check(code, what) and cuda_device_of(*tensors), which raise the package's exceptions
py::object* g_check = nullptr;
py::object* g_device_of = nullptr;

void init(const std::string& path, py::object check, py::object device_of) {
  void* h = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);
  if (h == nullptr) throw std::runtime_error(std::string("dlopen failed: ") + dlerror());
#define F(name)                                                                        \
  lib.name = reinterpret_cast<decltype(lib.name)>(dlsym(h, #name));                     \
  if (lib.name == nullptr) throw std::runtime_error(path + " does not export " #name);
  NVFP4_FOR_EACH(F)
#undef F
  g_check = new py::object(std::move(check));          // live as long as the process
  g_device_of = new py::object(std::move(device_of));
}

void check(int code, const char* what) {
  if (code != 0) (*g_check)(code, what);
}

[[noreturn]] void raise(PyObject* type, const std::string& msg) {
  if (!PyGILState_Check()) throw std::runtime_error(msg);      // a node of the backward pass, on autograd's thread
  PyErr_SetString(type, msg.c_str());
  throw py::error_already_set();
}

using OptTensor = c10::optional<at::Tensor>;

const at::Tensor* ptr_of(const OptTensor& t) { return t.has_value() ? &*t : nullptr; }

// The one CUDA device of all operands; anything else goes to _lib.cuda_device_of, which says what is wrong.
c10::Device device_of(std::initializer_list<const at::Tensor*> ts) {
  c10::optional<c10::Device> dev;
  bool good = true;
  for (const at::Tensor* t : ts) {
    if (t == nullptr) continue;
    if (!t->is_cuda() || (dev.has_value() && *dev != t->device())) { good = false; break; }
    dev = t->device();
  }
  if (!good || !dev.has_value()) {
    if (!PyGILState_Check()) throw std::runtime_error("operands are not on one CUDA device");
    py::list l;
    for (const at::Tensor* t : ts) {
      if (t == nullptr) l.append(py::none());
      else l.append(py::cast(*t));
    }
    (*g_device_of)(*l);
    throw std::runtime_error("operands are not on one CUDA device");
  }
  return *dev;
}

void* stream_of(c10::Device dev) { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }

// ---- scratch words ----------------------------------------------------------------------------------------------
struct Key {
  int device;
  void* stream;
  bool operator==(const Key& o) const { return device == o.device && stream == o.stream; }
};
struct KeyHash {
  size_t operator()(const Key& k) const { return std::hash<void*>()(k.stream) * 31 + (size_t)k.device; }
};
std::mutex g_mutex;
// never destroyed: tensors must not be freed after the CUDA context is gone
auto& g_workspaces = *new std::unordered_map<Key, at::Tensor, KeyHash>();
auto& g_status = *new std::unordered_map<int, at::Tensor>();
auto& g_ones = *new std::unordered_map<int, at::Tensor>();

// The entry of `key`, made by `make` if there is none.  The lock is not held while it is made: a dispatch mode may run Python
// there, which can give up the GIL or come back in here.  Of two tensors made at once the first one in stays.
template <class Map, class Make> at::Tensor find_or_make(Map& map, const typename Map::key_type& key, Make make) {
  {
    std::lock_guard<std::mutex> lock(g_mutex);
    const auto it = map.find(key);
    if (it != map.end()) return it->second;
  }
  at::Tensor made = make();
  std::lock_guard<std::mutex> lock(g_mutex);
  return map.emplace(key, std::move(made)).first->second;
}

at::TensorOptions on(c10::Device dev, at::ScalarType t) { return at::TensorOptions().device(dev).dtype(t); }

// 64-byte scratch of the single-launch quantizer, zeroed once, one per (device, stream): every launch leaves it ready
// for the next, and launches on one stream never overlap
at::Tensor workspace(int device) {
  const c10::Device dev(c10::kCUDA, (c10::DeviceIndex)device);
  const Key key{device, stream_of(dev)};
  return find_or_make(g_workspaces, key, [&] { return at::zeros({16}, on(dev, at::kInt)); });
}
// the workspace of the current stream if there is one yet
OptTensor workspace_if_any(int device) {
  const Key key{device, stream_of(c10::Device(c10::kCUDA, (c10::DeviceIndex)device))};
  std::lock_guard<std::mutex> lock(g_mutex);
  auto it = g_workspaces.find(key);
  return it == g_workspaces.end() ? OptTensor() : OptTensor(it->second);
}
at::Tensor status_word(int device) {
  return find_or_make(g_status, device,
                      [&] { return at::zeros({1}, on(c10::Device(c10::kCUDA, (c10::DeviceIndex)device), at::kInt)); });
}

at::Tensor signs_on(const OptTensor& signs, c10::Device dev) {
  if (!signs.has_value()) return find_or_make(g_ones, dev.index(), [&] { return at::ones({16}, on(dev, at::kFloat)); });
  at::Tensor s = *signs;
  if (s.device() != dev || s.scalar_type() != at::kFloat) s = s.to(dev, at::kFloat);
  s = s.contiguous();
  if (s.numel() != 16) raise(PyExc_ValueError, "signs must have 16 entries");
  return s;
}

void check_matrix(const at::Tensor& t) {
  if (t.dim() != 2) raise(PyExc_ValueError, "expected a 2-D tensor");
  if (!t.is_cuda()) device_of({&t});
}
// rows the kernels can read: unit column stride, a row pitch of 16-byte multiples, a 16-byte aligned start
bool readable_rows(const at::Tensor& x) {
  return x.stride(1) == 1 && x.stride(0) * x.element_size() % 16 == 0 && x.stride(0) >= x.size(1) &&
         reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0;
}
at::Tensor as_bf16_rows(const at::Tensor& t) {
  check_matrix(t);
  const at::Tensor x = t.scalar_type() == at::kBFloat16 ? t : t.to(at::kBFloat16);
  return readable_rows(x) ? x : x.contiguous();
}

// An fp32 matrix whose bf16 rounding and maximum (both maxima with signs: after the Hadamard transform along the rows
// too) one kernel finds: (bf16 copy, maxima).  For shapes that the kernel takes and memory it can read as it is: the
// cast of any other matrix makes an aligned copy, where an fp32 copy in front of this kernel would be a pass more.
bool can_round(const at::Tensor& t, bool rht) {
  return t.scalar_type() == at::kFloat && t.size(0) > 0 && t.size(1) > 0 && t.size(1) % 8 == 0 &&
         (!rht || t.size(0) % 16 == 0) && t.size(0) <= 64 * 65535LL && readable_rows(t) && !t.is_neg();
}
std::pair<at::Tensor, at::Tensor> round_amax(const at::Tensor& x, const at::Tensor* signs) {
  const c10::Device dev = device_of({&x, signs});
  at::Tensor out = at::empty({x.size(0), x.size(1)}, on(dev, at::kBFloat16));
  at::Tensor maxima = at::empty({signs != nullptr ? 2 : 1}, on(dev, at::kFloat));
  check(lib.nvfp4_round_amax_f32(static_cast<const float*>(x.data_ptr()), x.size(0), x.size(1), x.stride(0), out.data_ptr(),
                                 signs != nullptr ? static_cast<const float*>(signs->data_ptr()) : nullptr,
                                 static_cast<float*>(maxima.data_ptr()), 1, stream_of(dev)),
        "nvfp4_round_amax_f32");
  return {out, maxima};
}

struct Operand {
  at::Tensor q, s, p;
  uint8_t* qp() { return q.data_ptr<uint8_t>(); }
  uint8_t* sp() { return static_cast<uint8_t*>(s.data_ptr()); }
  float* pp() { return p.data_ptr<float>(); }
};
Operand alloc(c10::Device dev, int64_t m, int64_t k, bool scalar = true) {
  Operand o;
  o.q = at::empty({m, k / 2}, on(dev, at::kByte));
  o.s = at::empty({(m + 127) / 128 * 128, (k / 16 + 3) / 4 * 4}, on(dev, at::kFloat8_e4m3fn));
  if (scalar) o.p = at::empty({}, on(dev, at::kFloat));
  return o;
}

float* float_ptr(const at::Tensor& t) { return static_cast<float*>(t.data_ptr()); }

at::Tensor amax_rows(const at::Tensor& x, bool rht, const at::Tensor* sg, bool transpose, const OptTensor& out) {
  const at::Tensor a = out.has_value() ? *out : at::empty({1}, on(x.device(), at::kFloat));
  const c10::Device dev = device_of({&x, &a, sg});
  check(lib.nvfp4_amax_bf16(x.data_ptr(), x.size(0), x.size(1), x.stride(0), rht, transpose,
                            rht ? float_ptr(*sg) : nullptr, float_ptr(a), 1, stream_of(dev)),
        "nvfp4_amax_bf16");
  return a;
}

at::Tensor amax(const at::Tensor& t, bool rht, const OptTensor& signs, bool transpose, const OptTensor& out) {
  check_matrix(t);
  const c10::cuda::CUDAGuard guard(t.device());
  const at::Tensor x = as_bf16_rows(t);
  at::Tensor sg;
  if (rht) sg = signs_on(signs, x.device());
  return amax_rows(x, rht, rht ? &sg : nullptr, transpose, out);
}

at::Tensor amax_both_rows(const at::Tensor& x, const at::Tensor& sg) {
  const c10::Device dev = device_of({&x, &sg});
  at::Tensor m = at::empty({2}, on(dev, at::kFloat));
  check(lib.nvfp4_amax_both_bf16(x.data_ptr(), x.size(0), x.size(1), x.stride(0), float_ptr(sg), float_ptr(m), 1,
                                 stream_of(dev)),
        "nvfp4_amax_both_bf16");
  return m;
}

at::Tensor amax_both(const at::Tensor& t, const OptTensor& signs) {
  check_matrix(t);
  const c10::cuda::CUDAGuard guard(t.device());
  const at::Tensor x = as_bf16_rows(t);
  return amax_both_rows(x, signs_on(signs, x.device()));
}

// shard: pitch and base number the blocks; otherwise the tensor is whole
py::tuple quantize(const at::Tensor& t, bool stochastic, bool rht, const OptTensor& signs, uint64_t seed, bool transpose,
                   const OptTensor& amax_in, uint64_t offset, bool fused, bool shard, uint64_t pitch, uint64_t base) {
  check_matrix(t);
  const c10::cuda::CUDAGuard guard(t.device());
  // fp32 without a known maximum: the rounding finds it on the way.  Row-wise the single-launch kernel needs no pass of
  // its own for it, so there this pays only from 4M elements on (one read of the bf16 copy against one more launch).
  at::Tensor x, found;
  if (!amax_in.has_value() && !rht && fused && can_round(t, false) && (transpose || t.numel() >= (1 << 22)))
    std::tie(x, found) = round_amax(t, nullptr);
  else
    x = as_bf16_rows(t);
  const at::Tensor* known = amax_in.has_value() ? &*amax_in : (found.defined() ? &found : nullptr);
  const int64_t rows = x.size(0), cols = x.size(1), m = transpose ? cols : rows, k = transpose ? rows : cols;
  if (k % 16 != 0) raise(PyExc_AssertionError, "K=" + std::to_string(k) + " must be divisible by 16");
  at::Tensor sg;
  if (rht) sg = signs_on(signs, x.device());
  const c10::Device dev = device_of({&x, rht ? &sg : nullptr, known});
  Operand o = alloc(dev, m, k);
  void* stream = stream_of(dev);
  const float* sgp = rht ? float_ptr(sg) : nullptr;
  if (fused && known == nullptr && !transpose && rows * (cols / 16) < (1LL << 31)) {
    at::Tensor ws = workspace(dev.index());
    check(lib.nvfp4_quantize_fused_bf16(x.data_ptr(), rows, cols, x.stride(0), stochastic, rht, sgp, seed, offset, o.qp(),
                                        o.sp(), o.pp(), ws.data_ptr(), 64, stream),
          "nvfp4_quantize_fused_bf16");
    return py::make_tuple(o.q, o.s, o.p);
  }
  const at::Tensor a = known != nullptr ? *known : amax_rows(x, rht, rht ? &sg : nullptr, transpose, OptTensor());
  check(lib.nvfp4_quantize_shard_bf16(x.data_ptr(), rows, cols, x.stride(0), transpose, stochastic, rht, sgp, float_ptr(a),
                                      seed, offset, shard ? pitch : (uint64_t)(k / 16), shard ? base : 0, o.qp(),
                                      o.sp(), o.pp(), stream),
        "nvfp4_quantize_shard_bf16");
  return py::make_tuple(o.q, o.s, o.p);
}

// (q, scales) of w and of w^T and their one per-tensor scale
py::tuple quantize_weight(const at::Tensor& w, const OptTensor& amax_in, bool two_d) {
  check_matrix(w);
  const c10::cuda::CUDAGuard guard(w.device());
  at::Tensor x, a;
  if (!amax_in.has_value() && can_round(w, false)) std::tie(x, a) = round_amax(w, nullptr);
  else x = as_bf16_rows(w);
  const int64_t rows = x.size(0), cols = x.size(1);
  if (rows % 16 != 0 || cols % 16 != 0)
    raise(PyExc_AssertionError, "weight dims " + std::to_string(rows) + "x" + std::to_string(cols) + " must be divisible by 16");
  if (amax_in.has_value()) a = *amax_in;
  else if (!a.defined()) a = amax_rows(x, false, nullptr, false, OptTensor());
  const c10::Device dev = device_of({&x, &a});
  Operand r = alloc(dev, rows, cols), c = alloc(dev, cols, rows, false);
  check(lib.nvfp4_quantize_weight_bf16(x.data_ptr(), rows, cols, x.stride(0), two_d, float_ptr(a), r.qp(), r.sp(), c.qp(),
                                       c.sp(), r.pp(), stream_of(dev)),
        "nvfp4_quantize_weight_bf16");
  return py::make_tuple(r.q, r.s, c.q, c.s, r.p);
}

// counters: empty, or pitch and base of the row-wise and of the transposed layout
py::tuple quantize_dual(const at::Tensor& t, const OptTensor& signs, const OptTensor& amax_r, const OptTensor& amax_c,
                        bool sr_rows, bool sr_cols, uint64_t seed_r, uint64_t seed_c, uint64_t offset,
                        const std::vector<uint64_t>& counters) {
  check_matrix(t);
  const c10::cuda::CUDAGuard guard(t.device());
  const int64_t rows = t.size(0), cols = t.size(1);
  if (rows % 16 != 0 || cols % 16 != 0)
    raise(PyExc_AssertionError, "dims " + std::to_string(rows) + "x" + std::to_string(cols) + " must be divisible by 16");
  const at::Tensor sg = signs_on(signs, t.device());
  at::Tensor x, r, c, both;                                  // `both`: the two maxima found here
  if (amax_r.has_value()) r = *amax_r;
  if (amax_c.has_value()) c = *amax_c;
  if (!r.defined() && !c.defined() && can_round(t, true)) std::tie(x, both) = round_amax(t, &sg);
  else x = as_bf16_rows(t);
  if (both.defined()) {}
  else if (!r.defined() && !c.defined()) both = amax_both_rows(x, sg);
  else if (!c.defined()) c = amax_rows(x, true, &sg, true, OptTensor());
  else if (!r.defined()) r = amax_rows(x, false, nullptr, false, OptTensor());
  const c10::Device dev = device_of({&x, &sg, r.defined() ? &r : nullptr, c.defined() ? &c : nullptr});
  const float* rp = both.defined() ? float_ptr(both) : float_ptr(r);
  const float* cp = both.defined() ? float_ptr(both) + 1 : float_ptr(c);
  Operand a = alloc(dev, rows, cols), b = alloc(dev, cols, rows);
  check(lib.nvfp4_quantize_dual_bf16(x.data_ptr(), rows, cols, x.stride(0), sr_rows, sr_cols, float_ptr(sg), rp, cp, seed_r,
                                     seed_c, offset, counters.size() == 4 ? counters.data() : nullptr, a.qp(), a.sp(),
                                     a.pp(), b.qp(), b.sp(), b.pp(), stream_of(dev)),
        "nvfp4_quantize_dual_bf16");
  return py::make_tuple(a.q, a.s, a.p, b.q, b.s, b.p);
}

at::Tensor mm(const at::Tensor& aq, const at::Tensor& as, const at::Tensor& ap, const at::Tensor& bq, const at::Tensor& bs,
              const at::Tensor& bp, bool f32, const OptTensor& out, const OptTensor& amax_out) {
  const int64_t m = aq.size(0), k2 = aq.size(1), n = bq.size(0);
  const c10::Device dev = device_of({&aq, &as, &ap, &bq, &bs, &bp, ptr_of(out), ptr_of(amax_out)});
  const c10::cuda::CUDAGuard guard(dev);
  const at::Tensor d = out.has_value() ? *out : at::empty({m, n}, on(dev, f32 ? at::kFloat : at::kBFloat16));
  auto u8 = [](const at::Tensor& t) { return static_cast<const uint8_t*>(t.data_ptr()); };
  int32_t* status = status_word(dev.index()).data_ptr<int32_t>();
  const int type = f32 ? NVFP4_OUT_F32 : NVFP4_OUT_BF16;
  check(amax_out.has_value()
            ? lib.nvfp4_gemm_amax(u8(aq), u8(as), float_ptr(ap), u8(bq), u8(bs), float_ptr(bp), d.data_ptr(), type, m, n,
                                  k2 * 2, d.stride(0), float_ptr(*amax_out), status, stream_of(dev))
            : lib.nvfp4_gemm(u8(aq), u8(as), float_ptr(ap), u8(bq), u8(bs), float_ptr(bp), d.data_ptr(), type, m, n, k2 * 2,
                             d.stride(0), status, stream_of(dev)),
        "nvfp4_gemm");
  return d;
}

// the bf16 product in an fp32 tensor
at::Tensor mm_bf16_as_f32(const at::Tensor& aq, const at::Tensor& as, const at::Tensor& ap, const at::Tensor& bq,
                          const at::Tensor& bs, const at::Tensor& bp) {
  const int64_t m = aq.size(0), k2 = aq.size(1), n = bq.size(0);
  const c10::Device dev = device_of({&aq, &as, &ap, &bq, &bs, &bp});
  const c10::cuda::CUDAGuard guard(dev);
  const at::Tensor d = at::empty({m, n}, on(dev, at::kFloat));
  auto u8 = [](const at::Tensor& t) { return static_cast<const uint8_t*>(t.data_ptr()); };
  check(lib.nvfp4_gemm_bf16_as_f32(u8(aq), u8(as), float_ptr(ap), u8(bq), u8(bs), float_ptr(bp), float_ptr(d), m, n, k2 * 2,
                                   n, status_word(dev.index()).data_ptr<int32_t>(), stream_of(dev)),
        "nvfp4_gemm_bf16_as_f32");
  return d;
}

// ---- optimizer ------------------------------------------------------------------------------------------------------
const at::Tensor& tensor_of(PyObject* o) {
  if (!THPVariable_Check(o)) raise(PyExc_TypeError, "expected a tensor");
  return THPVariable_Unpack(o);
}
bool same_layout(const at::Tensor& a, const at::Tensor& b) {
  if (a.sizes() != b.sizes()) return false;
  if (a.is_contiguous() && b.is_contiguous()) return true;
  for (int64_t d = 0; d < a.dim(); ++d)
    if (a.size(d) > 1 && a.stride(d) != b.stride(d)) return false;
  return true;
}
// Is `strides` (a tuple) the tensor's, where they matter?
bool has_strides(const at::Tensor& t, PyObject* strides) {
  if (!PyTuple_Check(strides) || PyTuple_GET_SIZE(strides) != t.dim()) return false;
  for (int64_t d = 0; d < t.dim(); ++d) {
    const int64_t s = PyLong_AsLongLong(PyTuple_GET_ITEM(strides, d));
    if (s == -1 && PyErr_Occurred()) throw py::error_already_set();
    if (t.size(d) > 1 && s != t.stride(d)) return false;
  }
  return true;
}
// fp32 and bf16 tensors whose elements fill one piece of memory: the kernels go through it in its own order
void check_param(const at::Tensor& p, c10::optional<c10::Device>& dev) {
  if (!p.is_cuda() || (dev.has_value() && *dev != p.device())) {
    const at::Tensor first = dev.has_value() ? at::empty({0}, on(*dev, at::kFloat)) : p;
    device_of({&first, &p});                                // says what is wrong
  }
  dev = p.device();
  if (p.scalar_type() != at::kFloat && p.scalar_type() != at::kBFloat16)
    raise(PyExc_ValueError, std::string("parameters are fp32 or bf16, got ") + c10::toString(p.scalar_type()));
  if (p.is_neg()) raise(PyExc_ValueError, "a parameter must not be a lazily negated view");
  if (p.is_inference() && !c10::InferenceMode::is_enabled())
    raise(PyExc_ValueError, "a parameter made in inference mode cannot be changed outside it");
  if (p.layout() != at::kStrided || !p.is_non_overlapping_and_dense())
    raise(PyExc_ValueError, "parameters must fill their memory without gaps or overlaps");
}
// the gradient in the memory order of its parameter
at::Tensor grad_like(const at::Tensor& p, const at::Tensor& g) {
  if (g.layout() != at::kStrided) raise(PyExc_ValueError, "sparse gradients are not supported");
  if (g.device() != p.device() || g.scalar_type() != p.scalar_type() || g.sizes() != p.sizes())
    raise(PyExc_ValueError, "a gradient must have its parameter's device, dtype and shape");
  if (same_layout(p, g) && !g.is_neg()) return g;
  return at::empty_strided(p.sizes(), p.strides(), p.options().requires_grad(false)).copy_(g);
}

struct Grads {                                              // by dtype: bf16, fp32
  std::vector<const void*> ptr[2];
  std::vector<int64_t> n[2];
  void add(const at::Tensor& g) {
    const int k = g.scalar_type() == at::kFloat;
    ptr[k].push_back(g.data_ptr());
    n[k].push_back(g.numel());
  }
  // the partial sums of squares of all of them
  at::Tensor parts(c10::Device dev) const {
    int all = 0, some[2] = {0, 0};
    for (int k = 0; k < 2; ++k) {
      some[k] = lib.nvfp4_sumsq_parts((int)n[k].size(), n[k].data());
      if (some[k] < 0) check(some[k], "nvfp4_sumsq_parts");
      all += some[k];
    }
    at::Tensor parts = at::empty({all}, on(dev, at::kDouble));
    double* at_ = static_cast<double*>(parts.data_ptr());
    for (int k = 0; k < 2; ++k) {
      if (n[k].empty()) continue;
      check(lib.nvfp4_sumsq(ptr[k].data(), n[k].data(), (int)n[k].size(), k, at_, stream_of(dev)), "nvfp4_sumsq");
      at_ += some[k];
    }
    return parts;
  }
};

// Norm of the gradients of `params` (tensors that have none are skipped); None if none has one.
py::object grad_norm(const py::list& params) {
  Grads grads;
  std::vector<at::Tensor> held;
  c10::optional<c10::Device> dev;
  for (py::handle h : params) {
    const at::Tensor& p = tensor_of(h.ptr());
    const at::Tensor& g = p.grad();
    if (!g.defined() || g.numel() == 0) continue;
    check_param(p, dev);
    held.push_back(grad_like(p, g));
    grads.add(held.back());
  }
  if (held.empty()) return py::none();
  const c10::cuda::CUDAGuard guard(*dev);
  const at::Tensor parts = grads.parts(*dev);
  at::Tensor norm = at::empty({}, on(*dev, at::kFloat));
  check(lib.nvfp4_norm_of_sumsq(static_cast<const double*>(parts.data_ptr()), (int)parts.numel(), float_ptr(norm),
                                stream_of(*dev)),
        "nvfp4_norm_of_sumsq");
  return py::cast(norm);
}

struct Name {                                               // an interned string: looked up by its address
  PyObject* s;
  explicit Name(const char* n) : s(PyUnicode_InternFromString(n)) {}
};
PyObject* item(PyObject* dict, const Name& key) {
  PyObject* v = PyDict_GetItemWithError(dict, key.s);
  if (v == nullptr) {
    if (!PyErr_Occurred()) PyErr_SetObject(PyExc_KeyError, key.s);
    throw py::error_already_set();
  }
  return v;
}
// The entries of a dict whose keys come in the order they were put in: then no key is hashed (a tensor's hash is a Python call).
struct InOrder {
  PyObject* dict;
  Py_ssize_t pos = 0;
  PyObject* find(PyObject* key) {
    PyObject *k = nullptr, *v = nullptr;
    Py_ssize_t next = pos;
    if (PyDict_Next(dict, &next, &k, &v) && k == key) {
      pos = next;
      return v;
    }
    v = PyDict_GetItemWithError(dict, key);
    if (v == nullptr && PyErr_Occurred()) throw py::error_already_set();
    return v;
  }
};
double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw py::error_already_set();
  return v;
}
void check_state(const at::Tensor& t, c10::Device dev, at::ScalarType type, int64_t n, const char* name) {
  if (t.device() != dev || t.scalar_type() != type || t.numel() != n)
    raise(PyExc_ValueError, std::string("optimizer state '") + name + "' does not fit its parameter");
}

// One step of every parameter that has a gradient.  groups: the optimizer's param_groups; state: its state.  Returns, with
// nothing done, "capture" when the stream is being captured and else "state" when a parameter has no state yet; None when no
// parameter has a gradient; else the norm of all gradients (0-dim) if max_norm is given, or True.
py::object adamw_step(const py::list& groups, const py::dict& state, int bits, c10::optional<double> max_norm, uint64_t seed,
                      const OptTensor& norm_in) {
  struct Hyper {
    double lr, b1, b2, eps, wd;
  };
  struct Item {
    nvfp4_adamw_tensor t;
    int group, f32;
    int64_t step;
    PyObject* state;
    c10::TensorImpl* param;
  };
  std::vector<Hyper> hypers;
  std::vector<Item> items;
  std::vector<at::Tensor> held;                              // gradients that had to be copied live until the launch
  Grads grads;
  c10::optional<c10::Device> dev;
  uint64_t base = 0;
  const bool eight = bits == 8;
  static const Name kBetas("betas"), kLr("lr"), kEps("eps"), kDecay("weight_decay"), kParams("params"), kStep("step"),
      kFirst("exp_avg"), kSecond("exp_avg_sq"), kRoot("exp_avg_root"), kFirstScale("exp_avg_scale"),
      kRootScale("exp_avg_root_scale"), kLayout("layout");
  const auto captured = [&] {
    const c10::cuda::CUDAGuard guard(*dev);
    return c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None;
  };
  const at::NoGradGuard no_grad;
  InOrder states{state.ptr()};
  for (py::handle gh : groups) {
    PyObject* group = gh.ptr();
    if (!PyDict_Check(group)) raise(PyExc_TypeError, "param_groups holds dicts");
    const py::sequence betas = py::reinterpret_borrow<py::sequence>(item(group, kBetas));
    hypers.push_back({number(item(group, kLr)), number(py::object(betas[0]).ptr()), number(py::object(betas[1]).ptr()),
                      number(item(group, kEps)), number(item(group, kDecay))});
    for (py::handle ph : py::reinterpret_borrow<py::list>(item(group, kParams))) {
      const at::Tensor& p = tensor_of(ph.ptr());
      const int64_t n = p.numel(), blocks = (n + 255) / 256;
      const uint64_t at_ = base;
      base += (uint64_t)blocks * 32;                         // whether or not it has a gradient now
      const at::Tensor& g0 = p.grad();
      if (!g0.defined() || n == 0) continue;
      check_param(p, dev);
      at::Tensor g = grad_like(p, g0);
      PyObject* st = states.find(ph.ptr());
      if (st != nullptr && !PyDict_Check(st)) raise(PyExc_TypeError, "optimizer state holds dicts");
      // (an empty dict is what looking up a parameter in the optimizer's state leaves there)
      if (st == nullptr || PyDict_GET_SIZE(st) == 0) return py::str(captured() ? "capture" : "state");
      Item it{};
      it.t.param = p.data_ptr();
      it.t.grad = g.data_ptr();
      it.t.n = n;
      it.t.counter_base = at_;
      it.group = (int)hypers.size() - 1;
      it.f32 = p.scalar_type() == at::kFloat;
      it.step = PyLong_AsLongLong(item(st, kStep)) + 1;
      if (it.step == 0 && PyErr_Occurred()) throw py::error_already_set();
      it.state = st;
      it.param = p.unsafeGetTensorImpl();
      const at::Tensor& m = tensor_of(item(st, kFirst));
      const at::Tensor& v = tensor_of(item(st, eight ? kRoot : kSecond));
      if (eight) {
        const at::Tensor& ms = tensor_of(item(st, kFirstScale));
        const at::Tensor& vs = tensor_of(item(st, kRootScale));
        check_state(m, *dev, at::kFloat8_e4m3fn, blocks * 256, "exp_avg");
        check_state(v, *dev, at::kFloat8_e4m3fn, blocks * 256, "exp_avg_root");
        check_state(ms, *dev, at::kFloat8_e8m0fnu, blocks, "exp_avg_scale");
        check_state(vs, *dev, at::kFloat8_e8m0fnu, blocks, "exp_avg_root_scale");
        if (!m.is_contiguous() || !v.is_contiguous() || !ms.is_contiguous() || !vs.is_contiguous())
          raise(PyExc_ValueError, "optimizer state must be contiguous");
        if (!has_strides(p, item(st, kLayout)))
          raise(PyExc_ValueError, "a parameter's shape or strides changed: its 8-bit moments lie in the order of the old ones");
        it.t.first_scale = ms.data_ptr();
        it.t.second_scale = vs.data_ptr();
      } else {
        check_state(m, *dev, at::kFloat, n, "exp_avg");
        check_state(v, *dev, at::kFloat, n, "exp_avg_sq");
        if (!same_layout(p, m) || !same_layout(p, v))
          raise(PyExc_ValueError, "optimizer state must have its parameter's shape and strides");
      }
      it.t.first = m.data_ptr();
      it.t.second = v.data_ptr();
      grads.add(g);
      if (!g.is_same(g0)) held.push_back(std::move(g));
      items.push_back(it);
    }
  }
  if (items.empty()) return py::none();
  if (captured()) return py::str("capture");
  const c10::cuda::CUDAGuard guard(*dev);
  at::Tensor parts, norm;
  const double* parts_p = nullptr;
  const float* norm_p = nullptr;
  if (max_norm.has_value()) {
    if (norm_in.has_value()) {
      const at::Tensor anchor = at::empty({0}, on(*dev, at::kFloat));
      device_of({&anchor, &*norm_in});
      if (norm_in->scalar_type() != at::kFloat || norm_in->numel() != 1)
        raise(PyExc_ValueError, "grad_norm must be one fp32 element");
      norm = norm_in->resolve_neg();
      norm_p = float_ptr(norm);
    } else {
      parts = grads.parts(*dev);
      parts_p = static_cast<const double*>(parts.data_ptr());
      norm = at::empty({}, on(*dev, at::kFloat));
    }
  }
  // launches: one per dtype and up to eight different (group, step)
  std::vector<nvfp4_adamw_tensor> ts;
  std::vector<nvfp4_adamw_hyper> hs;
  bool norm_out = parts_p != nullptr;
  for (int f32 = 0; f32 < 2; ++f32) {
    size_t i = 0;
    while (i < items.size()) {
      ts.clear();
      hs.clear();
      std::vector<std::pair<int, int64_t>> keys;
      for (; i < items.size(); ++i) {
        Item& it = items[i];
        if (it.f32 != f32) continue;
        const std::pair<int, int64_t> key{it.group, it.step};
        size_t k = 0;
        while (k < keys.size() && keys[k] != key) ++k;
        if (k == keys.size()) {
          if (k == 8) break;
          keys.push_back(key);
          const Hyper& h = hypers[it.group];
          const double t = (double)it.step;
          hs.push_back({(float)(1.0 - h.lr * h.wd), (float)h.b1, (float)(1.0 - h.b1), (float)h.b2, (float)(1.0 - h.b2),
                        (float)(h.lr / (1.0 - std::pow(h.b1, t))), (float)(1.0 / std::sqrt(1.0 - std::pow(h.b2, t))),
                        (float)h.eps, (uint64_t)it.step});
        }
        it.t.hyper = (int32_t)k;
        ts.push_back(it.t);
      }
      if (ts.empty()) break;
      check(lib.nvfp4_adamw(ts.data(), (int)ts.size(), hs.data(), (int)hs.size(), f32, bits, seed, parts_p,
                            parts_p == nullptr ? 0 : (int)parts.numel(), norm_p, max_norm.value_or(0.0),
                            norm_out ? float_ptr(norm) : nullptr, stream_of(*dev)),
            "nvfp4_adamw");
      if (norm_out) {                                        // later launches take the norm that the first one left
        parts_p = nullptr;
        norm_p = float_ptr(norm);
        norm_out = false;
      }
    }
  }
  for (const Item& it : items) {
    const py::int_ step(it.step);
    if (PyDict_SetItem(it.state, kStep.s, step.ptr()) != 0) throw py::error_already_set();
    it.param->bump_version();                                // it changed in place, as any optimizer changes it
  }
  if (norm.defined()) return py::cast(norm);
  return py::bool_(true);
}

// ---- losses on logits -----------------------------------------------------------------------------------------------
// Logits [rows, vocab] or [batch, seq, vocab] and their labels as the kernels read them.
struct Logits {
  at::Tensor x, labels;                                     // x is the caller's tensor wherever the kernels can read that
  nvfp4_logit_rows rows;
  c10::Device dev{c10::kCUDA};
  Logits(const at::Tensor& logits, const at::Tensor& labels_in, int64_t ignore) {
    if (logits.dim() != 2 && logits.dim() != 3) raise(PyExc_ValueError, "logits must be [rows, vocab] or [batch, seq, vocab]");
    if (labels_in.sizes() != logits.sizes().slice(0, logits.dim() - 1))
      raise(PyExc_ValueError, "labels must have the shape of the logits without the last dimension");
    if (logits.scalar_type() != at::kFloat && logits.scalar_type() != at::kBFloat16)
      raise(PyExc_ValueError, std::string("logits are fp32 or bf16, got ") + c10::toString(logits.scalar_type()));
    if (!c10::isIntegralType(labels_in.scalar_type(), false)) raise(PyExc_ValueError, "labels must be integers");
    if (logits.numel() == 0) raise(PyExc_ValueError, "logits are empty");
    dev = device_of({&logits, &labels_in});
    x = logits.resolve_neg();
    if (x.stride(-1) != 1 && x.size(-1) > 1) x = x.contiguous();
    labels = labels_in.to(at::kLong).resolve_neg().contiguous();
    const bool three = x.dim() == 3;
    rows = nvfp4_logit_rows{x.data_ptr(), x.scalar_type() == at::kFloat, three ? x.size(0) : 1, x.size(-2), x.size(-1),
                            three ? x.stride(0) : 0, x.stride(-2), labels.data_ptr<int64_t>(), ignore};
  }
  int64_t count() const { return rows.batch * rows.seq; }
  at::Tensor per_row() const { return at::empty(labels.sizes(), on(dev, at::kFloat)); }
  // A vector of `shape` as the kernels read it.  Sizes of 1 and a flat vector are let through; the same number of values in another
  // shape (transposed, say) would be read in the wrong order.
  at::Tensor vec(const at::Tensor& t, c10::IntArrayRef shape, const char* name, at::ScalarType type = at::kFloat) const {
    device_of({&x, &t});
    const auto without_ones = [](c10::IntArrayRef s) {
      std::vector<int64_t> out;
      for (int64_t n : s)
        if (n != 1) out.push_back(n);
      return out;
    };
    int64_t n = 1;
    for (int64_t s : shape) n *= s;
    if (t.numel() != n || !t.is_floating_point() || (t.dim() != 1 && t.sizes() != shape && without_ones(t.sizes()) != without_ones(shape))) {
      std::string want = "[";
      for (int64_t s : shape) want += (want.size() > 1 ? ", " : "") + std::to_string(s);
      raise(PyExc_ValueError, std::string(name) + " must hold " + std::to_string(n) + " floating-point values, " + want + "]");
    }
    return t.to(type).resolve_neg().contiguous();
  }
};

// Do rows of these strides lie apart?
bool rows_apart(const nvfp4_logit_rows& r, int64_t stride_b, int64_t stride_t) {
  const bool time_inside = stride_t <= stride_b || r.batch == 1;
  const int64_t inner = time_inside ? stride_t : stride_b, outer = time_inside ? stride_b : stride_t;
  const int64_t n_inner = time_inside ? r.seq : r.batch, n_outer = time_inside ? r.batch : r.seq;
  return (n_inner == 1 || inner >= r.vocab) && (n_outer == 1 || outer >= (n_inner - 1) * inner + r.vocab);
}
// A tensor for the gradient of logits whose rows lie as the logits' own do, modulo 16 bytes: then both are read and written in
// whole vectors.  (A view of shifted logits has rows at other places than a contiguous tensor of its shape.)
at::Tensor gradient_like(const at::Tensor& x, const Logits& in) {
  const nvfp4_logit_rows& r = in.rows;
  const bool time_inside = r.stride_t <= r.stride_b || r.batch == 1;
  const int64_t inner = time_inside ? r.stride_t : r.stride_b, outer = time_inside ? r.stride_b : r.stride_t;
  const int64_t n_inner = time_inside ? r.seq : r.batch, n_outer = time_inside ? r.batch : r.seq;
  const int64_t span = (n_outer - 1) * outer + (n_inner - 1) * inner + r.vocab;
  const int64_t shift = (int64_t)(reinterpret_cast<uintptr_t>(r.logits) % 16) / (r.is_f32 ? 4 : 2);
  const auto opt = on(in.dev, x.scalar_type());
  if (!rows_apart(r, r.stride_b, r.stride_t) || !in.x.is_same(x) || span > 2 * x.numel()) return at::empty(x.sizes(), opt);
  if (shift == 0 && x.is_contiguous()) return at::empty(x.sizes(), opt);
  return at::empty({span + shift}, opt).as_strided(x.sizes(), x.strides(), shift);
}
int64_t batch_stride(const at::Tensor& t) { return t.dim() == 3 ? t.stride(0) : 0; }

// Nodes of the autograd graph.  In C++ because of the backward pass, which autograd runs on a thread of its own: a Python
// node has to wait there for the interpreter lock (a loss of 48 logit rows and its gradient: 122 us, 69 from here).
using torch::autograd::AutogradContext;
using torch::autograd::tensor_list;

void check_in_backward(int code, const char* what) {         // without the interpreter
  if (code != 0) throw std::runtime_error(std::string(what) + " failed: " + lib.nvfp4_status_string(code));
}
// A gradient that says so when it is differentiated again: it depends on the logits and on the gradient behind it, and without
// a node of its own a penalty on it would be lost without a word.
struct Once : torch::autograd::Function<Once> {
  static at::Tensor forward(AutogradContext*, const at::Tensor& gradient, const at::Tensor&, const at::Tensor&) { return gradient.detach(); }
  static tensor_list backward(AutogradContext*, tensor_list) { throw std::runtime_error("the losses on logits are differentiable once"); }
};
nvfp4_row_stat* stat_ptr(const at::Tensor& t) { return reinterpret_cast<nvfp4_row_stat*>(float_ptr(t)); }
// Gradient of the logits.  saved: logits, labels and, in one tensor, the rows' statistics and dloss / dlogp (one per row or per
// sequence, `per` rows each), or the former alone and `weight` for the latter.  They come back as a hook on saved tensors or an
// assignment to their .data left them, and are looked at again.  scale: what dloss / dlogp is to be multiplied with (one
// element); ready: the gradient for a scale of 1, used again where the scale is 1
at::Tensor dlogits(const torch::autograd::variable_list& saved, int64_t ignore, int64_t per, const at::Tensor& weight,
                   const at::Tensor& scale, const at::Tensor& ready) {
  const Logits in(saved[0], saved[1], ignore);
  const c10::cuda::CUDAGuard guard(in.dev);
  const int64_t n = in.count();
  const at::Tensor& kept = saved[2];
  if (kept.device() != in.dev || kept.scalar_type() != at::kFloat || !kept.is_contiguous() || kept.is_neg() || n % per != 0 ||
      kept.numel() != 2 * n + (weight.defined() ? 0 : n / per) || reinterpret_cast<uintptr_t>(kept.data_ptr()) % 8 != 0 ||
      (ready.defined() && (ready.sizes() != in.x.sizes() || ready.scalar_type() != in.x.scalar_type() || ready.device() != in.dev)))
    throw std::runtime_error("what a loss saved for its backward pass came back changed");
  const at::Tensor w = weight.defined() ? weight.to(at::kFloat).resolve_neg().contiguous() : kept,
                   sc = scale.defined() ? scale.to(at::kFloat).resolve_neg() : scale;
  const float* wp = float_ptr(w) + (weight.defined() ? 0 : 2 * n);
  at::Tensor out = ready.defined() ? ready.resolve_neg() : gradient_like(saved[0], in);
  if (ready.defined() && ((out.size(-1) > 1 && out.stride(-1) != 1) || !rows_apart(in.rows, batch_stride(out), out.stride(-2))))
    out = out.contiguous();                                  // (a hook laid it out anew)
  check_in_backward(lib.nvfp4_logprob_bwd(&in.rows, stat_ptr(kept), wp, per, sc.defined() ? float_ptr(sc) : nullptr,
                                          ready.defined(), out.data_ptr(), batch_stride(out), out.stride(-2), stream_of(in.dev)),
                    "nvfp4_logprob_bwd");
  return c10::GradMode::is_enabled() ? Once::apply(out, saved[0], weight.defined() ? weight : scale) : out;
}

struct TokenLogprobs : torch::autograd::Function<TokenLogprobs> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& labels, int64_t ignore) {
    const Logits in(logits, labels, ignore);
    const c10::cuda::CUDAGuard guard(in.dev);
    at::Tensor logp = in.per_row(), kept = at::empty({2 * in.count()}, on(in.dev, at::kFloat));
    check(lib.nvfp4_logprob_fwd(&in.rows, float_ptr(logp), stat_ptr(kept), stream_of(in.dev)), "nvfp4_logprob_fwd");
    ctx->save_for_backward({logits, labels, kept});
    ctx->saved_data["ignore"] = ignore;
    return logp;
  }
  static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
    return {dlogits(ctx->get_saved_variables(), ctx->saved_data["ignore"].toInt(), 1, grads[0], {}, {}), {}, {}};
  }
};

// scratch of a loss: the workspace and `more` bytes behind it
at::Tensor loss_scratch(c10::Device dev, int64_t more) { return at::empty({NVFP4_LOSS_WORKSPACE + more}, on(dev, at::kByte)); }

// -> loss, rewards
struct Preference : torch::autograd::Function<Preference> {
  static tensor_list forward(AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& labels, const at::Tensor& ref,
                             double beta, double smoothing, int64_t ignore) {
    const Logits in(logits, labels, ignore);
    if (logits.dim() != 3 || in.rows.batch % 2 != 0)
      raise(PyExc_ValueError, "logits must be [2 pairs, seq, vocab], the chosen sequences first");
    const bool halves = ref.dim() == 2 && ref.size(0) == 2;                        // [2, pairs]: they lie in the same order
    const at::Tensor r = in.vec(halves ? ref.reshape({-1}) : ref, {in.rows.batch}, "ref_logps",
                                    ref.scalar_type() == at::kDouble ? at::kDouble : at::kFloat);
    const c10::cuda::CUDAGuard guard(in.dev);
    const int64_t n = in.count();
    at::Tensor loss = at::empty({}, on(in.dev, at::kFloat)), rewards = at::empty({in.rows.batch}, on(in.dev, at::kFloat)),
               kept = at::empty({2 * n + in.rows.batch}, on(in.dev, at::kFloat));
    const at::Tensor scratch = loss_scratch(in.dev, 8 * n);
    uint8_t* ws = scratch.data_ptr<uint8_t>();
    double* logp = reinterpret_cast<double*>(ws + NVFP4_LOSS_WORKSPACE);
    const auto call = [&](auto entry, const auto* reference) {
      check(entry(&in.rows, reference, beta, smoothing, logp, stat_ptr(kept), float_ptr(loss), float_ptr(rewards), float_ptr(kept) + 2 * n, ws,
                  NVFP4_LOSS_WORKSPACE, stream_of(in.dev)),
            "nvfp4_preference_fwd");
    };
    if (r.scalar_type() == at::kDouble) call(lib.nvfp4_preference_fwd_ref64, r.const_data_ptr<double>());
    else call(lib.nvfp4_preference_fwd, r.const_data_ptr<float>());
    ctx->save_for_backward({logits, labels, kept});
    ctx->saved_data["ignore"] = ignore;
    ctx->saved_data["seq"] = in.rows.seq;
    ctx->mark_non_differentiable({rewards});
    ctx->set_materialize_grads(false);
    return {loss, rewards};
  }
  static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
    if (!grads[0].defined()) return tensor_list(6);          // the node behind this one gave no gradient
    return {dlogits(ctx->get_saved_variables(), ctx->saved_data["ignore"].toInt(), ctx->saved_data["seq"].toInt(), {}, grads[0], {}),
            {}, {}, {}, {}, {}};
  }
};

// A tensor that waits for the backward pass by itself: hooks on saved tensors see it like any other, and it is let go when it is
// taken, whether or not the rest of the graph is kept.
struct Waiting : torch::CustomClassHolder {
  torch::autograd::SavedVariable tensor;
  explicit Waiting(const at::Tensor& t) : tensor(t, false) {}
};

// -> loss, stats, log-probabilities.  The forward kernel writes the gradient for dloss = 1 while it has the rows at hand;
// the backward writes it again only where the loss arrives with another factor.
struct PolicyLoss : torch::autograd::Function<PolicyLoss> {
  static tensor_list forward(AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& labels, const at::Tensor& old_logps,
                             const at::Tensor& advantages, const OptTensor& ref, double low, double high, double kl,
                             int64_t ignore, bool want_grad) {
    const Logits in(logits, labels, ignore);
    const int64_t n = in.count();
    const bool per_sequence = advantages.dim() == 1 && logits.dim() == 3;
    const at::Tensor old = in.vec(old_logps, labels.sizes(), "old_logps"),
                     adv = in.vec(advantages, per_sequence ? c10::IntArrayRef(in.rows.batch) : labels.sizes(), "advantages");
    at::Tensor rf, grad;
    if (ref.has_value()) rf = in.vec(*ref, labels.sizes(), "ref_logps");
    const c10::cuda::CUDAGuard guard(in.dev);
    at::Tensor logp = in.per_row(), kept = at::empty({3 * n}, on(in.dev, at::kFloat)), loss = at::empty({}, on(in.dev, at::kFloat)),
               stats = at::empty({2}, on(in.dev, at::kFloat));
    if (want_grad) grad = gradient_like(logits, in);
    const at::Tensor scratch = loss_scratch(in.dev, 8 * n);
    uint8_t* ws = scratch.data_ptr<uint8_t>();
    check(lib.nvfp4_policy_fwd(&in.rows, float_ptr(old), float_ptr(adv), n / adv.numel(), rf.defined() ? float_ptr(rf) : nullptr,
                               low, high, kl, float_ptr(logp), stat_ptr(kept), float_ptr(kept) + 2 * n,
                               reinterpret_cast<float*>(ws + NVFP4_LOSS_WORKSPACE), float_ptr(loss), float_ptr(stats),
                               want_grad ? grad.data_ptr() : nullptr, want_grad ? batch_stride(grad) : 0,
                               want_grad ? grad.stride(-2) : 0, ws, NVFP4_LOSS_WORKSPACE, stream_of(in.dev)),
          "nvfp4_policy_fwd");
    ctx->save_for_backward({logits, labels, kept});
    ctx->saved_data["ignore"] = ignore;
    if (want_grad) ctx->saved_data["grad"] = at::IValue::make_capsule(c10::make_intrusive<Waiting>(grad));
    ctx->mark_non_differentiable({stats, logp});
    ctx->set_materialize_grads(false);
    return {loss, stats, logp};
  }
  static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
    if (!grads[0].defined()) return tensor_list(10);
    at::Tensor ready;
    if (auto it = ctx->saved_data.find("grad"); it != ctx->saved_data.end()) {      // (a second backward writes its own)
      const auto waiting = it->second.toCapsule();
      ctx->saved_data.erase(it);
      ready = static_cast<Waiting*>(waiting.get())->tensor.unpack();
    }
    return {dlogits(ctx->get_saved_variables(), ctx->saved_data["ignore"].toInt(), 1, {}, grads[0], ready), {}, {}, {}, {}, {}, {}, {}, {}, {}};
  }
};

at::Tensor token_logprobs(const at::Tensor& logits, const at::Tensor& labels, int64_t ignore) {
  return TokenLogprobs::apply(logits, labels, ignore);
}
py::tuple preference_loss(const at::Tensor& logits, const at::Tensor& labels, const at::Tensor& ref, double beta, double smoothing,
                          int64_t ignore) {
  const tensor_list out = Preference::apply(logits, labels, ref, beta, smoothing, ignore);
  const int64_t pairs = out[1].numel() / 2;
  return py::make_tuple(out[0], out[1].narrow(0, 0, pairs), out[1].narrow(0, pairs, pairs));
}
py::tuple policy_loss(const at::Tensor& logits, const at::Tensor& labels, const at::Tensor& old_logps, const at::Tensor& advantages,
                      const OptTensor& ref, double low, double high, double kl, int64_t ignore) {
  const bool want_grad = c10::GradMode::is_enabled() && logits.requires_grad();
  const tensor_list out = PolicyLoss::apply(logits, labels, old_logps, advantages, ref, low, high, kl, ignore, want_grad);
  return py::make_tuple(out[0], out[2], out[1].select(0, 0), out[1].select(0, 1));
}

}  // namespace

PYBIND11_MODULE(_host, m) {
  m.def("init", &init);
  m.def("workspace", &workspace);
  m.def("workspace_if_any", &workspace_if_any);
  m.def("status_word", &status_word);
  m.def("amax", &amax);
  m.def("amax_both", &amax_both);
  m.def("quantize", &quantize);
  m.def("quantize_weight", &quantize_weight);
  m.def("quantize_dual", &quantize_dual);
  m.def("mm", &mm);
  m.def("mm_bf16_as_f32", &mm_bf16_as_f32);
  m.def("grad_norm", &grad_norm);
  m.def("adamw_step", &adamw_step);
  m.def("token_logprobs", &token_logprobs);
  m.def("preference_loss", &preference_loss);
  m.def("policy_loss", &policy_loss);
}
