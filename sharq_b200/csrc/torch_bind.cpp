// Native form of the per-call host work of the operators in ops.py: argument checks, output allocation and the C-ABI
// calls, without a Python view, attribute access or ctypes conversion per buffer.  A decode step issues one prepare and
// one GEMM per linear, a few microseconds of GPU work each; as Python this host work took 30 to 40 us per linear, several
// times the kernels it launched (see ops.py for the operators and their meaning; the checks and messages are those).
//
// Tensors are borrowed; outputs come from the torch caching allocator on the current stream of the input's device.
#include <torch/csrc/utils/pybind.h>

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContextLight.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <optional>
#include <stdexcept>
#include <string>
#include <utility>
#include <vector>

#include "../../include/sharq_b200.h"

namespace py = pybind11;

namespace {

using at::Tensor;

[[noreturn]] void fail(const std::string &msg) { throw std::runtime_error(msg); }

inline void need(bool ok, const char *msg) {
  if (!ok) fail(msg);
}

// A non-zero status of an entry point; becomes sharq_b200._lib.SharqError.
struct LibraryError : std::runtime_error {
  using std::runtime_error::runtime_error;
};

inline void check(int status) {
  if (status != 0) throw LibraryError(sharq_last_error());
}

inline void *ptr(const Tensor &t) { return t.data_ptr(); }
inline void *stream_of(const Tensor &t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

inline Tensor empty_like_on(const Tensor &ref, at::IntArrayRef sizes, at::ScalarType type) {
  return at::empty(sizes, ref.options().dtype(type).layout(at::kStrided).requires_grad(false));
}

// ... made without the dispatcher, which takes a microsecond of the six that a small call takes on the host.  The device must be the current one.
inline Tensor fresh(at::IntArrayRef sizes, at::ScalarType type) {
  int64_t n = 1;
  for (const int64_t s : sizes) n *= s;
  const size_t bytes = (size_t)n * c10::elementSize(type);
  c10::Allocator *from = c10::cuda::CUDACachingAllocator::get();
  Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(c10::Storage::use_byte_size_t(), bytes, from->allocate(bytes), from, true),
                                                      c10::DispatchKeySet(c10::DispatchKey::CUDA), c10::scalarTypeToTypeMeta(type));
  t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
  return t;
}

inline bool is_plain(const Tensor &t, at::ScalarType type) { return t.is_cuda() && t.scalar_type() == type && t.is_contiguous(); }

inline int64_t round256(int64_t n) { return (n + 255) & ~int64_t(255); }
inline int64_t sf_bytes(int64_t rows, int64_t k) { return (rows / 128 + 1) * 128 * k / 16; }

void check_x(const Tensor &x) {
  need(x.is_cuda(), "X must be a CUDA tensor");
  need(x.is_contiguous(), "X must be contiguous");
  need(x.scalar_type() == at::kBFloat16, "X must be torch.bfloat16");
  need(x.dim() == 2, "X must be shaped [M, K]");
}

void check_k128(const char *op, const char *verb, int64_t k) {
  if (k % 128 != 0) fail(std::string(op) + " " + verb + " K to be a multiple of 128, got " + std::to_string(k));
}

// The five prepare outputs and `extra` trailing bytes in one allocation, at 256-byte aligned offsets.
struct Prepared {
  Tensor buf;
  int64_t m, k, sa, se, ssf, sq, o_e, o_sfa, o_q, o_sf, o_tail;
  uint8_t *base;

  Prepared(const Tensor &ref, int64_t m_, int64_t k_, int64_t extra) : m(m_), k(k_) {
    const int64_t k256 = (k + 255) / 256 * 256;
    sa = m * k256 / 4;
    se = ((m + 127) / 128 * 128) * k256 / 16;
    ssf = sf_bytes(m, k);
    sq = m * (k / 2);
    o_e = round256(sa);
    o_sfa = o_e + round256(se);
    o_q = o_sfa + round256(ssf);
    o_sf = o_q + round256(sq);
    o_tail = o_sf + round256(ssf);
    buf = empty_like_on(ref, {o_tail + extra}, at::kByte);
    base = static_cast<uint8_t *>(buf.data_ptr());
  }
  uint8_t *a_comp() const { return base; }
  uint8_t *e() const { return base + o_e; }
  uint8_t *sfa() const { return base + o_sfa; }
  uint8_t *q_res() const { return base + o_q; }
  uint8_t *sf_res() const { return base + o_sf; }
  uint8_t *tail() const { return base + o_tail; }
  // A contiguous tensor in the allocation, `offset` bytes into it, made without the dispatcher: with as_strided and view the six to eight
  // outputs of a prepare were 5 of its 12 us on the host.
  Tensor part(int64_t offset, at::IntArrayRef sizes, at::ScalarType type) const {
    Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(buf.storage()), buf.key_set(), c10::scalarTypeToTypeMeta(type));
    c10::TensorImpl *impl = t.unsafeGetTensorImpl();
    impl->set_storage_offset(offset / (int64_t)c10::elementSize(type));
    impl->set_sizes_contiguous(sizes);
    return t;
  }
  Tensor view(int64_t offset, int64_t n) const { return part(offset, {n}, at::kByte); }
  // a 0-dim float32 view at `offset` bytes behind the tail
  Tensor scalar(int64_t offset) const { return part(o_tail + offset, {}, at::kFloat); }
  std::vector<Tensor> outputs() const {
    return {view(0, sa), view(o_e, se), view(o_sfa, ssf), part(o_q, {m, k / 2}, at::kByte), view(o_sf, ssf)};
  }
};

// Scaled (RMSNorm-fused when gamma is given) prepare; workspace and scale live in the tail of the outputs.
struct Scaled {
  Prepared p;
  int64_t ws_bytes, scale_at;
  Tensor total;

  Scaled(const Tensor &x, const std::optional<Tensor> &gamma, double eps, int64_t n, const std::optional<Tensor> &residual)
      : p(x, x.size(0), x.size(1), round256((int64_t)sharq_prepare_workspace_best_bytes((int)x.size(0))) + 256) {
    ws_bytes = (int64_t)sharq_prepare_workspace_best_bytes((int)p.m);
    scale_at = round256(ws_bytes);
    const int m = (int)p.m, k = (int)p.k;
    c10::cuda::OptionalCUDAGuard guard(x.device());
    float *scale = reinterpret_cast<float *>(p.tail() + scale_at);
    if (residual) {
      total = at::empty_like(x);
      check(sharq_fused_add_rmsnorm_sparse_residual_quantize_x(ptr(x), ptr(*residual), ptr(total), ptr(*gamma), (float)eps, m,
                                                               (int)n, k, p.tail(), (size_t)ws_bytes, p.a_comp(), p.e(), p.sfa(),
                                                               p.q_res(), p.sf_res(), scale, stream_of(x)));
    } else if (gamma) {
      check(sharq_fused_rmsnorm_sparse_residual_quantize_x(ptr(x), ptr(*gamma), (float)eps, m, (int)n, k, p.tail(),
                                                           (size_t)ws_bytes, p.a_comp(), p.e(), p.sfa(), p.q_res(), p.sf_res(),
                                                           scale, stream_of(x)));
    } else {
      check(sharq_scaled_sparse_residual_quantize_x(ptr(x), m, (int)n, k, p.tail(), (size_t)ws_bytes, p.a_comp(), p.e(),
                                                    p.sfa(), p.q_res(), p.sf_res(), scale, stream_of(x)));
    }
  }
};

std::vector<Tensor> scaled_prepare(const Tensor &x, const std::optional<Tensor> &gamma, double eps, int64_t n,
                         const std::optional<Tensor> &residual, bool return_workspace) {
  check_x(x);
  const int64_t k = x.size(1);
  const char *op = residual ? "fused_add_rmsnorm_sparse_residual_quantize_x"
                            : (gamma ? "fused_rmsnorm_sparse_residual_quantize_x" : "scaled_sparse_residual_quantize_x");
  if (residual)
    need(is_plain(*residual, at::kBFloat16) && residual->sizes() == x.sizes() && residual->device() == x.device(),
         "residual must be a contiguous CUDA bfloat16 tensor shaped like X on the same device");
  if (gamma) {
    const Tensor &w = *gamma;
    if (residual) {
      need(is_plain(w, at::kBFloat16) && w.dim() == 1 && w.size(0) == k && w.device() == x.device(),
           "rmsnorm_weight must be a contiguous CUDA bfloat16 tensor shaped [K] on X's device");
    } else {
      need(w.is_cuda(), "rmsnorm_weight must be a CUDA tensor");
      need(w.is_contiguous(), "rmsnorm_weight must be contiguous");
      need(w.scalar_type() == at::kBFloat16, "rmsnorm_weight must be torch.bfloat16");
      need(w.dim() == 1, "rmsnorm_weight must be shaped [K]");
      need(w.device() == x.device(), "rmsnorm_weight must be on the same device as X");
      if (w.size(0) != k)
        fail("rmsnorm_weight size mismatch: expected " + std::to_string(k) + ", got " + std::to_string(w.size(0)));
    }
  }
  check_k128(op, gamma && !residual ? "currently requires" : "requires", k);
  if (gamma && k / 32 > 1024) fail(std::string(op) + " requires K/32 <= 1024, got " + std::to_string(k / 32));
  Scaled s(x, gamma, eps, n, residual);
  std::vector<Tensor> out = s.p.outputs();
  out.push_back(s.p.scalar(s.scale_at));
  if (residual)
    out.push_back(s.total);
  else if (return_workspace)
    out.push_back(s.p.view(s.p.o_tail, 256 + 4 * s.p.m));
  return out;
}

std::vector<Tensor> swiglu_prepare(const Tensor &gate_up, int64_t n) {
  need(is_plain(gate_up, at::kBFloat16) && gate_up.dim() == 2, "gate_up must be a contiguous CUDA bfloat16 matrix");
  const int64_t m = gate_up.size(0), f2 = gate_up.size(1), k = f2 / 2;
  if (f2 % 2 != 0 || k % 128 != 0)
    fail("swiglu_sparse_residual_quantize_x requires K to be a multiple of 128, got " + std::to_string(k));
  const int64_t h_bytes = m * k * 2;
  constexpr int64_t kWs = 256 + 8192;  // with a word for the maximum of every CTA of the SwiGLU kernel
  Prepared p(gate_up, m, k, kWs + 256 + h_bytes);
  c10::cuda::OptionalCUDAGuard guard(gate_up.device());
  check(sharq_swiglu_sparse_residual_quantize_x(ptr(gate_up), (int)m, (int)n, (int)k, p.tail() + kWs + 256, p.tail(), (size_t)kWs, p.a_comp(),
                                                p.e(), p.sfa(), p.q_res(), p.sf_res(),
                                                reinterpret_cast<float *>(p.tail() + kWs), stream_of(gate_up)));
  std::vector<Tensor> out = p.outputs();
  out.push_back(p.scalar(kWs));
  return out;
}

void check_u8(const Tensor &t, const at::Device &dev, int64_t want, const char *name) {
  if (!(t.is_cuda() && t.device() == dev && t.scalar_type() == at::kByte && t.is_contiguous()))
    fail(std::string(name) + " must be a contiguous CUDA uint8 tensor on the device of Q_res");
  if (t.numel() != want)
    fail(std::string(name) + ".numel() mismatch: expected " + std::to_string(want) + ", got " + std::to_string(t.numel()));
}

const float *scale_ptr(const Tensor &scale, const at::Device &dev, const char *name) {
  const std::string n(name);
  if (!scale.is_cuda()) fail(n + " must be a CUDA tensor");
  if (!scale.is_contiguous()) fail(n + " must be contiguous");
  if (scale.scalar_type() != at::kFloat) fail(n + " must be torch.float32");
  if (scale.numel() != 1) fail(n + " must contain exactly one element");
  if (scale.device() != dev) fail(n + " must be on the same device as the inputs");
  return static_cast<const float *>(scale.data_ptr());
}

Tensor output(const Tensor &ref, int64_t m, int64_t n, const std::optional<Tensor> &out) {
  if (!out) return empty_like_on(ref, {m, n}, at::kBFloat16);
  need(out->is_cuda() && out->device() == ref.device() && out->scalar_type() == at::kBFloat16 && out->is_contiguous() &&
           out->dim() == 2 && out->size(0) == m && out->size(1) == n,
       "out must be a contiguous CUDA bfloat16 tensor shaped [M, N]");
  return *out;
}

void check_bias(const std::optional<Tensor> &bias, int64_t n, const at::Device &dev) {
  if (!bias) return;
  need(is_plain(*bias, at::kBFloat16) && bias->numel() == n, "bias must be a contiguous CUDA bfloat16 tensor with N elements");
  need(bias->device() == dev, "bias must be on the same device as the inputs");
}

void check_weight(const Tensor &qw, const Tensor &sfs, const Tensor &sfd, const at::Device &dev, int64_t n, int64_t k) {
  check_u8(qw, dev, n * (k / 2), "QW");
  check_u8(sfs, dev, sf_bytes(n, k), "SFW_sparse");
  check_u8(sfd, dev, sf_bytes(n, k), "SFW_dense");
}

// flag: the device's error flag; with split_k it also stands for the GEMM's (unwritten) workspace.
Tensor linear_gemm(const Tensor &a_comp, const Tensor &e, const Tensor &sfa, const Tensor &q_res, const Tensor &sf_res,
                   const Tensor &qw, const Tensor &sfs, const Tensor &sfd, const std::optional<Tensor> &alpha_t, double alpha,
                   const std::optional<Tensor> &bias, const std::optional<Tensor> &out, const std::optional<Tensor> &residual,
                   const Tensor &flag, bool split_k) {
  const int64_t m = q_res.size(0), k = q_res.size(1) * 2, n = qw.size(0);
  const at::Device dev = q_res.device();
  const int64_t k256 = (k + 255) / 256 * 256;
  check_u8(a_comp, dev, m * k256 / 4, "A_comp");
  check_u8(e, dev, ((m + 127) / 128 * 128) * k256 / 16, "E");
  check_u8(sfa, dev, sf_bytes(m, k), "SFA_sparse");
  check_u8(q_res, dev, m * (k / 2), "Q_res");
  check_u8(sf_res, dev, sf_bytes(m, k), "SF_res");
  check_weight(qw, sfs, sfd, dev, n, k);
  check_bias(bias, n, dev);
  if (residual)
    need(is_plain(*residual, at::kBFloat16) && residual->device() == dev && residual->numel() == m * n,
         "residual must be a contiguous CUDA bfloat16 tensor with M * N elements on the device of Q_res");
  Tensor d = output(q_res, m, n, out);
  const float *alpha_dev = alpha_t ? scale_ptr(*alpha_t, dev, "alpha") : nullptr;
  c10::cuda::OptionalCUDAGuard guard(dev);
  check(sharq_linear_gemm_residual(ptr(a_comp), ptr(e), ptr(sfa), ptr(q_res), ptr(sf_res), ptr(qw), ptr(sfs), ptr(sfd), (int)m,
                                   (int)n, (int)k, (float)alpha, alpha_dev, bias ? ptr(*bias) : nullptr,
                                   residual ? ptr(*residual) : nullptr, ptr(d), split_k ? ptr(flag) : nullptr, split_k ? 16 : 0,
                                   static_cast<int *>(ptr(flag)), stream_of(q_res)));
  return d;
}

// Prepare and fused GEMM of a whole linear in one call.
Tensor linear_forward(const Tensor &x, const Tensor &qw, const Tensor &sfs, const Tensor &sfd, double weight_scale,
                      const std::optional<Tensor> &bias, const Tensor &flag, bool split_k) {
  check_x(x);
  const int64_t m = x.size(0), k = x.size(1), n = qw.size(0);
  check_k128("scaled_sparse_residual_quantize_x", "requires", k);
  check_weight(qw, sfs, sfd, x.device(), n, k);
  check_bias(bias, n, x.device());
  Scaled s(x, std::nullopt, 0.0, n, std::nullopt);
  Tensor d = empty_like_on(x, {m, n}, at::kBFloat16);
  c10::cuda::OptionalCUDAGuard guard(x.device());
  check(sharq_linear_gemm_ws(s.p.a_comp(), s.p.e(), s.p.sfa(), s.p.q_res(), s.p.sf_res(), ptr(qw), ptr(sfs), ptr(sfd), (int)m,
                             (int)n, (int)k, (float)weight_scale, reinterpret_cast<float *>(s.p.tail() + s.scale_at),
                             bias ? ptr(*bias) : nullptr, ptr(d), split_k ? ptr(flag) : nullptr, split_k ? 16 : 0,
                             static_cast<int *>(ptr(flag)), stream_of(x)));
  return d;
}

Tensor dense_gemm(const Tensor &a, const Tensor &b, const Tensor &sfa, const Tensor &sfb, double alpha,
                  const std::optional<Tensor> &alpha_t, const std::optional<Tensor> &c_in, double beta,
                  const std::optional<Tensor> &bias, const std::optional<Tensor> &out, const Tensor &flag, bool split_k) {
  need(a.is_cuda() && b.is_cuda() && sfa.is_cuda() && sfb.is_cuda(), "A, B, SFA and SFB must be CUDA tensors");
  const int64_t m = a.size(0), n = b.size(0), k = a.size(1) * 2;
  const at::Device dev = a.device();
  check_bias(bias, n, dev);
  Tensor d = output(a, m, n, out);
  const float *alpha_dev = alpha_t ? scale_ptr(*alpha_t, dev, "scale") : nullptr;
  c10::cuda::OptionalCUDAGuard guard(dev);
  check(sharq_matmul_bias_ws(ptr(a), ptr(b), ptr(sfa), ptr(sfb), (int)m, (int)n, (int)k, (float)alpha, alpha_dev,
                             c_in ? ptr(*c_in) : nullptr, (float)beta, bias ? ptr(*bias) : nullptr, ptr(d),
                             split_k ? ptr(flag) : nullptr, split_k ? 16 : 0, static_cast<int *>(ptr(flag)), stream_of(a)));
  return d;
}

Tensor sparse_gemm(const std::string &name, const Tensor &a_comp, const Tensor &b, const Tensor &e, const Tensor &sfa,
                   const Tensor &sfb, int64_t m, int64_t n, int64_t k, double alpha, const std::optional<Tensor> &alpha_t,
                   double beta, const Tensor &flag, bool split_k) {
  need(m > 0 && n > 0 && k > 0, "M, N, K must be positive");
  if (beta != 0.0) fail(name + " currently requires beta == 0");
  const Tensor *ts[5] = {&a_comp, &b, &e, &sfa, &sfb};
  const char *names[5] = {"A_comp", "B", "E", "SFA", "SFB"};
  for (const Tensor *t : ts)
    if (!t->is_cuda()) fail(name + " inputs must be CUDA tensors");
  for (const Tensor *t : ts)
    if (!t->is_contiguous()) fail(name + " inputs must be contiguous");
  for (int i = 0; i < 5; ++i)
    if (ts[i]->scalar_type() != at::kByte) fail(std::string(names[i]) + " must be torch.uint8");
  for (const Tensor *t : ts)
    if (t->device() != a_comp.device()) fail(name + " inputs must be on the same device");
  int64_t want[4];
  check(sharq_get_sparse_nvfp4_buffer_sizes((int)m, (int)n, (int)k, want));
  const Tensor *sized[4] = {&a_comp, &e, &sfa, &sfb};
  const char *sized_names[4] = {"A_comp", "E", "SFA", "SFB"};
  for (int i = 0; i < 4; ++i)
    if (sized[i]->numel() != want[i])
      fail(std::string(sized_names[i]) + ".numel() mismatch: expected " + std::to_string(want[i]) + ", got " +
           std::to_string(sized[i]->numel()));
  need(b.dim() == 2, "B must be a 2D tensor shaped [N, K/2]");
  if (b.size(0) != n) fail("B.size(0) mismatch: expected " + std::to_string(n) + ", got " + std::to_string(b.size(0)));
  if (b.size(1) != k / 2) fail("B.size(1) mismatch: expected " + std::to_string(k / 2) + ", got " + std::to_string(b.size(1)));
  Tensor d = empty_like_on(a_comp, {m, n}, at::kBFloat16);
  const float *alpha_dev = alpha_t ? scale_ptr(*alpha_t, a_comp.device(), "alpha") : nullptr;
  c10::cuda::OptionalCUDAGuard guard(a_comp.device());
  check(sharq_sparse_matmul_ws(ptr(a_comp), ptr(b), ptr(e), ptr(sfa), ptr(sfb), (int)m, (int)n, (int)k, (float)alpha, alpha_dev,
                               (float)beta, ptr(d), split_k ? ptr(flag) : nullptr, split_k ? 16 : 0,
                               static_cast<int *>(ptr(flag)), stream_of(a_comp)));
  return d;
}

// x: a 16-byte aligned contiguous CUDA bf16 matrix (ops._scaled_quantize_input)
std::vector<Tensor> scaled_quantize(const Tensor &x, bool shared) {
  const int64_t rows = x.size(0), k = x.size(1);
  const size_t ws_bytes = sharq_scaled_quantize_workspace_bytes();
  Tensor q = empty_like_on(x, {rows, k / 2}, at::kByte), sf = empty_like_on(x, {sf_bytes(rows, k)}, at::kByte);
  Tensor ws = empty_like_on(x, {(int64_t)ws_bytes}, at::kByte), scale = empty_like_on(x, {}, at::kFloat);
  c10::cuda::OptionalCUDAGuard guard(x.device());
  if (!shared) {
    check(sharq_scaled_quantize_nvfp4(ptr(x), (int)rows, (int)k, ptr(ws), ws_bytes, ptr(q), ptr(sf),
                                      static_cast<float *>(ptr(scale)), stream_of(x)));
    return {q, sf, scale};
  }
  Tensor sf2 = empty_like_on(x, {sf_bytes(rows, k)}, at::kByte);
  check(sharq_scaled_quantize_w32_shared(ptr(x), (int)rows, (int)k, ptr(ws), ws_bytes, ptr(q), ptr(sf), ptr(sf2),
                                         static_cast<float *>(ptr(scale)), stream_of(x)));
  return {q, sf, sf2, scale};
}

// Fused GEMM of a merged gate_up weight with SwiGLU in its epilogue -> (h, bits of max|h|)
std::vector<Tensor> linear_gemm_swiglu(const Tensor &a_comp, const Tensor &e, const Tensor &sfa, const Tensor &q_res,
                                       const Tensor &sf_res, const Tensor &qw, const Tensor &sfs, const Tensor &sfd,
                                       const Tensor &alpha_t, double alpha, const Tensor &flag) {
  const int64_t m = q_res.size(0), k = q_res.size(1) * 2, n = qw.size(0);
  const at::Device dev = q_res.device();
  if (n % 256 != 0) fail("the merged gate_up weight must have a multiple of 256 rows, got " + std::to_string(n));
  const int64_t k256 = (k + 255) / 256 * 256;
  check_u8(a_comp, dev, m * k256 / 4, "A_comp");
  check_u8(e, dev, ((m + 127) / 128 * 128) * k256 / 16, "E");
  check_u8(sfa, dev, sf_bytes(m, k), "SFA_sparse");
  check_u8(q_res, dev, m * (k / 2), "Q_res");
  check_u8(sf_res, dev, sf_bytes(m, k), "SF_res");
  check_weight(qw, sfs, sfd, dev, n, k);
  c10::cuda::OptionalCUDAGuard guard(dev);
  Tensor h = empty_like_on(q_res, {m, n / 2}, at::kBFloat16);
  Tensor amax = empty_like_on(q_res, {sharq_gemm_swiglu_absmax_words((int)m, (int)(n / 2))}, at::kInt);
  check(sharq_linear_gemm_swiglu(ptr(a_comp), ptr(e), ptr(sfa), ptr(q_res), ptr(sf_res), ptr(qw), ptr(sfs), ptr(sfd), (int)m,
                                 (int)(n / 2), (int)k, (float)alpha, scale_ptr(alpha_t, dev, "alpha"), ptr(h), ptr(amax),
                                 static_cast<int *>(ptr(flag)), stream_of(q_res)));
  return {h, amax};
}

std::vector<Tensor> absmax_prepare(const Tensor &x, int64_t n, const Tensor &amax_bits) {
  check_x(x);
  check_k128("absmax_sparse_residual_quantize_x", "requires", x.size(1));
  need(amax_bits.is_cuda() && amax_bits.device() == x.device() && amax_bits.scalar_type() == at::kInt && amax_bits.is_contiguous() &&
           amax_bits.numel() >= 1,
       "amax_bits must be a contiguous CUDA int32 vector on X's device");
  Prepared p(x, x.size(0), x.size(1), 256);
  c10::cuda::OptionalCUDAGuard guard(x.device());
  check(sharq_absmax_sparse_residual_quantize_x(ptr(x), (int)p.m, (int)n, (int)p.k, ptr(amax_bits), (int)amax_bits.numel(), p.a_comp(), p.e(), p.sfa(),
                                                p.q_res(), p.sf_res(), reinterpret_cast<float *>(p.tail()), stream_of(x)));
  std::vector<Tensor> out = p.outputs();
  out.push_back(p.scalar(0));
  return out;
}

void rope_inplace(const Tensor &qkv, int64_t heads, int64_t head_dim, const Tensor &cos, const Tensor &sin, int64_t seq_len) {
  need(qkv.is_cuda() && qkv.scalar_type() == at::kBFloat16 && qkv.dim() == 2 && qkv.stride(1) == 1,
       "qkv must be a CUDA bfloat16 matrix with unit column stride");
  const Tensor *tables[2] = {&cos, &sin};
  for (int i = 0; i < 2; ++i)
    if (!(is_plain(*tables[i], at::kBFloat16) && tables[i]->dim() == 2 && tables[i]->size(0) == seq_len &&
          tables[i]->size(1) == head_dim))
      fail(std::string(i == 0 ? "cos" : "sin") + " must be a contiguous CUDA bfloat16 tensor shaped [seq_len, head_dim]");
  need(heads * head_dim <= qkv.size(1), "heads * head_dim exceeds the row width");
  c10::cuda::OptionalCUDAGuard guard(qkv.device());
  check(sharq_rope_inplace(ptr(qkv), (int)qkv.size(0), (int)qkv.stride(0), (int)seq_len, (int)heads, (int)head_dim, ptr(cos),
                           ptr(sin), stream_of(qkv)));
}

// A paged key/value cache as the C ABI takes it (include/sharq_b200.h): k and v [pages, kv_heads, page_size, head_dim].
sharq_paged_cache cache_of(const Tensor &k, const Tensor &v, const Tensor &table, const std::optional<Tensor> &k_scale,
                           const std::optional<Tensor> &v_scale, const at::Device &dev) {
  need(k.is_cuda() && v.is_cuda() && k.device() == dev && v.device() == dev, "k_cache and v_cache must be CUDA tensors on the device of the input");
  need(k.dim() == 4 && k.sizes() == v.sizes() && k.strides() == v.strides() && k.scalar_type() == v.scalar_type(),
       "k_cache and v_cache must be shaped [pages, kv_heads, page_size, head_dim], alike in shape, strides and type");
  const bool fp8 = k.scalar_type() == at::kFloat8_e4m3fn;
  need(fp8 || k.scalar_type() == at::kBFloat16, "k_cache and v_cache must be torch.bfloat16 or torch.float8_e4m3fn");
  need(k.numel() > 0 && k.stride(3) == 1, "the cache must have pages, and the elements of a head must be contiguous");
  // no two elements at one address: every stride reaches over the dimensions with smaller ones
  std::vector<int> order;
  for (int d = 0; d < 3; ++d)
    if (k.size(d) > 1) order.push_back(d);
  std::sort(order.begin(), order.end(), [&](int a, int b) { return k.stride(a) < k.stride(b); });
  int64_t reach = k.size(3);
  for (int d : order) {
    need(k.stride(d) >= reach, "elements of the cache must not overlap");
    reach = k.stride(d) * k.size(d);
  }
  for (int d = 0; d < 3; ++d) need(k.size(d) <= INT32_MAX, "a dimension of the cache is too large");
  need(table.is_cuda() && table.device() == dev && table.scalar_type() == at::kInt && table.dim() == 2 &&
           (table.size(1) <= 1 || table.stride(1) == 1),
       "page_table must be a CUDA int32 matrix [sequences, pages] with unit column stride on the device of the input");
  need(table.numel() > 0 && table.size(0) <= INT32_MAX && table.size(1) <= INT32_MAX, "page_table must not be empty");
  need(table.size(0) == 1 || table.stride(0) >= table.size(1), "rows of page_table must not overlap");
  const std::optional<Tensor> *scales[2] = {&k_scale, &v_scale};
  for (const auto *s : scales) {
    need(s->has_value() == fp8, "k_scale and v_scale are given for a torch.float8_e4m3fn cache and for no other");
    if (fp8)
      need(is_plain(**s, at::kFloat) && (*s)->device() == dev && (*s)->dim() == 1 && (*s)->size(0) == k.size(1),
           "k_scale and v_scale must be contiguous CUDA float32 vectors with one entry per key/value head");
  }
  sharq_paged_cache c = {};
  c.k = ptr(k);
  c.v = ptr(v);
  c.page_table = static_cast<const int *>(ptr(table));
  c.page_table_stride = table.size(0) > 1 ? table.stride(0) : table.size(1);
  // a dimension of one element has no stride to speak of
  c.page_stride = k.size(0) > 1 ? k.stride(0) : 0;
  c.head_stride = k.size(1) > 1 ? k.stride(1) : 0;
  c.token_stride = k.size(2) > 1 ? k.stride(2) : 0;
  if (fp8) {
    c.k_scale = static_cast<const float *>(ptr(*k_scale));
    c.v_scale = static_cast<const float *>(ptr(*v_scale));
  }
  c.sequences = (int)table.size(0);
  c.max_pages = (int)table.size(1);
  c.pages = (int)k.size(0);
  c.page_size = (int)k.size(2);
  c.kv_heads = (int)k.size(1);
  c.head_dim = (int)k.size(3);
  return c;
}

int *flag_of(const Tensor &flag) { return static_cast<int *>(ptr(flag)); }

void check_indices(const Tensor &t, int64_t n, const at::Device &dev, const char *name) {
  if (!(is_plain(t, at::kInt) && t.device() == dev && t.dim() == 1 && t.size(0) == n))
    fail(std::string(name) + " must be a contiguous CUDA int32 vector with " + std::to_string(n) + " entries on the device of the input");
}

// -> q [rows, heads, head_dim] and, with return_k, k [rows, kv_heads, head_dim]
std::vector<Tensor> rope_append_paged(const Tensor &qkv, int64_t heads, int64_t kv_heads, int64_t head_dim, const Tensor &cos,
                                      const Tensor &sin, const Tensor &positions, const Tensor &table, const Tensor &k_cache,
                                      const Tensor &v_cache, const std::optional<Tensor> &sequences,
                                      const std::optional<Tensor> &k_scale, const std::optional<Tensor> &v_scale, bool return_k,
                                      const Tensor &flag) {
  need(qkv.is_cuda() && qkv.scalar_type() == at::kBFloat16 && qkv.dim() == 2 && qkv.stride(1) == 1,
       "qkv must be a CUDA bfloat16 matrix with unit column stride");
  const at::Device dev = qkv.device();
  const int64_t rows = qkv.size(0);
  need(heads > 0 && kv_heads > 0 && head_dim > 0 && heads <= 65536 && kv_heads <= 65536 && head_dim <= 256,
       "heads and kv_heads must be in [1, 65536], head_dim in [1, 256]");
  need((heads + 2 * kv_heads) * head_dim <= qkv.size(1), "(heads + 2 * kv_heads) * head_dim exceeds the row width");
  const Tensor *tables[2] = {&cos, &sin};
  for (int i = 0; i < 2; ++i)
    if (!(is_plain(*tables[i], at::kBFloat16) && tables[i]->device() == dev && tables[i]->dim() == 2 && tables[i]->size(0) > 0 &&
          tables[i]->sizes() == cos.sizes() && tables[i]->size(1) == head_dim))
      fail(std::string(i == 0 ? "cos" : "sin") + " must be a contiguous CUDA bfloat16 tensor shaped [positions, head_dim]");
  need(rows <= INT32_MAX && cos.size(0) <= INT32_MAX, "too many rows");
  const sharq_paged_cache c = cache_of(k_cache, v_cache, table, k_scale, v_scale, dev);
  need(c.kv_heads == kv_heads && c.head_dim == head_dim, "the cache must have kv_heads heads of head_dim elements");
  check_indices(positions, rows, dev, "positions");
  if (sequences)
    check_indices(*sequences, rows, dev, "sequences");
  else
    need(rows <= c.sequences, "page_table must have a row for every row of qkv when sequences is not given");
  c10::cuda::OptionalCUDAGuard guard(dev);
  Tensor q = empty_like_on(qkv, {rows, heads, head_dim}, at::kBFloat16);
  std::vector<Tensor> out = {q};
  if (return_k) out.push_back(empty_like_on(qkv, {rows, kv_heads, head_dim}, at::kBFloat16));
  if (rows > 0)
    check(sharq_rope_append_paged(ptr(qkv), rows > 1 ? qkv.stride(0) : qkv.size(1) / 8 * 8, (int)rows, (int)heads, ptr(cos), ptr(sin),
                                  (int)cos.size(0), static_cast<const int *>(ptr(positions)),
                                  sequences ? static_cast<const int *>(ptr(*sequences)) : nullptr, &c, ptr(q), return_k ? ptr(out[1]) : nullptr,
                                  flag_of(flag), stream_of(qkv)));
  return out;
}

// A window as the C ABI takes it.
int window_of(const std::optional<int64_t> &window, int64_t sinks) {
  need(!window || *window >= 1, "window must be at least 1, or None");
  need(sinks >= 0, "sinks must not be negative");
  return !window ? 0 : (int)std::min<int64_t>(*window, INT32_MAX);
}

Tensor paged_attention(const Tensor &q, const Tensor &k_cache, const Tensor &v_cache, const Tensor &table, const Tensor &lengths,
                       const std::optional<double> &scale, const std::optional<Tensor> &k_scale, const std::optional<Tensor> &v_scale,
                       const std::optional<Tensor> &out, const Tensor &flag, const std::optional<int64_t> &window, int64_t sinks) {
  const int w = window_of(window, sinks), first = (int)std::min<int64_t>(sinks, INT32_MAX);
  need(q.is_cuda() && q.scalar_type() == at::kBFloat16 && q.dim() == 3 && q.stride(2) == 1,
       "q must be a CUDA bfloat16 tensor shaped [sequences, heads, head_dim] whose heads are contiguous");
  const at::Device dev = q.device();
  const sharq_paged_cache c = cache_of(k_cache, v_cache, table, k_scale, v_scale, dev);
  const int64_t seqs = q.size(0), heads = q.size(1), d = q.size(2);
  need(table.size(0) >= seqs, "page_table must have a row for every row of q");
  need(d == c.head_dim && heads > 0 && heads % c.kv_heads == 0,
       "q must have head_dim elements per head and a multiple of the cache's heads");
  check_indices(lengths, seqs, dev, "lengths");
  if (out)
    need(is_plain(*out, at::kBFloat16) && out->device() == dev && out->sizes() == q.sizes(),
         "out must be a contiguous CUDA bfloat16 tensor shaped like q");
  c10::cuda::OptionalCUDAGuard guard(dev);
  Tensor o = out ? *out : fresh({seqs, heads, d}, at::kBFloat16);
  if (seqs == 0) return o;
  sharq_paged_cache used = c;
  used.sequences = (int)seqs;
  const int64_t ws_bytes = (int64_t)sharq_paged_attention_windowed_workspace_bytes((int)heads, &used, w, first);
  Tensor ws;
  if (ws_bytes > 0) ws = fresh({ws_bytes}, at::kByte);
  check(sharq_paged_attention_windowed(ptr(q), seqs > 1 ? q.stride(0) : 0, heads > 1 ? q.stride(1) : 0, (int)heads, &used,
                                       static_cast<const int *>(ptr(lengths)), (float)(scale ? *scale : 1.0 / std::sqrt((double)d)), w, first, ptr(o),
                                       ws_bytes > 0 ? ptr(ws) : nullptr, (size_t)ws_bytes, flag_of(flag), stream_of(q)));
  return o;
}

Tensor weight_only_linear(const Tensor &x, const Tensor &qw, const Tensor &sf, const std::optional<Tensor> &scale_t, double scale,
                          const std::optional<Tensor> &bias, const std::optional<Tensor> &out, const Tensor &flag) {
  need(x.is_cuda() && x.scalar_type() == at::kBFloat16 && x.dim() == 2 && (x.size(1) <= 1 || x.stride(1) == 1),
       "x must be a CUDA bfloat16 matrix with unit column stride");
  const at::Device dev = x.device();
  const int64_t m = x.size(0), k = x.size(1);
  need(qw.is_cuda() && qw.dim() == 2 && qw.size(0) > 0 && qw.size(0) <= INT32_MAX && k <= INT32_MAX, "qw must be a CUDA matrix [N, K/2]");
  const int64_t n = qw.size(0);
  if (qw.size(1) * 2 != k) fail("qw must have K/2 = " + std::to_string(k / 2) + " columns, got " + std::to_string(qw.size(1)));
  if (k == 0 || k % 64 != 0) fail("weight_only_linear requires K to be a multiple of 64, got " + std::to_string(k));
  if (m > 16) fail("weight_only_linear takes at most 16 rows, got " + std::to_string(m));
  const Tensor *held[2] = {&qw, &sf};
  for (int i = 0; i < 2; ++i)
    if (!(is_plain(*held[i], at::kByte) && held[i]->device() == dev && held[i]->numel() == (i == 0 ? n * (k / 2) : sf_bytes(n, k))))
      fail(std::string(i == 0 ? "qw" : "sfw_dense") + " must be a contiguous CUDA uint8 tensor of " +
           std::to_string(i == 0 ? n * (k / 2) : sf_bytes(n, k)) + " bytes on the device of x");
  check_bias(bias, n, dev);
  const float *scale_dev = scale_t ? scale_ptr(*scale_t, dev, "weight_scale") : nullptr;
  c10::cuda::OptionalCUDAGuard guard(dev);
  Tensor y = output(x, m, n, out);
  if (m == 0) return y;
  check(sharq_weight_only_linear(ptr(x), x.stride(0), (int)m, (int)n, (int)k, ptr(qw), ptr(sf), scale_dev, (float)scale,
                                 bias ? ptr(*bias) : nullptr, ptr(y), flag_of(flag), stream_of(x)));
  return y;
}

Tensor prompt_attention(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &offsets, const std::optional<int64_t> &window,
                        int64_t sinks, const std::optional<double> &scale, const std::optional<Tensor> &k_offsets, const std::optional<Tensor> &out,
                        const Tensor &flag) {
  need(q.is_cuda(), "q must be a CUDA tensor");
  const at::Device dev = q.device();
  const Tensor *held[3] = {&q, &k, &v};
  for (int i = 0; i < 3; ++i)
    if (!(held[i]->is_cuda() && held[i]->device() == dev && held[i]->scalar_type() == at::kBFloat16 && held[i]->dim() == 3 &&
          (held[i]->size(2) <= 1 || held[i]->stride(2) == 1)))
      fail(std::string(1, "qkv"[i]) + " must be a CUDA bfloat16 tensor [rows, heads, head_dim] whose heads are contiguous, on the device of q");
  const int64_t rows = q.size(0), heads = q.size(1), d = q.size(2), k_rows = k.size(0), kv_heads = k.size(1);
  need(k.sizes() == v.sizes(), "k and v must be shaped alike");
  need(k.size(2) == d && kv_heads > 0 && heads > 0 && heads % kv_heads == 0,
       "q must have head_dim elements per head and a multiple of the heads of k");
  if (d != 64 && d != 128) fail("head_dim must be 64 or 128, got " + std::to_string(d));
  need(rows <= 1 << 30 && k_rows <= 1 << 30 && heads <= 65536, "too many rows or heads");
  need(offsets.dim() == 1 && offsets.size(0) >= 2 && offsets.size(0) <= (1 << 24) + 1, "offsets must have an entry for every sequence, at most 2^24, and one more");
  check_indices(offsets, offsets.size(0), dev, "offsets");
  if (k_offsets)
    check_indices(*k_offsets, offsets.size(0), dev, "k_offsets");
  else
    need(k_rows == rows, "without k_offsets k and v must have a row for every row of q");
  const int w = window_of(window, sinks);
  if (out)
    need(is_plain(*out, at::kBFloat16) && out->device() == dev && out->sizes() == q.sizes(),
         "out must be a contiguous CUDA bfloat16 tensor shaped like q");
  int64_t strides[3][2];
  for (int i = 0; i < 3; ++i)
    for (int j = 0; j < 2; ++j) {  // a dimension of one element has no stride to speak of
      strides[i][j] = held[i]->size(j) > 1 ? held[i]->stride(j) : d;
      if (strides[i][j] <= 0 || strides[i][j] % 8 != 0)
        fail(std::string("strides of ") + "qkv"[i] + " must be positive multiples of 8");
    }
  if (out) {  // over the queries, element for element, each block has read its own when it writes; anywhere else the order would matter
    const char *begin = static_cast<const char *>(ptr(*out)), *end = begin + out->nbytes();
    for (int i = 0; i < 3; ++i) {
      const Tensor &t = *held[i];
      if (t.numel() == 0 || out->numel() == 0 || (i == 0 && ptr(t) == begin && t.is_contiguous())) continue;
      const char *from = static_cast<const char *>(ptr(t));
      const int64_t span = ((t.size(0) - 1) * strides[i][0] + (t.size(1) - 1) * strides[i][1] + d) * t.element_size();
      need(from + span <= begin || end <= from, "out must be q or not overlap q, k and v");
    }
  }
  c10::cuda::OptionalCUDAGuard guard(dev);
  Tensor o = out ? *out : fresh({rows, heads, d}, at::kBFloat16);
  if (rows == 0) return o;
  // without any key nothing is read, but the addresses must be some: those of the queries
  const Tensor &keys = k_rows > 0 ? k : q, &values = k_rows > 0 ? v : q;
  const int first = (int)std::min<int64_t>(sinks, INT32_MAX);
  const int64_t ws_bytes = (int64_t)sharq_prompt_attention_workspace_bytes((int)rows, (int)k_rows, (int)heads, (int)kv_heads, (int)d, (int)offsets.size(0) - 1, w, first);
  Tensor ws;
  if (ws_bytes > 0) ws = fresh({ws_bytes}, at::kByte);
  check(sharq_prompt_attention(ptr(q), strides[0][0], strides[0][1], ptr(keys), strides[1][0], strides[1][1], ptr(values), strides[2][0], strides[2][1],
                               (int)rows, (int)k_rows, (int)heads, (int)kv_heads, (int)d, static_cast<const int *>(ptr(offsets)),
                               k_offsets ? static_cast<const int *>(ptr(*k_offsets)) : nullptr, (int)offsets.size(0) - 1, w,
                               first, (float)(scale ? *scale : 1.0 / std::sqrt((double)d)), ptr(o), !out, ws_bytes > 0 ? ptr(ws) : nullptr,
                               (size_t)ws_bytes, flag_of(flag), stream_of(q)));
  return o;
}

// -> offsets [sequences + 1], positions [rows], sequences [rows], views of one allocation
std::vector<Tensor> plan_paged_step(const Tensor &table, const Tensor &lengths, const Tensor &counts, const Tensor &free_pages,
                                    const Tensor &free_count, int64_t page_size, int64_t rows, const std::optional<Tensor> &released,
                                    const std::optional<int64_t> &max_tokens, const Tensor &flag, bool strict) {
  need(table.is_cuda() && table.scalar_type() == at::kInt && table.dim() == 2 && table.numel() > 0 && (table.size(1) <= 1 || table.stride(1) == 1),
       "page_table must be a CUDA int32 matrix [sequences, pages] with unit column stride");
  const at::Device dev = table.device();
  const int64_t n = table.size(0);
  need(n < INT32_MAX && table.size(1) <= INT32_MAX, "page_table is too large");
  need(n == 1 || table.stride(0) >= table.size(1), "rows of page_table must not overlap");
  check_indices(lengths, n, dev, "lengths");
  check_indices(counts, n, dev, "counts");
  need(free_pages.dim() == 1 && free_pages.size(0) <= 1 << 30, "free_pages must be a contiguous CUDA int32 vector of at most 2^30 on the device of the input");
  check_indices(free_pages, free_pages.size(0), dev, "free_pages");
  check_indices(free_count, 1, dev, "free_count");
  need(page_size > 0 && page_size <= INT32_MAX, "page_size must be positive");
  need(rows >= 0 && rows <= 1 << 30, "rows must be in [0, 2^30]");
  need(!max_tokens || *max_tokens > 0, "max_tokens must be positive, or None");
  if (released)
    need((is_plain(*released, at::kBool) || is_plain(*released, at::kByte)) && released->device() == dev && released->dim() == 1 && released->size(0) == n,
         "released must be a contiguous CUDA bool vector with one entry per sequence");
  c10::cuda::OptionalCUDAGuard guard(dev);
  // the parts begin at multiples of 16 bytes, and are made without the dispatcher
  const int64_t at_rows = (n + 4) & ~int64_t(3), padded = (rows + 3) & ~int64_t(3);
  const Tensor out = fresh({at_rows + 2 * padded}, at::kInt);
  int *at = static_cast<int *>(ptr(out));
  auto part = [&](int64_t offset, int64_t size) {
    Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(out.storage()), out.key_set(), c10::scalarTypeToTypeMeta(at::kInt));
    t.unsafeGetTensorImpl()->set_storage_offset(offset);
    t.unsafeGetTensorImpl()->set_sizes_contiguous({size});
    return t;
  };
  const auto plan = strict ? sharq_plan_paged_step_strict : sharq_plan_paged_step;
  check(plan(static_cast<int *>(ptr(table)), n > 1 ? table.stride(0) : table.size(1), (int)n, (int)table.size(1), (int)page_size,
             max_tokens ? (int)std::min<int64_t>(*max_tokens, INT32_MAX) : 0, static_cast<int *>(ptr(lengths)), static_cast<const int *>(ptr(counts)),
             released ? static_cast<const unsigned char *>(ptr(*released)) : nullptr, static_cast<int *>(ptr(free_pages)),
             (int)free_pages.size(0), static_cast<int *>(ptr(free_count)), (int)rows, at, at + at_rows, at + at_rows + padded,
             flag_of(flag), stream_of(table)));
  return {part(0, n + 1), part(at_rows, rows), part(at_rows + padded, rows)};
}

using OptionalTensor = std::optional<Tensor>;

Tensor adjust_logits(const Tensor &logits, const OptionalTensor &tokens, const OptionalTensor &lengths, const OptionalTensor &prompt_lengths,
                     const OptionalTensor &repetition, const OptionalTensor &presence, const OptionalTensor &frequency,
                     const std::optional<std::vector<Tensor>> &bias, const OptionalTensor &mask, const OptionalTensor &out, const Tensor &flag) {
  need(logits.is_cuda() && (logits.scalar_type() == at::kFloat || logits.scalar_type() == at::kBFloat16) && logits.dim() == 2 &&
           (logits.size(1) <= 1 || logits.stride(1) == 1),
       "logits must be a CUDA float32 or bfloat16 matrix [rows, vocab] with unit column stride");
  const at::Device dev = logits.device();
  const int64_t rows = logits.size(0), vocab = logits.size(1);
  need(vocab > 0 && vocab <= 0x7ff00000 && rows <= 65535, "logits must have at most 65535 rows of 1 to 2^31 - 2^20 tokens");
  need(rows <= 1 || logits.stride(0) >= vocab, "rows of logits must not overlap");
  sharq_logit_rules r = {};
  need(tokens.has_value() == lengths.has_value(), "tokens and lengths go together");
  if (tokens) {
    need(tokens->is_cuda() && tokens->device() == dev && (tokens->scalar_type() == at::kInt || tokens->scalar_type() == at::kLong) &&
             tokens->dim() == 2 && tokens->size(0) == rows && tokens->size(1) <= 1 << 30 && (tokens->size(1) <= 1 || tokens->stride(1) == 1),
         "tokens must be a CUDA int32 or int64 matrix of at most 2^30 columns, with a row per row of logits and unit column stride, on their device");
    check_indices(*lengths, rows, dev, "lengths");
    r.tokens = ptr(*tokens);
    r.tokens_stride = rows > 1 ? tokens->stride(0) : 0;
    r.width = (int)tokens->size(1);
    r.wide_tokens = tokens->scalar_type() == at::kLong;
    r.lengths = static_cast<const int *>(ptr(*lengths));
  }
  if (prompt_lengths) {
    check_indices(*prompt_lengths, rows, dev, "prompt_lengths");
    r.prompt_lengths = static_cast<const int *>(ptr(*prompt_lengths));
  }
  const std::pair<const OptionalTensor *, const float **> penalties[3] = {{&repetition, &r.repetition}, {&presence, &r.presence}, {&frequency, &r.frequency}};
  for (const auto &p : penalties)
    if (p.first->has_value()) {
      const Tensor &t = **p.first;
      need(is_plain(t, at::kFloat) && t.device() == dev && t.dim() == 1 && t.size(0) == rows,
           "repetition, presence and frequency must be contiguous CUDA float32 vectors with one entry per row of logits");
      *p.second = static_cast<const float *>(ptr(t));
    }
  need(tokens || !(prompt_lengths || repetition || presence || frequency), "prompt_lengths and the penalties need tokens");
  if (bias) {
    need(bias->size() == 3, "bias must be (offsets, ids, values)");
    const Tensor &ids = (*bias)[1], &values = (*bias)[2];
    check_indices((*bias)[0], rows + 1, dev, "offsets of the biases");
    need(ids.dim() == 1 && ids.size(0) <= 1 << 30, "ids of the biases must be a vector of at most 2^30");
    check_indices(ids, ids.size(0), dev, "ids of the biases");
    need(is_plain(values, at::kFloat) && values.device() == dev && values.sizes() == ids.sizes(),
         "values of the biases must be a contiguous CUDA float32 vector with one entry per id");
    r.bias_offsets = static_cast<const int *>(ptr((*bias)[0]));
    r.bias_ids = static_cast<const int *>(ptr(ids));
    r.bias_values = static_cast<const float *>(ptr(values));
    r.biases = (int)ids.size(0);
  }
  if (mask) {
    need(mask->is_cuda() && mask->device() == dev && mask->scalar_type() == at::kInt && mask->dim() == 2 && mask->size(0) == rows &&
             mask->size(1) == (vocab + 31) / 32 && (mask->size(1) <= 1 || mask->stride(1) == 1),
         "mask must be a CUDA int32 matrix [rows, ceil(vocab / 32)] with unit column stride, on the device of logits");
    r.mask = static_cast<const unsigned *>(ptr(*mask));
    r.mask_stride = rows > 1 ? mask->stride(0) : 0;
  }
  if (out)
    need(out->is_cuda() && out->device() == dev && out->scalar_type() == logits.scalar_type() && out->sizes() == logits.sizes() &&
             (vocab <= 1 || out->stride(1) == 1) && (rows <= 1 || out->stride(0) >= vocab),
         "out must be a CUDA matrix like logits");
  if (out && ptr(*out) != ptr(logits)) {
    const char *a = static_cast<const char *>(ptr(logits)), *b = static_cast<const char *>(ptr(*out));
    const int64_t size = logits.element_size(), last = rows > 0 ? rows - 1 : 0;
    need(a + (last * logits.stride(0) + vocab) * size <= b || b + (last * out->stride(0) + vocab) * size <= a, "out must be logits or not overlap them");
  } else if (out) {
    need(rows <= 1 || out->stride(0) == logits.stride(0), "out must be logits or not overlap them");
  }
  c10::cuda::OptionalCUDAGuard guard(dev);
  Tensor o = out ? *out : fresh({rows, vocab}, logits.scalar_type());
  if (rows == 0) return o;
  check(sharq_adjust_logits(ptr(logits), rows > 1 ? logits.stride(0) : vocab, ptr(o), rows > 1 ? o.stride(0) : vocab, (int)rows, (int)vocab,
                            logits.scalar_type() == at::kBFloat16, &r, flag_of(flag), stream_of(logits)));
  return o;
}

// The GIL is released while a call allocates and launches (a launch waits when the queue of the GPU is full).
template <typename... Args>
auto as_tuple(std::vector<Tensor> (*fn)(Args...)) {
  return [fn](Args... args) {
    std::vector<Tensor> v;
    {
      py::gil_scoped_release nogil;
      v = fn(args...);
    }
    py::tuple t(v.size());
    for (size_t i = 0; i < v.size(); ++i) t[i] = std::move(v[i]);
    return t;
  };
}

}  // namespace

PYBIND11_MODULE(sharq_native, m) {
  static py::object sharq_error = py::module_::import("sharq_b200._lib").attr("SharqError");
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const LibraryError &e) {
      PyErr_SetString(sharq_error.ptr(), e.what());
    }
  });
  using nogil = py::call_guard<py::gil_scoped_release>;
  m.def("scaled_prepare", as_tuple(&scaled_prepare));
  m.def("swiglu_prepare", as_tuple(&swiglu_prepare));
  m.def("scaled_quantize", as_tuple(&scaled_quantize));
  m.def("linear_gemm_swiglu", as_tuple(&linear_gemm_swiglu));
  m.def("absmax_prepare", as_tuple(&absmax_prepare));
  m.def("rope_append_paged", as_tuple(&rope_append_paged));
  m.def("paged_attention", &paged_attention, nogil());
  m.def("weight_only_linear", &weight_only_linear, nogil());
  m.def("prompt_attention", &prompt_attention, nogil());
  m.def("plan_paged_step", as_tuple(&plan_paged_step));
  m.def("adjust_logits", &adjust_logits, nogil());
  m.def("rope_inplace", &rope_inplace, nogil());
  m.def("linear_gemm", &linear_gemm, nogil());
  m.def("linear_forward", &linear_forward, nogil());
  m.def("dense_gemm", &dense_gemm, nogil());
  m.def("sparse_gemm", &sparse_gemm, nogil());
}
