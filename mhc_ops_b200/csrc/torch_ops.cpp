// TORCH_LIBRARY(mhc, ...): the mHC pre-op as registered torch operators over
// the C ABI of libmhc_ops.so (include/mhc_ops.h).
//
//   mhc::fwd(x, phi, alpha, bias, norm_eps, hc_eps)
//       -> (h_in, h_post, h_res, inv_rms, h_mix, h_pre)
//     the reference's mhc_forward_pre(..., outflag=True)
//     (src/forward/golden.py:10-69; Triton call site
//     src/forward/mhc_forward_pre_triton.py:409-417);
//   mhc::bwd(x, phi, alpha, inv_rms, h_mix, h_pre, h_post, dh_in, dh_post,
//            dh_res, gamma?, norm_eps, hc_eps) -> (dx, dphi, dalpha, dbias, dgamma)
//     the reference's mhc_backward_manual (src/backward/golden.py:10-96;
//     Triton call site src/backward/mhc_backward_triton.py:467-473).
//
//   mhc::qk_norm_rope, mhc::qk_norm_rope_bwd, mhc::qk_norm_rope_bwd_into,
//   mhc::orthogonalize, mhc::muon_step_
//     the operators around a training step that the reference has no
//     counterpart of; schemas at the end of this file, semantics in
//     include/mhc_ops.h.
//
// CUDA kernels convert tensors to the ABI's argument structs, allocate the
// outputs, launch on at::cuda::getCurrentCUDAStream() and turn error codes
// into TORCH_CHECK failures.  There is no CPU kernel: CPU tensors fail in the
// dispatcher.  Meta kernels give the output shapes, so FakeTensor tracing
// (torch.compile, torch.export) sees the ops without running them.
//
// Workspaces are cached per (device, stream) and zero-filled once.  After
// every call the workspace's device status word (set when a kernel's bounded
// wait expired) is copied to pinned host memory on a side stream, without
// making the caller's stream wait; the next call through the same workspace,
// or mhc::check_status, reports it as an error.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_runtime.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/library.h>

#include <algorithm>
#include <map>
#include <memory>
#include <mutex>
#include <string>
#include <tuple>
#include <utility>
#include <vector>

#include "mhc_ops.h"

namespace {

// Numbers go into messages as text: streaming one into a message aborted the
// process where the installed torch and this library brought different C++
// runtimes.
std::string str(int64_t v) { return std::to_string(v); }
std::string str(double v) { return std::to_string(v); }
std::string str(at::IntArrayRef v) {
  std::string s = "[";
  for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + std::to_string(v[i]);
  return s + "]";
}

void check_cuda(cudaError_t e, const char* what) {
  TORCH_CHECK(e == cudaSuccess, what, ": ", cudaGetErrorString(e));
}

void check_status(int st, const char* where) {
  TORCH_CHECK(st == MHC_OK, where, ": mhc status ", str((int64_t)st), ": ", mhc_status_string(st),
              st == MHC_ERR_CUDA ? std::string(" (") + mhc_last_cuda_error() + ")" : std::string());
}

// One cached workspace and the watch over its status word.
struct Workspace {
  at::Tensor buf;
  int* host = nullptr;          // pinned copy of the status word
  cudaStream_t side = nullptr;  // where the copy runs
  cudaEvent_t call_done = nullptr, copied = nullptr;
  bool pending = false;
  const char* where = "";

  ~Workspace() {
    // Process teardown may already have unloaded CUDA; errors are ignored.
    if (copied) cudaEventDestroy(copied);
    if (call_done) cudaEventDestroy(call_done);
    if (side) cudaStreamDestroy(side);
    if (host) cudaFreeHost(host);
  }

  void init(int64_t nbytes, const at::Device& dev) {
    buf = at::zeros({std::max<int64_t>(nbytes, 1 << 16)}, at::TensorOptions().dtype(at::kByte).device(dev));
    if (!host) {
      check_cuda(cudaHostAlloc(reinterpret_cast<void**>(&host), sizeof(int), cudaHostAllocDefault), "cudaHostAlloc");
      *host = 0;
      check_cuda(cudaStreamCreateWithFlags(&side, cudaStreamNonBlocking), "cudaStreamCreate");
      check_cuda(cudaEventCreateWithFlags(&call_done, cudaEventDisableTiming), "cudaEventCreate");
      check_cuda(cudaEventCreateWithFlags(&copied, cudaEventDisableTiming), "cudaEventCreate");
    }
  }

  // Raise if an earlier call reported an expired device wait (its outputs are
  // invalid); the word is cleared first.  wait: block until the last copy lands.
  void raise_if_timed_out(cudaStream_t stream, bool wait) {
    if (!pending) return;
    if (wait) {
      check_cuda(cudaEventSynchronize(copied), "cudaEventSynchronize");
    } else if (cudaEventQuery(copied) != cudaSuccess) {
      (void)cudaGetLastError();   // cudaErrorNotReady: look again at the next call
      return;
    }
    pending = false;
    const int code = *host;
    if (code != MHC_OK) {
      *host = 0;
      check_cuda(cudaMemsetAsync(buf.data_ptr(), 0, sizeof(int), stream), "cudaMemsetAsync");
      check_status(code, (std::string(where) + " (an earlier call; its outputs are invalid)").c_str());
    }
  }

  void watch(cudaStream_t stream, const char* name) {
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    check_cuda(cudaStreamIsCapturing(stream, &cap), "cudaStreamIsCapturing");
    if (cap != cudaStreamCaptureStatusNone) return;   // no host-visible copy inside a graph capture
    where = name;
    check_cuda(cudaEventRecord(call_done, stream), "cudaEventRecord");
    check_cuda(cudaStreamWaitEvent(side, call_done, 0), "cudaStreamWaitEvent");
    check_cuda(cudaMemcpyAsync(host, buf.data_ptr(), sizeof(int), cudaMemcpyDeviceToHost, side), "cudaMemcpyAsync");
    check_cuda(cudaEventRecord(copied, side), "cudaEventRecord");
    pending = true;
  }
};

std::mutex g_ws_mu;
std::map<std::pair<int, cudaStream_t>, std::unique_ptr<Workspace>> g_ws;

Workspace& workspace(int64_t nbytes, const at::Device& dev, cudaStream_t stream) {
  std::lock_guard<std::mutex> lk(g_ws_mu);
  auto& slot = g_ws[{dev.index(), stream}];
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  check_cuda(cudaStreamIsCapturing(stream, &cap), "cudaStreamIsCapturing");
  if (cap != cudaStreamCaptureStatusNone) {
    // inside a CUDA graph capture nothing may be allocated or synchronised:
    // the workspace must come from a call on this stream before the capture
    TORCH_CHECK(slot && slot->buf.defined() && slot->buf.numel() >= nbytes,
                "mhc: no workspace for this stream while it is capturing a CUDA graph; run the same call once "
                "on the capturing stream before the capture");
    return *slot;
  }
  if (!slot) slot = std::make_unique<Workspace>();
  if (slot->buf.defined()) slot->raise_if_timed_out(stream, /*wait=*/slot->buf.numel() < nbytes);
  if (!slot->buf.defined() || slot->buf.numel() < nbytes) slot->init(nbytes, dev);
  return *slot;
}

at::Tensor f32(const at::Tensor& t, const at::Device& dev, const char* name) {
  TORCH_CHECK(t.device() == dev, name, " is on ", t.device(), ", x is on ", dev);
  return t.to(at::kFloat).contiguous();
}

void check_x(const at::Tensor& x) {
  TORCH_CHECK(x.dim() == 4, "x must be [B, S, n, D]");
  TORCH_CHECK(x.is_cuda(), "mhc ops run on CUDA only (there is no CPU fallback)");
  TORCH_CHECK(x.scalar_type() == at::kBFloat16, "x must be bfloat16, got ", x.scalar_type());
}

void check_shape(const at::Tensor& t, at::IntArrayRef want, const char* name) {
  TORCH_CHECK(t.sizes() == want, name, " must be ", str(want), ", got ", str(t.sizes()));
}

}  // namespace

// ----------------------------------------------------------------- CUDA kernels
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> mhc_fwd_cuda(
    const at::Tensor& x_in, const at::Tensor& phi_in, const at::Tensor& alpha_in, const at::Tensor& bias_in,
    double norm_eps, double hc_eps) {
  check_x(x_in);
  const at::Device dev = x_in.device();
  c10::cuda::CUDAGuard guard(dev);
  const int64_t B = x_in.size(0), S = x_in.size(1), n = x_in.size(2), D = x_in.size(3);
  const int64_t N = n * n + 2 * n, T = B * S;
  const at::Tensor x = x_in.contiguous();
  const at::Tensor phi = f32(phi_in, dev, "phi"), alpha = f32(alpha_in, dev, "alpha"), bias = f32(bias_in, dev, "bias");
  check_shape(phi, {N, n * D}, "phi");
  TORCH_CHECK(alpha.numel() == 3 && bias.numel() == N, "alpha must have 3 elements and bias n*n+2n");
  const auto o = x.options();
  at::Tensor h_in = at::empty({B, S, D}, o);
  at::Tensor h_post = at::empty({B, S, n}, o.dtype(at::kFloat));
  at::Tensor h_res = at::empty({B, S, n, n}, o.dtype(at::kFloat));
  at::Tensor inv_rms = at::empty({B, S}, o.dtype(at::kFloat));
  at::Tensor h_mix = at::empty({B, S, N}, o.dtype(at::kFloat));
  at::Tensor h_pre = at::empty({B, S, n}, o.dtype(at::kFloat));
  size_t nbytes = 0;
  check_status(mhc_fwd_workspace_size(T, (int32_t)n, (int32_t)D, &nbytes), "mhc_fwd_workspace_size");
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(dev.index()).stream();
  Workspace& ws = workspace((int64_t)nbytes, dev, stream);
  mhc_fwd_args a{};
  a.x = static_cast<const uint16_t*>(x.data_ptr());
  a.phi = phi.data_ptr<float>();
  a.alpha = alpha.data_ptr<float>();
  a.bias = bias.data_ptr<float>();
  a.h_in = static_cast<uint16_t*>(h_in.data_ptr());
  a.h_post = h_post.data_ptr<float>();
  a.h_res = h_res.data_ptr<float>();
  a.inv_rms = inv_rms.data_ptr<float>();
  a.h_mix = h_mix.data_ptr<float>();
  a.h_pre = h_pre.data_ptr<float>();
  a.tokens = T;
  a.n = (int32_t)n;
  a.D = (int32_t)D;
  a.norm_eps = (float)norm_eps;
  a.hc_eps = (float)hc_eps;
  a.workspace = ws.buf.data_ptr();
  a.workspace_bytes = (size_t)ws.buf.numel();
  check_status(mhc_fwd(&a, stream), "mhc::fwd");
  ws.watch(stream, "mhc::fwd");
  return {h_in, h_post, h_res, inv_rms, h_mix, h_pre};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> mhc_bwd_cuda(
    const at::Tensor& x_in, const at::Tensor& phi_in, const at::Tensor& alpha_in, const at::Tensor& inv_rms_in,
    const at::Tensor& h_mix_in, const at::Tensor& h_pre_in, const at::Tensor& h_post_in, const at::Tensor& dh_in_in,
    const at::Tensor& dh_post_in, const at::Tensor& dh_res_in, const c10::optional<at::Tensor>& gamma_in,
    double norm_eps, double hc_eps) {
  check_x(x_in);
  const at::Device dev = x_in.device();
  c10::cuda::CUDAGuard guard(dev);
  const int64_t B = x_in.size(0), S = x_in.size(1), n = x_in.size(2), D = x_in.size(3);
  const int64_t N = n * n + 2 * n, nD = n * D, T = B * S;
  const at::Tensor x = x_in.contiguous();
  const at::Tensor phi = f32(phi_in, dev, "phi"), alpha = f32(alpha_in, dev, "alpha");
  const at::Tensor inv_rms = f32(inv_rms_in, dev, "inv_rms"), h_mix = f32(h_mix_in, dev, "h_mix");
  const at::Tensor h_pre = f32(h_pre_in, dev, "h_pre"), h_post = f32(h_post_in, dev, "h_post");
  const at::Tensor dh_post = f32(dh_post_in, dev, "dh_post"), dh_res = f32(dh_res_in, dev, "dh_res");
  TORCH_CHECK(dh_in_in.device() == dev, "dh_in must be on x's device");
  const at::Tensor dh_in = dh_in_in.to(at::kBFloat16).contiguous();
  at::Tensor gamma;
  if (gamma_in.has_value() && gamma_in->defined()) {
    gamma = f32(*gamma_in, dev, "gamma");
    TORCH_CHECK(gamma.numel() == nD, "gamma must have n*D elements");
  }
  check_shape(phi, {N, nD}, "phi");
  check_shape(inv_rms, {B, S}, "inv_rms");
  check_shape(h_mix, {B, S, N}, "h_mix");
  check_shape(h_pre, {B, S, n}, "h_pre");
  check_shape(h_post, {B, S, n}, "h_post");
  check_shape(dh_in, {B, S, D}, "dh_in");
  check_shape(dh_post, {B, S, n}, "dh_post");
  check_shape(dh_res, {B, S, n, n}, "dh_res");
  TORCH_CHECK(alpha.numel() == 3, "alpha must have 3 elements");
  const auto o = x.options();
  at::Tensor dx = at::empty({B, S, n, D}, o);
  at::Tensor dphi = at::empty({N, nD}, o.dtype(at::kFloat));
  at::Tensor dalpha = at::empty({3}, o.dtype(at::kFloat));
  at::Tensor dbias = at::empty({N}, o.dtype(at::kFloat));
  at::Tensor dgamma = at::empty({nD}, o.dtype(at::kFloat));
  size_t nbytes = 0;
  check_status(mhc_bwd_workspace_size(T, (int32_t)n, (int32_t)D, &nbytes), "mhc_bwd_workspace_size");
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(dev.index()).stream();
  Workspace& ws = workspace((int64_t)nbytes, dev, stream);
  mhc_bwd_args a{};
  a.x = static_cast<const uint16_t*>(x.data_ptr());
  a.phi = phi.data_ptr<float>();
  a.alpha = alpha.data_ptr<float>();
  a.bias = nullptr;
  a.inv_rms = inv_rms.data_ptr<float>();
  a.h_mix = h_mix.data_ptr<float>();
  a.h_pre = h_pre.data_ptr<float>();
  a.h_post = h_post.data_ptr<float>();
  a.dh_in = static_cast<const uint16_t*>(dh_in.data_ptr());
  a.dh_post = dh_post.data_ptr<float>();
  a.dh_res = dh_res.data_ptr<float>();
  a.gamma = gamma.defined() ? gamma.data_ptr<float>() : nullptr;
  a.dx = static_cast<uint16_t*>(dx.data_ptr());
  a.dphi = dphi.data_ptr<float>();
  a.dalpha = dalpha.data_ptr<float>();
  a.dbias = dbias.data_ptr<float>();
  a.dgamma = dgamma.data_ptr<float>();
  a.tokens = T;
  a.n = (int32_t)n;
  a.D = (int32_t)D;
  a.norm_eps = (float)norm_eps;
  a.hc_eps = (float)hc_eps;
  a.workspace = ws.buf.data_ptr();
  a.workspace_bytes = (size_t)ws.buf.numel();
  check_status(mhc_bwd(&a, stream), "mhc::bwd");
  ws.watch(stream, "mhc::bwd");
  return {dx, dphi, dalpha, dbias, dgamma};
}

// Waits for the status copies of every workspace of the op layer and raises
// if any call reported an expired device wait.
int64_t mhc_check_status() {
  std::lock_guard<std::mutex> lk(g_ws_mu);
  for (auto& kv : g_ws) {
    c10::cuda::CUDAGuard guard(kv.first.first);
    if (kv.second->buf.defined()) kv.second->raise_if_timed_out(kv.first.second, /*wait=*/true);
  }
  return 0;
}

// ----------------------------------------------------------------- queries, keys, positions
namespace {

using OptTensor = c10::optional<at::Tensor>;

bool given(const OptTensor& t) { return t.has_value() && t->defined(); }

// Scratch of one call, from torch's allocator on the current stream: two
// streams, threads or captured graphs never share it.
at::Tensor scratch(size_t nbytes, const at::Device& dev) {
  return at::detail::empty_cuda({(int64_t)nbytes}, at::TensorOptions().dtype(at::kByte).device(dev));
}

// Autograd has to see that these were written.
void mark_written(at::TensorList tensors) {
  for (const at::Tensor& t : tensors)
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

int dtype_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return MHC_BF16;
    case at::kHalf: return MHC_F16;
    case at::kFloat: return MHC_F32;
    default: return -1;
  }
}

at::Tensor f32_of(const at::Tensor& t, const at::Device& dev, const char* name) {
  TORCH_CHECK_VALUE(t.device() == dev, name, " is on ", t.device(), ", q is on ", dev);
  return t.to(at::kFloat).contiguous();
}

mhc_heads heads_of(const at::Tensor& t) {
  mhc_heads h{};
  h.data = t.data_ptr();
  h.batch_stride = t.stride(0);
  h.seq_stride = t.stride(1);
  h.head_stride = t.stride(2);
  return h;
}

// A [B, S, heads, d] tensor of the call; heads < 0: any number.
void check_heads(const at::Tensor& t, const char* name, const at::Tensor& like, int64_t heads) {
  TORCH_CHECK_VALUE(t.dim() == 4, name, " must be a tensor of shape [B, S, heads, d]");
  TORCH_CHECK_TYPE(dtype_code(t) >= 0, name, " must be bfloat16, float16 or float32, got ", t.scalar_type());
  TORCH_CHECK_VALUE(t.size(0) == like.size(0) && t.size(1) == like.size(1) && t.size(3) == like.size(3) &&
                        (heads < 0 || t.size(2) == heads),
                    name, " must be [", str(like.size(0)), ", ", str(like.size(1)), ", ",
                    heads < 0 ? std::string("heads") : str(heads), ", ", str(like.size(3)), "], got ", str(t.sizes()));
  TORCH_CHECK_VALUE(t.scalar_type() == like.scalar_type() && t.device() == like.device(), name, " is ",
                    t.scalar_type(), " on ", t.device(), ", expected ", like.scalar_type(), " on ", like.device());
}

at::Tensor unit_inner(const at::Tensor& t) { return t.size(3) <= 1 || t.stride(3) == 1 ? t : t.contiguous(); }

// The checked inputs of either direction and the tensors that own them.
struct QkInputs {
  mhc_qk_args a{};
  at::Tensor q, k, v, inv_freq, q_weight, k_weight, row_scale, positions;
};

QkInputs qk_inputs(const at::Tensor& q, const at::Tensor& k, const OptTensor& positions, const at::Tensor& inv_freq,
                   const OptTensor& q_weight, const OptTensor& k_weight, const OptTensor& v,
                   const OptTensor& row_scale, double eps, bool interleaved) {
  QkInputs in;
  check_heads(q, "q", q, -1);
  check_heads(k, "k", q, -1);
  const at::Device dev = q.device();
  const int64_t B = q.size(0), S = q.size(1), d = q.size(3);
  in.q = unit_inner(q);
  in.k = unit_inner(k);
  in.a.q = heads_of(in.q);
  in.a.k = heads_of(in.k);
  TORCH_CHECK_VALUE(d >= 1 && d <= 1024, "d must be at least 1 and at most 1024, got ", str(d));
  TORCH_CHECK_VALUE(q.size(2) >= 1 && k.size(2) >= 1, "q and k need at least one head");
  if (given(v)) {
    check_heads(*v, "v", q, -1);
    TORCH_CHECK_VALUE(v->size(2) >= 1, "v needs at least one head");
    in.v = unit_inner(*v);
    in.a.v = heads_of(in.v);
    in.a.v_heads = (int32_t)v->size(2);
  }
  in.inv_freq = f32_of(inv_freq, dev, "inv_freq");
  const int64_t rot = 2 * in.inv_freq.numel();
  TORCH_CHECK_VALUE(in.inv_freq.dim() == 1 && rot <= d, "inv_freq must be [rot / 2] with rot <= d = ", str(d), ", got ",
                    str(inv_freq.sizes()));
  in.a.inv_freq = in.inv_freq.data_ptr<float>();
  auto weight = [&](const OptTensor& w, const char* name, at::Tensor& keep, const float*& dst) {
    if (!given(w)) return;
    TORCH_CHECK_VALUE(w->dim() == 1 && w->size(0) == d, name, " must be [", str(d), "], got ", str(w->sizes()));
    keep = f32_of(*w, dev, name);
    dst = keep.data_ptr<float>();
  };
  weight(q_weight, "q_weight", in.q_weight, in.a.q_weight);
  weight(k_weight, "k_weight", in.k_weight, in.a.k_weight);
  if (given(row_scale)) {
    TORCH_CHECK_VALUE(row_scale->dim() == 2 && row_scale->size(0) == B && row_scale->size(1) == S,
                      "row_scale must be [", str(B), ", ", str(S), "], got ", str(row_scale->sizes()));
    in.row_scale = f32_of(*row_scale, dev, "row_scale");
    in.a.row_scale = in.row_scale.data_ptr<float>();
  }
  if (given(positions)) {
    const at::Tensor& p = *positions;
    TORCH_CHECK_TYPE(p.scalar_type() == at::kInt || p.scalar_type() == at::kLong,
                     "positions must be an int32 or int64 tensor");
    TORCH_CHECK_VALUE(p.device() == dev, "positions is on ", p.device(), ", q is on ", dev);
    if (p.dim() == 2 && p.size(0) == B && p.size(1) == S) {
      in.a.position_batch_stride = p.stride(0);
      in.a.position_seq_stride = p.stride(1);
    } else {
      TORCH_CHECK_VALUE(p.dim() == 1 && p.size(0) == S, "positions must be [", str(B), ", ", str(S), "] or [", str(S),
                        "], got ", str(p.sizes()));
      in.a.position_seq_stride = p.stride(0);
    }
    in.positions = p;
    in.a.positions = p.data_ptr();
    in.a.position_bytes = (int32_t)p.element_size();
  }
  TORCH_CHECK_VALUE(eps >= 0, "eps must not be negative, got ", str(eps));
  in.a.batch = B;
  in.a.seq = S;
  in.a.q_heads = (int32_t)q.size(2);
  in.a.k_heads = (int32_t)k.size(2);
  in.a.d = (int32_t)d;
  in.a.rot = (int32_t)rot;
  in.a.interleaved = interleaved ? 1 : 0;
  in.a.dtype = dtype_code(q);
  in.a.eps = (float)eps;
  return in;
}

// Past the dispatcher: some 0.3 us less for each tensor of a call.
at::Tensor empty_like_heads(const at::Tensor& t) { return at::detail::empty_cuda(t.sizes(), t.options()); }

// First byte and the byte behind the last one a strided tensor reaches.
std::pair<uintptr_t, uintptr_t> span_of(const at::Tensor& t) {
  int64_t last = 0;
  for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
  const uintptr_t lo = reinterpret_cast<uintptr_t>(t.data_ptr());
  return {lo, lo + (uintptr_t)(last + 1) * t.element_size()};
}

// Whether two [B, S, heads, d] tensors of unit stride along d share a byte.  Equal
// strides decide it (slices of one packed tensor interleave without meeting): a
// row of one meets a row of the other when the distance of the bases is off a sum
// of strides by less than a row.  Other strides leave it open where the spans meet.
enum class Shared { kNo, kYes, kOpen };
struct Axis {
  int64_t stride, a, b;   // bytes; sizes in either tensor
};
Shared rows_meet(int64_t gap, const Axis* axis, int n, int64_t row) {
  if (n == 0) return gap < row && -gap < row ? Shared::kYes : Shared::kNo;
  int64_t reach = row;   // rows of the inner axes meet only when the rest of the gap is below this
  for (int i = 1; i < n; ++i) reach += axis[i].stride * (std::max(axis[i].a, axis[i].b) - 1);
  const int64_t s = axis->stride;
  auto floor_div = [](int64_t x, int64_t y) { return x / y - (x % y != 0 && x < 0); };
  const int64_t lo = std::max(1 - axis->a, floor_div(-reach - gap, s) + 1), hi = std::min(axis->b - 1, floor_div(reach - gap, s));
  if (hi - lo > 64) return Shared::kOpen;
  Shared seen = Shared::kNo;
  for (int64_t k = lo; k <= hi && seen != Shared::kYes; ++k) {
    const Shared r = rows_meet(gap + k * s, axis + 1, n - 1, row);
    if (r != Shared::kNo) seen = r;
  }
  return seen;
}
Shared shared(const at::Tensor& t, const at::Tensor& u) {
  const auto a = span_of(t), b = span_of(u);
  if (a.first >= b.second || b.first >= a.second) return Shared::kNo;
  Axis axis[3];
  int n = 0;
  for (int64_t j = 0; j < 3; ++j) {
    const int64_t st = t.size(j) > 1 ? t.stride(j) : u.stride(j), su = u.size(j) > 1 ? u.stride(j) : t.stride(j);
    if (t.size(j) == 1 && u.size(j) == 1) continue;
    if (st != su || st == 0) return Shared::kOpen;
    axis[n++] = {st * (int64_t)t.element_size(), t.size(j), u.size(j)};
  }
  std::sort(axis, axis + n, [](const Axis& x, const Axis& y) { return x.stride > y.stride; });
  return rows_meet((int64_t)(b.first - a.first), axis, n, t.size(3) * (int64_t)t.element_size());
}

}  // namespace

std::vector<at::Tensor> qk_norm_rope_cuda(const at::Tensor& q, const at::Tensor& k, const OptTensor& positions,
                                          const at::Tensor& inv_freq, const OptTensor& q_weight,
                                          const OptTensor& k_weight, const OptTensor& v, const OptTensor& row_scale,
                                          double eps, bool interleaved) {
  c10::cuda::CUDAGuard guard(q.device());
  QkInputs in = qk_inputs(q, k, positions, inv_freq, q_weight, k_weight, v, row_scale, eps, interleaved);
  std::vector<at::Tensor> out{empty_like_heads(q), empty_like_heads(k)};
  in.a.q_out = heads_of(out[0]);
  in.a.k_out = heads_of(out[1]);
  if (in.v.defined()) {
    out.push_back(empty_like_heads(in.v));
    in.a.v_out = heads_of(out[2]);
  }
  check_status(mhc_qk_norm_rope(&in.a, at::cuda::getCurrentCUDAStream().stream()), "mhc::qk_norm_rope");
  return out;
}

std::vector<at::Tensor> qk_norm_rope_bwd_into_cuda(
    const at::Tensor& q, const at::Tensor& k, const OptTensor& positions, const at::Tensor& inv_freq,
    const at::Tensor& dq_out, const at::Tensor& dk_out, const OptTensor& q_weight, const OptTensor& k_weight,
    const OptTensor& v, const OptTensor& dv_out, const OptTensor& row_scale, double eps, bool interleaved,
    bool weight_grads, bool row_scale_grad, at::TensorList grad_out) {
  c10::cuda::CUDAGuard guard(q.device());
  mhc_qk_bwd_args b{};
  QkInputs in = qk_inputs(q, k, positions, inv_freq, q_weight, k_weight, v, row_scale, eps, interleaved);
  TORCH_CHECK_VALUE(given(v) == given(dv_out), "v and dv_out go together");
  const size_t count = given(v) ? 3 : 2;
  static const char* const up_names[3] = {"dq_out", "dk_out", "dv_out"};
  static const char* const grad_names[3] = {"grad_out dq", "grad_out dk", "grad_out dv"};
  const at::Tensor inputs[3] = {in.q, in.k, in.v};
  at::Tensor ups[3] = {dq_out, dk_out, given(dv_out) ? *dv_out : at::Tensor()};
  mhc_heads* const up_dst[3] = {&b.dq_out, &b.dk_out, &b.dv_out};
  mhc_heads* const grad_dst[3] = {&b.dq, &b.dk, &b.dv};
  TORCH_CHECK_VALUE(grad_out.size() == count, "grad_out must hold ", str((int64_t)count), " tensors");
  for (size_t i = 0; i < count; ++i) {
    check_heads(ups[i], up_names[i], in.q, inputs[i].size(2));
    ups[i] = unit_inner(ups[i]);
    *up_dst[i] = heads_of(ups[i]);
    const at::Tensor& g = grad_out[i];
    check_heads(g, grad_names[i], in.q, inputs[i].size(2));
    TORCH_CHECK_VALUE(g.size(3) == 1 || g.stride(3) == 1, grad_names[i], " must have unit stride along d");
    for (int64_t j = 0; j < 3; ++j) {
      TORCH_CHECK_VALUE(g.stride(j) != 0 || g.size(j) <= 1, grad_names[i], " must not be an expanded tensor");
      TORCH_CHECK_VALUE(g.stride(j) >= g.size(3) || g.size(j) <= 1, grad_names[i], " overlaps itself");
    }
    *grad_dst[i] = heads_of(g);
  }
  if (q.numel() > 0)
    for (size_t i = 0; i < count; ++i) {
      for (size_t j = 0; j < 2 * count; ++j)
        TORCH_CHECK_VALUE(shared(grad_out[i], j < count ? inputs[j] : ups[j - count]) == Shared::kNo, grad_names[i],
                          " overlaps an input");
      const auto w = span_of(grad_out[i]);
      for (const at::Tensor& t : {in.q_weight, in.k_weight, in.row_scale, in.inv_freq, in.positions})
        if (t.defined() && t.numel() > 0) {
          const auto r = span_of(t);
          TORCH_CHECK_VALUE(w.first >= r.second || r.first >= w.second, grad_names[i], " overlaps an input");
        }
      // of another layout: the caller's word
      for (size_t j = 0; j < i; ++j)
        TORCH_CHECK_VALUE(shared(grad_out[i], grad_out[j]) != Shared::kYes, grad_names[i], " overlaps ", grad_names[j]);
    }
  std::vector<at::Tensor> out;
  const auto f = q.options().dtype(at::kFloat);
  if (in.q_weight.defined() && weight_grads) {
    out.push_back(at::detail::empty_cuda({q.size(3)}, f));
    b.dq_weight = out.back().data_ptr<float>();
  }
  if (in.k_weight.defined() && weight_grads) {
    out.push_back(at::detail::empty_cuda({q.size(3)}, f));
    b.dk_weight = out.back().data_ptr<float>();
  }
  if (in.row_scale.defined() && row_scale_grad) {
    out.push_back(at::detail::empty_cuda({q.size(0), q.size(1)}, f));
    b.d_row_scale = out.back().data_ptr<float>();
  }
  at::Tensor ws;
  if (b.dq_weight || b.dk_weight) {
    check_status(mhc_qk_norm_rope_bwd_workspace_size(q.size(0) * q.size(1), in.a.d, &b.workspace_bytes),
                 "mhc_qk_norm_rope_bwd_workspace_size");
    ws = scratch(b.workspace_bytes, q.device());
    b.workspace = ws.data_ptr();
  }
  b.fwd = in.a;
  check_status(mhc_qk_norm_rope_bwd(&b, at::cuda::getCurrentCUDAStream().stream()), "mhc::qk_norm_rope_bwd");
  mark_written(grad_out);
  return out;
}

std::vector<at::Tensor> qk_norm_rope_bwd_cuda(const at::Tensor& q, const at::Tensor& k, const OptTensor& positions,
                                              const at::Tensor& inv_freq, const at::Tensor& dq_out,
                                              const at::Tensor& dk_out, const OptTensor& q_weight,
                                              const OptTensor& k_weight, const OptTensor& v, const OptTensor& dv_out,
                                              const OptTensor& row_scale, double eps, bool interleaved,
                                              bool weight_grads, bool row_scale_grad) {
  c10::cuda::CUDAGuard guard(q.device());
  std::vector<at::Tensor> grads{empty_like_heads(q), empty_like_heads(k)};
  if (given(v)) grads.push_back(empty_like_heads(*v));
  for (auto& t : qk_norm_rope_bwd_into_cuda(q, k, positions, inv_freq, dq_out, dk_out, q_weight, k_weight, v, dv_out,
                                            row_scale, eps, interleaved, weight_grads, row_scale_grad, grads))
    grads.push_back(std::move(t));
  return grads;
}

// ----------------------------------------------------------------- updates of phi
namespace {

// Equal matrices: one [rows, cols] or [count, rows, cols] tensor, or a list of [rows, cols].
struct Mats {
  std::vector<at::Tensor> keep;   // contiguous copies
  std::vector<void*> ptrs;
  int64_t rows = 0, cols = 0;
  int dtype = 0;
  at::Device dev = at::kCPU;
};

Mats mats_of(at::TensorList x, const char* name, bool copy) {
  Mats m;
  TORCH_CHECK_VALUE(!x.empty(), name, " must not be an empty sequence");
  const at::Tensor& t0 = x[0];
  const int64_t dim = t0.dim();
  TORCH_CHECK_VALUE(dim == 2 || (dim == 3 && x.size() == 1), name,
                    " must be [rows, cols], [count, rows, cols] or a sequence of [rows, cols]");
  m.rows = t0.size(dim - 2);
  m.cols = t0.size(dim - 1);
  m.dev = t0.device();
  m.dtype = dtype_code(t0);
  TORCH_CHECK_TYPE(m.dtype == MHC_F32 || m.dtype == MHC_BF16, name, " must be float32 or bfloat16, got ",
                   t0.scalar_type());
  TORCH_CHECK_VALUE(std::min(m.rows, m.cols) <= 80, name, " is ", str(m.rows), " x ", str(m.cols),
                    ": the shorter side may have at most 80 rows");
  m.ptrs.reserve(dim == 3 ? (size_t)t0.size(0) : x.size());
  for (size_t i = 0; i < x.size(); ++i) {
    at::Tensor t = x[i];
    TORCH_CHECK_VALUE(t.sizes() == t0.sizes() && t.scalar_type() == t0.scalar_type() && t.device() == m.dev, name, "[",
                      str((int64_t)i), "] is ", t.scalar_type(), " ", str(t.sizes()), " on ", t.device(), ", ", name,
                      "[0] is ", t0.scalar_type(), " ", str(t0.sizes()), " on ", m.dev);
    if (!t.is_contiguous()) {
      TORCH_CHECK_VALUE(copy, name, "[", str((int64_t)i), "] must be contiguous");
      t = t.contiguous();
      m.keep.push_back(t);
    }
    char* p = static_cast<char*>(t.data_ptr());
    if (dim == 2) {
      m.ptrs.push_back(p);
    } else {
      for (int64_t j = 0; j < t.size(0); ++j) m.ptrs.push_back(p + j * m.rows * m.cols * t.element_size());
    }
  }
  return m;
}

// Host doubles of the steps; count of triples.
int32_t check_coeffs(at::ArrayRef<double> coeffs, double eps) {
  TORCH_CHECK_VALUE(!coeffs.empty() && coeffs.size() % 3 == 0 && coeffs.size() <= 48,
                    "coeffs must be 1 to 16 triples (a, b, c)");
  TORCH_CHECK_VALUE(eps >= 1e-20, "eps must be at least 1e-20, got ", str(eps));
  return (int32_t)(coeffs.size() / 3);
}

at::Tensor ortho_workspace(const Mats& m, size_t* nbytes, void** ptr) {
  check_status(mhc_ortho_workspace_size((int64_t)m.ptrs.size(), (int32_t)m.rows, (int32_t)m.cols, nbytes),
               "mhc_ortho_workspace_size");
  at::Tensor ws;
  if (*nbytes > 0) ws = scratch(*nbytes, m.dev);
  *ptr = ws.defined() ? ws.data_ptr() : nullptr;
  return ws;
}

void check_sizes(const Mats& m) {
  TORCH_CHECK_VALUE(std::max(m.rows, m.cols) <= (1 << 30), "a side of more than 2^30");
}

}  // namespace

std::vector<at::Tensor> orthogonalize_cuda(at::TensorList g, at::ArrayRef<double> coeffs, double eps) {
  mhc_ortho_args a{};
  a.steps = check_coeffs(coeffs, eps);
  c10::cuda::CUDAGuard guard(g.empty() ? at::Device(at::kCUDA, at::cuda::current_device()) : g[0].device());
  const Mats m = mats_of(g, "g", true);
  check_sizes(m);
  const int64_t count = (int64_t)m.ptrs.size();
  // a tensor for each given one: outputs of an operator do not share memory
  std::vector<at::Tensor> out;
  std::vector<void*> dst;
  out.reserve(g.size());
  dst.reserve(m.ptrs.size());
  for (size_t i = 0; i < g.size(); ++i) {
    out.push_back(at::detail::empty_cuda(g[i].sizes(), g[i].options()));   // past the dispatcher: lists are long
    char* p = static_cast<char*>(out.back().data_ptr());
    const int64_t mats = g[i].dim() == 3 ? count : 1, step = m.rows * m.cols * (int64_t)out.back().element_size();
    for (int64_t j = 0; j < mats; ++j) dst.push_back(p + j * step);
  }
  const at::Tensor ws = ortho_workspace(m, &a.workspace_bytes, &a.workspace);
  a.in = m.ptrs.data();
  a.out = dst.data();
  a.count = count;
  a.rows = (int32_t)m.rows;
  a.cols = (int32_t)m.cols;
  a.dtype = m.dtype;
  a.coeffs = coeffs.data();
  a.eps = eps;
  check_status(mhc_orthogonalize(&a, at::cuda::getCurrentCUDAStream().stream()), "mhc::orthogonalize");
  return out;
}

void muon_step_cuda(at::TensorList params, at::TensorList grads, at::TensorList momenta, const OptTensor& lr_tensor,
                    double lr, double momentum, bool nesterov, double weight_decay, double scale,
                    at::ArrayRef<double> coeffs, double eps) {
  mhc_muon_args a{};
  a.steps = check_coeffs(coeffs, eps);
  c10::cuda::CUDAGuard guard(params.empty() ? at::Device(at::kCUDA, at::cuda::current_device()) : params[0].device());
  const Mats p = mats_of(params, "params", false), g = mats_of(grads, "grads", true),
             m = mats_of(momenta, "momenta", false);
  check_sizes(p);
  TORCH_CHECK_VALUE(p.ptrs.size() == g.ptrs.size() && p.ptrs.size() == m.ptrs.size() && p.rows == g.rows &&
                        p.rows == m.rows && p.cols == g.cols && p.cols == m.cols,
                    "params, grads and momenta differ: ", str((int64_t)p.ptrs.size()), " of ", str(p.rows), " x ",
                    str(p.cols), ", ", str((int64_t)g.ptrs.size()), " of ", str(g.rows), " x ", str(g.cols), ", ",
                    str((int64_t)m.ptrs.size()), " of ", str(m.rows), " x ", str(m.cols));
  TORCH_CHECK_VALUE(p.dev == g.dev && p.dev == m.dev, "params are on ", p.dev, ", grads on ", g.dev, ", momenta on ",
                    m.dev);
  TORCH_CHECK_TYPE(m.dtype == MHC_F32, "momenta must be float32, got ", momenta[0].scalar_type());
  if (given(lr_tensor)) {
    TORCH_CHECK_VALUE(lr_tensor->numel() == 1 && lr_tensor->scalar_type() == at::kFloat && lr_tensor->device() == p.dev,
                      "lr must be a number or a one-element float32 tensor on ", p.dev);
    a.lr_device = lr_tensor->data_ptr<float>();
  }
  const at::Tensor ws = ortho_workspace(p, &a.workspace_bytes, &a.workspace);
  a.params = p.ptrs.data();
  a.grads = g.ptrs.data();
  a.momenta = reinterpret_cast<float* const*>(m.ptrs.data());
  a.count = (int64_t)p.ptrs.size();
  a.rows = (int32_t)p.rows;
  a.cols = (int32_t)p.cols;
  a.param_dtype = p.dtype;
  a.grad_dtype = g.dtype;
  a.nesterov = nesterov ? 1 : 0;
  a.coeffs = coeffs.data();
  a.eps = eps;
  a.momentum = momentum;
  a.weight_decay = (float)weight_decay;
  a.scale = (float)scale;
  a.lr = (float)lr;
  check_status(mhc_muon_step(&a, at::cuda::getCurrentCUDAStream().stream()), "mhc::muon_step_");
  mark_written(params);
  mark_written(momenta);
}

// ----------------------------------------------------------------- Meta kernels (shapes only)
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> mhc_fwd_meta(
    const at::Tensor& x, const at::Tensor& phi, const at::Tensor& alpha, const at::Tensor& bias, double, double) {
  TORCH_CHECK(x.dim() == 4, "x must be [B, S, n, D]");
  const auto B = x.sym_size(0), S = x.sym_size(1), n = x.sym_size(2), D = x.sym_size(3);
  const auto N = n * n + 2 * n;
  const auto f = x.options().dtype(at::kFloat);
  return {at::empty_symint({B, S, D}, x.options()), at::empty_symint({B, S, n}, f),
          at::empty_symint({B, S, n, n}, f), at::empty_symint({B, S}, f), at::empty_symint({B, S, N}, f),
          at::empty_symint({B, S, n}, f)};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> mhc_bwd_meta(
    const at::Tensor& x, const at::Tensor& phi, const at::Tensor&, const at::Tensor&, const at::Tensor&,
    const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
    const c10::optional<at::Tensor>&, double, double) {
  TORCH_CHECK(x.dim() == 4, "x must be [B, S, n, D]");
  const auto n = x.sym_size(2), D = x.sym_size(3);
  const auto N = n * n + 2 * n;
  const auto f = x.options().dtype(at::kFloat);
  return {at::empty_symint(x.sym_sizes(), x.options()), at::empty_symint({N, n * D}, f), at::empty_symint({3}, f),
          at::empty_symint({N}, f), at::empty_symint({n * D}, f)};
}

std::vector<at::Tensor> qk_norm_rope_meta(const at::Tensor& q, const at::Tensor& k, const OptTensor&,
                                          const at::Tensor&, const OptTensor&, const OptTensor&, const OptTensor& v,
                                          const OptTensor&, double, bool) {
  std::vector<at::Tensor> out{at::empty_symint(q.sym_sizes(), q.options()),
                              at::empty_symint(k.sym_sizes(), k.options())};
  if (given(v)) out.push_back(at::empty_symint(v->sym_sizes(), v->options()));
  return out;
}

std::vector<at::Tensor> qk_norm_rope_bwd_into_meta(const at::Tensor& q, const at::Tensor&, const OptTensor&,
                                                   const at::Tensor&, const at::Tensor&, const at::Tensor&,
                                                   const OptTensor& q_weight, const OptTensor& k_weight,
                                                   const OptTensor&, const OptTensor&, const OptTensor& row_scale,
                                                   double, bool, bool weight_grads, bool row_scale_grad,
                                                   at::TensorList) {
  std::vector<at::Tensor> out;
  const auto f = q.options().dtype(at::kFloat);
  if (given(q_weight) && weight_grads) out.push_back(at::empty_symint({q.sym_size(3)}, f));
  if (given(k_weight) && weight_grads) out.push_back(at::empty_symint({q.sym_size(3)}, f));
  if (given(row_scale) && row_scale_grad) out.push_back(at::empty_symint({q.sym_size(0), q.sym_size(1)}, f));
  return out;
}

std::vector<at::Tensor> qk_norm_rope_bwd_meta(const at::Tensor& q, const at::Tensor& k, const OptTensor& positions,
                                              const at::Tensor& inv_freq, const at::Tensor& dq_out,
                                              const at::Tensor& dk_out, const OptTensor& q_weight,
                                              const OptTensor& k_weight, const OptTensor& v, const OptTensor& dv_out,
                                              const OptTensor& row_scale, double eps, bool interleaved,
                                              bool weight_grads, bool row_scale_grad) {
  auto out = qk_norm_rope_meta(q, k, positions, inv_freq, q_weight, k_weight, v, row_scale, eps, interleaved);
  for (auto& t : qk_norm_rope_bwd_into_meta(q, k, positions, inv_freq, dq_out, dk_out, q_weight, k_weight, v, dv_out,
                                            row_scale, eps, interleaved, weight_grads, row_scale_grad, {}))
    out.push_back(std::move(t));
  return out;
}

std::vector<at::Tensor> orthogonalize_meta(at::TensorList g, at::ArrayRef<double>, double) {
  std::vector<at::Tensor> out;
  for (const at::Tensor& t : g) out.push_back(at::empty_symint(t.sym_sizes(), t.options()));
  return out;
}

void muon_step_meta(at::TensorList, at::TensorList, at::TensorList, const OptTensor&, double, double, bool, double,
                    double, at::ArrayRef<double>, double) {}

TORCH_LIBRARY(mhc, m) {
  m.def("fwd(Tensor x, Tensor phi, Tensor alpha, Tensor bias, float norm_eps=1e-6, float hc_eps=1e-6) -> "
        "(Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("bwd(Tensor x, Tensor phi, Tensor alpha, Tensor inv_rms, Tensor h_mix, Tensor h_pre, Tensor h_post, "
        "Tensor dh_in, Tensor dh_post, Tensor dh_res, Tensor? gamma, float norm_eps=1e-6, float hc_eps=1e-6) -> "
        "(Tensor, Tensor, Tensor, Tensor, Tensor)");
  // q [B,S,Hq,d], k [B,S,Hk,d], v [B,S,Hv,d] -> q_out, k_out (, v_out)
  m.def("qk_norm_rope(Tensor q, Tensor k, Tensor? positions, Tensor inv_freq, Tensor? q_weight, Tensor? k_weight, "
        "Tensor? v, Tensor? row_scale, float eps, bool interleaved) -> Tensor[]");
  // -> dq, dk (, dv) (, dq_weight) (, dk_weight) (, drow_scale): what is given and wanted
  m.def("qk_norm_rope_bwd(Tensor q, Tensor k, Tensor? positions, Tensor inv_freq, Tensor dq_out, Tensor dk_out, "
        "Tensor? q_weight, Tensor? k_weight, Tensor? v, Tensor? dv_out, Tensor? row_scale, float eps, "
        "bool interleaved, bool weight_grads, bool row_scale_grad) -> Tensor[]");
  // dq, dk (, dv) written into grad_out -> the rest
  m.def("qk_norm_rope_bwd_into(Tensor q, Tensor k, Tensor? positions, Tensor inv_freq, Tensor dq_out, Tensor dk_out, "
        "Tensor? q_weight, Tensor? k_weight, Tensor? v, Tensor? dv_out, Tensor? row_scale, float eps, "
        "bool interleaved, bool weight_grads, bool row_scale_grad, Tensor(a!)[] grad_out) -> Tensor[]");
  // equal matrices, or one stack of them; coeffs flat
  m.def("orthogonalize(Tensor[] g, float[] coeffs, float eps) -> Tensor[]");
  m.def("muon_step_(Tensor(a!)[] params, Tensor[] grads, Tensor(b!)[] momenta, Tensor? lr_tensor, float lr, "
        "float momentum, bool nesterov, float weight_decay, float scale, float[] coeffs, float eps) -> ()");
  m.def("check_status() -> int");
  m.impl("check_status", &mhc_check_status);
}

TORCH_LIBRARY_IMPL(mhc, CUDA, m) {
  m.impl("fwd", &mhc_fwd_cuda);
  m.impl("bwd", &mhc_bwd_cuda);
  m.impl("qk_norm_rope", &qk_norm_rope_cuda);
  m.impl("qk_norm_rope_bwd", &qk_norm_rope_bwd_cuda);
  m.impl("qk_norm_rope_bwd_into", &qk_norm_rope_bwd_into_cuda);
  m.impl("orthogonalize", &orthogonalize_cuda);
  m.impl("muon_step_", &muon_step_cuda);
}

TORCH_LIBRARY_IMPL(mhc, Meta, m) {
  m.impl("fwd", &mhc_fwd_meta);
  m.impl("bwd", &mhc_bwd_meta);
  m.impl("qk_norm_rope", &qk_norm_rope_meta);
  m.impl("qk_norm_rope_bwd", &qk_norm_rope_bwd_meta);
  m.impl("qk_norm_rope_bwd_into", &qk_norm_rope_bwd_into_meta);
  m.impl("orthogonalize", &orthogonalize_meta);
  m.impl("muon_step_", &muon_step_meta);
}

// No gradient goes through these.  The ones that return results refuse a backward
// pass through them, and forward-mode tangents, rather than drop them; the ones
// that write into given tensors (leaves that require a gradient among them) pass.
// (torch's boxed fallback does the same, for 1 us more of a 17 us call.)
namespace {

struct Inputs {   // what autograd has to know of a call's tensors
  torch::autograd::edge_list edges;
  const bool recording = at::GradMode::is_enabled();
  bool any = false;
  void add(const at::Tensor& t) {
    if (!t.defined()) return;
    TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), "the mhc operators do not support forward AD");
    any = any || (recording && t.requires_grad());
  }
  void add(const OptTensor& t) {
    if (given(t)) add(*t);
  }
  void add(at::TensorList l) {
    for (const at::Tensor& t : l) add(t);
  }
  template <class T>
  void add(const T&) {}
  void edge(const at::Tensor& t) {
    if (t.defined() && t.requires_grad()) edges.push_back(torch::autograd::impl::gradient_edge(t));
  }
  void edge(const OptTensor& t) {
    if (given(t)) edge(*t);
  }
  void edge(at::TensorList l) {
    for (const at::Tensor& t : l) edge(t);
  }
  template <class T>
  void edge(const T&) {}
};

template <class F, class... A>
std::vector<at::Tensor> without_gradient(const c10::TypedOperatorHandle<F>& op, const char* name, const A&... args) {
  Inputs in;
  (in.add(args), ...);
  std::vector<at::Tensor> out;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    out = op.call(args...);
  }
  if (in.any) {
    (in.edge(args), ...);
    const std::shared_ptr<torch::autograd::Node> node(
        new torch::autograd::NotImplemented(name, std::move(in.edges)), torch::autograd::deleteNode);
    for (at::Tensor& t : out) torch::autograd::impl::set_gradient_edge(t, {node, node->add_input_metadata(t)});
  }
  return out;
}

template <class F>
c10::TypedOperatorHandle<F> handle(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}

std::vector<at::Tensor> qk_norm_rope_autograd(const at::Tensor& q, const at::Tensor& k, const OptTensor& positions,
                                              const at::Tensor& inv_freq, const OptTensor& q_weight,
                                              const OptTensor& k_weight, const OptTensor& v, const OptTensor& row_scale,
                                              double eps, bool interleaved) {
  static const auto op = handle<decltype(qk_norm_rope_meta)>("mhc::qk_norm_rope");
  return without_gradient(op, "mhc::qk_norm_rope", q, k, positions, inv_freq, q_weight, k_weight, v, row_scale, eps,
                          interleaved);
}

std::vector<at::Tensor> qk_norm_rope_bwd_autograd(const at::Tensor& q, const at::Tensor& k, const OptTensor& positions,
                                                  const at::Tensor& inv_freq, const at::Tensor& dq_out,
                                                  const at::Tensor& dk_out, const OptTensor& q_weight,
                                                  const OptTensor& k_weight, const OptTensor& v, const OptTensor& dv_out,
                                                  const OptTensor& row_scale, double eps, bool interleaved,
                                                  bool weight_grads, bool row_scale_grad) {
  static const auto op = handle<decltype(qk_norm_rope_bwd_meta)>("mhc::qk_norm_rope_bwd");
  return without_gradient(op, "mhc::qk_norm_rope_bwd", q, k, positions, inv_freq, dq_out, dk_out, q_weight, k_weight, v,
                          dv_out, row_scale, eps, interleaved, weight_grads, row_scale_grad);
}

std::vector<at::Tensor> orthogonalize_autograd(at::TensorList g, at::ArrayRef<double> coeffs, double eps) {
  static const auto op = handle<decltype(orthogonalize_meta)>("mhc::orthogonalize");
  return without_gradient(op, "mhc::orthogonalize", g, coeffs, eps);
}

}  // namespace

TORCH_LIBRARY_IMPL(mhc, Autograd, m) {
  m.impl("qk_norm_rope", &qk_norm_rope_autograd);
  m.impl("qk_norm_rope_bwd", &qk_norm_rope_bwd_autograd);
  m.impl("orthogonalize", &orthogonalize_autograd);
  for (const char* op : {"qk_norm_rope_bwd_into", "muon_step_"}) m.impl(op, torch::CppFunction::makeFallthrough());
}
