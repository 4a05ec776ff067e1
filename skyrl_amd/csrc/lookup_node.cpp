// The autograd node of an embedding lookup, as a Python extension.
//
// Autograd runs a node on a thread of its own, and a node that is Python makes each object of the interpreter that it touches travel to that thread's core.  A
// pass of 611 rows and the gradient of a table of 32001 x 1023 took 45 us with a node in Python where the processor woke the thread beside its caller and 105 to
// 115 where it did not; 33 and 58 with this one (the kernels are 31; torch's own embedding takes 62, without autograd on one thread 34 either way).
// Everything is checked by embedding_lookup (skyrl_amd/embedding.py) before it calls; the library's functions come in by address.
#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/profiler/api.h>
#include <torch/csrc/utils/pybind.h>

#include "../../include/skyrl_lmhead.h"

namespace {

struct Library {
  decltype(&skyrl_lmhead_embedding_fwd) fwd = nullptr;
  decltype(&skyrl_lmhead_embedding_bwd) bwd = nullptr;
  decltype(&skyrl_lmhead_embedding_bwd_workspace_bytes) workspace_bytes = nullptr;
  decltype(&skyrl_lmhead_strerror) strerror = nullptr;
} lib;

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

int type_of(const at::Tensor& t) { return t.scalar_type() == at::kFloat ? SKYRL_LOGITS_F32 : SKYRL_LOGITS_BF16; }

void* stream_of(const at::Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

void check(int status, const char* what) {
  TORCH_CHECK_VALUE(status >= 0, what, " failed with status ", status, ": ", lib.strerror(status));
  TORCH_CHECK(status == 0, what, " failed with status ", status, ": ", lib.strerror(status));
}

// Whether the gradient may be computed here: real memory that is its value, and nobody who follows the ops of this call or records them.  Everything else goes
// to the op, whose dispatcher layers know what to do with it, or that a second derivative must raise.
bool plain(const at::Tensor& d) {
  constexpr c10::DispatchKeySet others({c10::DispatchKey::Python, c10::DispatchKey::Negative, c10::DispatchKey::Conjugate, c10::DispatchKey::ZeroTensor,
                                        c10::DispatchKey::Functionalize, c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper});
  return d.is_cuda() && !d.key_set().has_any(others) && !(at::GradMode::is_enabled() && d.requires_grad()) && !c10::impl::dispatch_mode_enabled() &&
         !at::tracer::impl::is_dispatch_enabled() && !torch::profiler::impl::profilerEnabled();
}

at::Tensor by_the_op(const at::Tensor& d, const at::Tensor& ids, int64_t vocab, double scale, int64_t padding) {
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("skyrl_amd::lmhead_embedding_bwd", "")
                             .typed<at::Tensor(const at::Tensor&, const at::Tensor&, c10::SymInt, double, c10::SymInt)>();
  return op.call(d, ids, vocab, scale, padding);
}

struct Lookup : public torch::autograd::Function<Lookup> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& weight, const at::Tensor& ids, double scale, int64_t padding) {
    const int64_t T = ids.size(0), V = weight.size(0), H = weight.size(1);
    ctx->save_for_backward({ids});
    ctx->saved_data["vocab"] = V;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    at::Tensor out = at::empty({T, H}, weight.options());
    if (T == 0 || H == 0) return out;
    if (V == 0) return out.zero_();  // every id lies outside
    const c10::DeviceGuard guard(weight.device());
    check(lib.fwd(weight.data_ptr(), type_of(weight), V > 1 ? weight.stride(0) : H, (const int64_t*)ids.data_ptr(), T, H, V, (float)scale, out.data_ptr(), stream_of(weight)),
          "skyrl_lmhead_embedding_fwd");
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const at::Tensor ids = ctx->get_saved_variables()[0];
    const int64_t V = ctx->saved_data["vocab"].toInt(), padding = ctx->saved_data["padding"].toInt();
    const double scale = ctx->saved_data["scale"].toDouble();
    at::Tensor d = grads[0];
    const int64_t T = d.size(0), H = d.size(1);
    if (!((d.stride(1) == 1 || H <= 1) && (d.stride(0) >= H || d.stride(0) == 0 || T <= 1))) d = d.contiguous();
    at::Tensor d_weight;
    if (!plain(d)) {
      d_weight = by_the_op(d, ids, V, scale, padding);
    } else if (d.numel() == 0 || V == 0) {
      d_weight = at::zeros({V, H}, d.options());
    } else {
      const c10::DeviceGuard guard(d.device());
      const size_t bytes = lib.workspace_bytes(T, H, V);
      TORCH_CHECK_VALUE(bytes > 0, "no workspace for T=", T, ", H=", H, ", V=", V, ": an extent is out of range");
      d_weight = at::empty({V, H}, d.options());
      const at::Tensor workspace = at::empty({(int64_t)bytes}, d.options().dtype(at::kByte));
      check(lib.bwd(d.data_ptr(), type_of(d), T > 1 ? d.stride(0) : H, (const int64_t*)ids.data_ptr(), padding, T, H, V, (float)scale, 0, d_weight.data_ptr(),
                    workspace.data_ptr(), bytes, stream_of(d)),
            "skyrl_lmhead_embedding_bwd");
    }
    return {d_weight, at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

}  // namespace

PYBIND11_MODULE(lookup_node, m) {
  m.def("bind", [](uintptr_t fwd, uintptr_t bwd, uintptr_t workspace_bytes, uintptr_t strerror) {
    lib.fwd = (decltype(lib.fwd))fwd;
    lib.bwd = (decltype(lib.bwd))bwd;
    lib.workspace_bytes = (decltype(lib.workspace_bytes))workspace_bytes;
    lib.strerror = (decltype(lib.strerror))strerror;
  });
  m.def("lookup", [](const at::Tensor& weight, const at::Tensor& ids, double scale, int64_t padding) { return Lookup::apply(weight, ids, scale, padding); });
}
