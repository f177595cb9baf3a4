// Host path of the rotary positions and of the paged 8-bit cache: checks, outputs and scratch from torch's allocator, the calls of the C ABI, and the
// autograd node of the positions.  The *_raw functions take ordinary tensors and raise on what the kernels do not take; they are also what the
// custom ops of a traced graph run.  The others return None where a call is not plain eager work (tracing, fake or wrapped tensors,
// dispatch modes), and the caller takes the custom op.
#include "torch_host.h"

#include <c10/hip/HIPGraphsC10Utils.h>
#include <torch/csrc/autograd/variable.h>

#include <cmath>
#include <optional>
#include <string>
#include <vector>

namespace {

using namespace fmoba_host;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void require(bool ok, const char *what) {
  if (!ok) throw std::runtime_error(what);
}
void *current_stream(const Tensor &t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
py::object none() { return py::none(); }
py::object wrap(const Tensor &t) { return py::reinterpret_steal<py::object>(THPVariable_Wrap(t)); }

// as the kernels read rows: dense features, 16-byte vectors (a dense tensor may still begin off them: a copy all the same)
Tensor as_rows(const Tensor &t) { return is_rows(t, t.scalar_type(), t.device()) ? t : t.clone(at::MemoryFormat::Contiguous); }

// ---------------------------------------------------------------------------------------------------------------- positions
struct RotaryForm {
  std::vector<int64_t> sections;
  double base;
  int64_t rotary_dim;
  bool interleaved, inverse;
};

void check_rotary(const Tensor &q, const Tensor &k, const Tensor &positions, const RotaryForm &f) {
  const at::ScalarType dt = q.scalar_type();
  require(dt == at::kHalf || dt == at::kBFloat16, "FlashMoBA only supports fp16 and bf16 data types");
  require(q.is_cuda() && k.device() == q.device() && positions.device() == q.device(), "q, k and positions must be on one GPU");
  require(k.scalar_type() == dt, "q and k must have the same dtype");
  require(q.dim() == 3 && k.dim() == 3 && k.size(0) == q.size(0) && k.size(2) == q.size(2), "q and k must be (tokens, heads, head_size) of the same tokens and head size");
  require(positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong, "positions must be int32 or int64");
  require(positions.dim() == 2 && positions.size(1) == q.size(0), "positions must have shape (axes, tokens)");
  require(positions.size(0) >= 1 && positions.size(0) <= FMOBA_ROTARY_AXES && positions.size(0) == static_cast<int64_t>(f.sections.size()), "positions must have 1 to 4 axes, as many as sections");
  require(f.base >= 1.0 && std::isfinite(f.base), "base must be a finite number from 1 on");
  require(q.size(1) >= 1 && q.size(1) <= 65535 && k.size(1) >= 1 && k.size(1) <= 65535, "q and k must have 1 to 65535 heads");
  require(q.size(2) >= 8 && q.size(2) <= 256 && q.size(2) % 8 == 0, "head_size must be a multiple of 8 up to 256");
  require(f.rotary_dim >= 8 && f.rotary_dim <= q.size(2) && f.rotary_dim % 8 == 0, "rotary_dim must be a multiple of 8 up to the head size");
  int64_t pairs = 0;
  for (int64_t n : f.sections) {
    require(n >= 0 && n <= f.rotary_dim, "a section is a number of pairs");
    pairs += n;
  }
  require(pairs == f.rotary_dim / 2, "the sections must have rotary_dim / 2 pairs together");
}

// q and k, or only one of them (the other undefined): what is given comes back turned
std::pair<Tensor, Tensor> turn(Tensor q, Tensor k, const Tensor &positions, const RotaryForm &f) {
  const Tensor &x = q.defined() ? q : k;
  const c10::DeviceGuard guard(x.device());
  check_device(x.device().index());
  fmoba_rotary_args a{};
  Tensor qo, ko, pos = positions.size(1) > 1 && positions.stride(1) != 1 ? positions.contiguous() : positions;
  if (q.defined()) {
    q = as_rows(q);
    qo = at::empty(q.sizes(), q.options());
    a.q = q.data_ptr(), a.q_out = qo.data_ptr(), a.heads = q.size(1);
    a.q_row_stride = q.stride(0), a.q_head_stride = q.stride(1), a.qo_row_stride = qo.stride(0), a.qo_head_stride = qo.stride(1);
  }
  if (k.defined()) {
    k = as_rows(k);
    ko = at::empty(k.sizes(), k.options());
    a.k = k.data_ptr(), a.k_out = ko.data_ptr(), a.heads_k = k.size(1);
    a.k_row_stride = k.stride(0), a.k_head_stride = k.stride(1), a.ko_row_stride = ko.stride(0), a.ko_head_stride = ko.stride(1);
  }
  a.positions = pos.data_ptr(), a.positions_64 = pos.scalar_type() == at::kLong, a.pos_axis_stride = pos.stride(0);
  a.log2_base = std::log2(f.base), a.total = x.size(0), a.head_dim = x.size(2), a.rotary_dim = f.rotary_dim;
  a.axes = f.sections.size();
  for (int i = 0; i < a.axes; ++i) a.sections[i] = f.sections[i];
  a.interleaved = f.interleaved, a.inverse = f.inverse, a.dtype = x.scalar_type() == at::kBFloat16 ? FMOBA_DTYPE_BF16 : FMOBA_DTYPE_F16;
  check(fmoba_rotary(&a, current_stream(x)));
  return {qo, ko};
}

// The turn is linear, its gradient the turn back: the backward of a backward is the node itself again.
struct Rotary : public torch::autograd::Function<Rotary> {
  static variable_list forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &positions, const RotaryForm &f) {
    ctx->save_for_backward({positions});
    ctx->saved_data["sections"] = f.sections;
    ctx->saved_data["base"] = f.base;
    ctx->saved_data["rotary_dim"] = f.rotary_dim;
    ctx->saved_data["interleaved"] = f.interleaved;
    ctx->saved_data["inverse"] = f.inverse;
    ctx->saved_data["tokens"] = q.size(0);
    at::AutoDispatchBelowADInplaceOrView below;
    auto r = turn(q, k, positions, f);
    return {r.first, r.second};
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const Tensor positions = ctx->get_saved_variables()[0];
    const RotaryForm f{ctx->saved_data["sections"].toIntVector(), ctx->saved_data["base"].toDouble(), ctx->saved_data["rotary_dim"].toInt(),
                       ctx->saved_data["interleaved"].toBool(), !ctx->saved_data["inverse"].toBool()};
    // (what was saved may have been through saved-tensor hooks, and its address goes to a kernel)
    check_rotary(grads[0], grads[1], positions, f);
    require(positions.size(1) == ctx->saved_data["tokens"].toInt(), "flash_moba: the positions were saved and came back in another shape");
    if (at::GradMode::is_enabled()) {
      variable_list r = Rotary::apply(grads[0], grads[1], positions, f);
      return {r[0], r[1], Tensor(), Tensor()};
    }
    at::AutoDispatchBelowADInplaceOrView below;
    auto r = turn(ctx->needs_input_grad(0) ? grads[0] : Tensor(), ctx->needs_input_grad(1) ? grads[1] : Tensor(), positions, f);
    return {r.first, r.second, Tensor(), Tensor()};
  }
};

// A leaf keeps one node that takes its gradient, for as long as any graph has it, and with it the stream that was current when the first of these graphs
// was made.  The engine makes that stream wait for the one that the gradient comes from: where the latter is being captured into a HIP graph,
// the former is drawn into the capture, which then cannot end (the process does, with a segmentation fault).
void refuse_leaf_of_another_stream(const Tensor &t) {
  if (!t.requires_grad() || !t.is_leaf() || c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  const auto node = torch::autograd::impl::try_get_grad_accumulator(t);
  if (node == nullptr) return;
  const auto stream = node->stream();
  require(!stream.has_value() || *stream == c10::hip::getCurrentHIPStream(t.device().index()).unwrap(),
          "flash_moba: an input is a leaf of a graph that was made on another stream and is still alive: its backward cannot be captured");
}

RotaryForm rotary_form(std::vector<int64_t> sections, double base, int64_t rotary_dim, bool interleaved, bool inverse) {
  return RotaryForm{std::move(sections), base, rotary_dim, interleaved, inverse};
}

py::object rotary(const py::handle &hq, const py::handle &hk, const py::handle &hp, std::vector<int64_t> sections, double base, int64_t rotary_dim, bool interleaved) {
  if (!eager() || !plain(hq) || !plain(hk) || !plain(hp)) return none();
  const Tensor &q = THPVariable_Unpack(hq.ptr()), &k = THPVariable_Unpack(hk.ptr()), &positions = THPVariable_Unpack(hp.ptr());
  const RotaryForm f = rotary_form(std::move(sections), base, rotary_dim, interleaved, false);
  check_rotary(q, k, positions, f);
  Tensor qo, ko;
  {
    py::gil_scoped_release nogil;
    if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad())) {
      const c10::DeviceGuard guard(q.device());
      refuse_leaf_of_another_stream(q);
      refuse_leaf_of_another_stream(k);
      variable_list r = Rotary::apply(q, k, positions, f);
      qo = r[0], ko = r[1];
    } else {
      at::AutoDispatchBelowADInplaceOrView below;
      std::tie(qo, ko) = turn(q, k, positions, f);
    }
  }
  return py::make_tuple(wrap(qo), wrap(ko));
}

std::pair<Tensor, Tensor> rotary_raw(const Tensor &q, const Tensor &k, const Tensor &positions, std::vector<int64_t> sections, double base, int64_t rotary_dim, bool interleaved, bool inverse) {
  const RotaryForm f = rotary_form(std::move(sections), base, rotary_dim, interleaved, inverse);
  check_rotary(q, k, positions, f);
  py::gil_scoped_release nogil;
  at::AutoDispatchBelowADInplaceOrView below;
  return turn(q, k, positions, f);
}

}  // namespace

void fmoba_host::bind_cache_ops(py::module_ &m) {
  m.def("rotary", &rotary);
  m.def("rotary_raw", &rotary_raw);
}
