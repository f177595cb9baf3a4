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

// the positions of x's tokens and how they turn; pos: a tensor that keeps them alive
fmoba_rotary_args rotary_args(const Tensor &x, const Tensor &positions, const RotaryForm &f, Tensor &pos) {
  fmoba_rotary_args a{};
  pos = positions.size(1) > 1 && positions.stride(1) != 1 ? positions.contiguous() : positions;
  a.positions = pos.data_ptr(), a.positions_64 = pos.scalar_type() == at::kLong, a.pos_axis_stride = pos.stride(0);
  a.log2_base = std::log2(f.base), a.total = x.size(0), a.head_dim = x.size(2), a.rotary_dim = f.rotary_dim;
  a.axes = f.sections.size();
  for (int i = 0; i < a.axes; ++i) a.sections[i] = f.sections[i];
  a.interleaved = f.interleaved, a.inverse = f.inverse, a.dtype = x.scalar_type() == at::kBFloat16 ? FMOBA_DTYPE_BF16 : FMOBA_DTYPE_F16;
  return a;
}
// dense queries and the place of the turned ones
Tensor rotary_queries(fmoba_rotary_args &a, Tensor &q) {
  q = as_rows(q);
  const Tensor qo = at::empty(q.sizes(), q.options());
  a.q = q.data_ptr(), a.q_out = qo.data_ptr(), a.heads = q.size(1);
  a.q_row_stride = q.stride(0), a.q_head_stride = q.stride(1), a.qo_row_stride = qo.stride(0), a.qo_head_stride = qo.stride(1);
  return qo;
}

// q and k, or only one of them (the other undefined): what is given comes back turned
std::pair<Tensor, Tensor> turn(Tensor q, Tensor k, const Tensor &positions, const RotaryForm &f) {
  const Tensor &x = q.defined() ? q : k;
  const c10::DeviceGuard guard(x.device());
  check_device(x.device().index());
  Tensor qo, ko, pos;
  fmoba_rotary_args a = rotary_args(x, positions, f, pos);
  if (q.defined()) qo = rotary_queries(a, q);
  if (k.defined()) {
    k = as_rows(k);
    ko = at::empty(k.sizes(), k.options());
    a.k = k.data_ptr(), a.k_out = ko.data_ptr(), a.heads_k = k.size(1);
    a.k_row_stride = k.stride(0), a.k_head_stride = k.stride(1), a.ko_row_stride = ko.stride(0), a.ko_head_stride = ko.stride(1);
  }
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

// -------------------------------------------------------------------------------------------------------------------- cache
// The tensors of a cache in the order of MobaKVCache; weight may be undefined.
struct Cache {
  Tensor k, v, k_scale, v_scale, k_sum, k_mean, weight;
};
constexpr int kCacheTensors = 7;

bool dense(const Tensor &t, at::ScalarType type, const at::Device &dev) { return t.defined() && t.scalar_type() == type && t.device() == dev && t.is_contiguous(); }

fmoba_kv_cache cache_view(const Cache &c) {
  const Tensor &k = c.k, &v = c.v;
  require(k.is_cuda(), "the cache must be on a GPU");
  const at::Device dev = k.device();
  require(k.dim() == 4 && v.dim() == 4 && v.sizes() == k.sizes() && v.device() == dev, "k and v of a cache must be (pages, heads, page_size, head_size) tensors of one shape on one GPU");
  require(k.scalar_type() == v.scalar_type() && (k.scalar_type() == at::kFloat8_e4m3fn || k.scalar_type() == at::kChar), "k and v of a cache must be float8_e4m3fn or int8");
  require(k.size(3) == 1 || (k.stride(3) == 1 && v.stride(3) == 1), "k and v of a cache must be contiguous on the last dim");
  const int64_t pages = k.size(0), heads = k.size(1);
  require(pages <= INT32_MAX && heads >= 1 && heads <= 65535 && k.size(2) <= 1024 && k.size(3) <= 256, "cache: too many pages or heads, or page_size above 1024 or head_size above 256");
  auto per_head = [&](const Tensor &t, at::ScalarType type, int64_t more) {
    return dense(t, type, dev) && t.dim() == (more ? 3 : 2) && t.size(0) == pages && t.size(1) == heads && (more == 0 || t.size(2) == more);
  };
  require(per_head(c.k_scale, at::kFloat, 0) && per_head(c.v_scale, at::kFloat, 0), "k_scale and v_scale of a cache must be dense fp32 (pages, heads)");
  require(per_head(c.k_sum, at::kFloat, k.size(3)), "k_sum of a cache must be dense fp32 (pages, heads, head_size)");
  const at::ScalarType dt = c.k_mean.defined() ? c.k_mean.scalar_type() : at::kFloat;
  require(dt == at::kHalf || dt == at::kBFloat16, "FlashMoBA only supports fp16 and bf16 data types");
  require(per_head(c.k_mean, dt, k.size(3)), "k_mean of a cache must be dense (pages, heads, head_size)");
  require(!c.weight.defined() || per_head(c.weight, at::kLong, 0), "weight of a cache must be dense int64 (pages, heads)");
  for (const Tensor *t : {&c.k, &c.v, &c.k_scale, &c.v_scale, &c.k_sum, &c.k_mean}) require(!t->requires_grad(), "the cache has no gradients");
  fmoba_kv_cache a{};
  a.k = k.data_ptr(), a.v = v.data_ptr(), a.k_scale = c.k_scale.data_ptr<float>(), a.v_scale = c.v_scale.data_ptr<float>(), a.k_sum = c.k_sum.data_ptr<float>();
  a.k_mean = c.k_mean.data_ptr(), a.weight = c.weight.defined() ? c.weight.data_ptr<int64_t>() : nullptr;
  a.k_page_stride = k.stride(0), a.k_head_stride = k.stride(1), a.k_token_stride = k.stride(2);
  a.v_page_stride = v.stride(0), a.v_head_stride = v.stride(1), a.v_token_stride = v.stride(2);
  a.num_pages = pages, a.page_size = k.size(2), a.heads_k = heads, a.head_dim = k.size(3);
  a.format = k.scalar_type() == at::kChar ? FMOBA_CACHE_INT8 : FMOBA_CACHE_E4M3, a.dtype = dt == at::kBFloat16 ? FMOBA_DTYPE_BF16 : FMOBA_DTYPE_F16;
  return a;
}

// lengths and tables of a call's sequences; returns how many there are
int64_t check_sequences(const Tensor &cu, const Tensor &seqlens_k, const Tensor &table, const at::Device &dev) {
  require(seqlens_k.dim() == 1 && dense(seqlens_k, at::kInt, dev) && seqlens_k.size(0) >= 1 && seqlens_k.size(0) <= 65535, "seqlens_k must be dense int32 (batch) on the cache's GPU, batch up to 65535");
  const int64_t batch = seqlens_k.size(0);
  require(!cu.defined() || is_cu(cu, batch + 1, dev), "cu_seqlens must be dense int32 (batch + 1) on the cache's GPU");
  require(table.dim() == 2 && table.scalar_type() == at::kInt && table.device() == dev && table.size(0) == batch && (table.size(1) <= 1 || table.stride(1) == 1) && table.size(1) <= INT32_MAX,
          "block_table must be int32 (batch, pages of a sequence) on the cache's GPU, its rows dense");
  return batch;
}

void check_inference(std::initializer_list<const Tensor *> ts) {
  for (const Tensor *t : ts)
    require(!(at::GradMode::is_enabled() && t->requires_grad()), "the cache functions have no backward pass: call them under torch.no_grad(), or with detached tensors");
}

// turn: the queries and positions, if the keys are to be turned first
void append_raw(const Cache &c, const Tensor &k_in, const Tensor &v_in, const Tensor &cu, int64_t max_seqlen, const Tensor &seqlens_k, const Tensor &table, fmoba_rotary_args *turn = nullptr) {
  fmoba_cache_append_args a{};
  a.cache = cache_view(c);
  const at::Device dev = c.k.device();
  const at::ScalarType dt = c.k_mean.scalar_type();
  check_inference({&k_in, &v_in});
  require(k_in.dim() == 3 && v_in.sizes() == k_in.sizes() && k_in.scalar_type() == dt && v_in.scalar_type() == dt && k_in.device() == dev && v_in.device() == dev,
          "k and v must be (tokens, heads, head_size) of the cache's k_mean dtype on its GPU");
  require(k_in.size(1) == c.k.size(1) && k_in.size(2) == c.k.size(3), "heads and head size of k and v must be the cache's");
  require(k_in.size(0) <= INT32_MAX && max_seqlen >= 0 && max_seqlen <= INT32_MAX, "max_seqlen or the number of tokens is out of range");
  a.batch = check_sequences(cu, seqlens_k, table, dev);
  require(cu.defined(), "cu_seqlens must be given");
  const Tensor k = as_rows(k_in), v = as_rows(v_in);
  a.k = k.data_ptr(), a.v = v.data_ptr(), a.cu_seqlens = cu.data_ptr<int32_t>(), a.seqlens_k = seqlens_k.data_ptr<int32_t>(), a.block_table = table.data_ptr<int32_t>();
  a.k_row_stride = k.stride(0), a.k_head_stride = k.stride(1), a.v_row_stride = v.stride(0), a.v_head_stride = v.stride(1), a.table_stride = table.stride(0);
  a.total_new = k.size(0), a.max_seqlen_new = max_seqlen, a.max_pages = table.size(1);
  const c10::DeviceGuard guard(dev);
  check_device(dev.index());
  if (turn) {
    turn->k = a.k, turn->heads_k = k.size(1), turn->k_row_stride = a.k_row_stride, turn->k_head_stride = a.k_head_stride;
    check(fmoba_cache_append_turned(&a, turn, current_stream(c.k)));
  } else {
    check(fmoba_cache_append(&a, current_stream(c.k)));
  }
}

struct AttnForm {
  int64_t max_q, max_k, topk;
  std::optional<double> scale;
  bool add_weight;
};

void check_attn(const Tensor &q, const Cache &c, const AttnForm &f) {
  check_inference({&q});
  require(q.dim() == 3 && q.scalar_type() == c.k_mean.scalar_type() && q.device() == c.k.device(), "q must be (tokens, heads, head_size) of the cache's k_mean dtype on its GPU");
  require(q.size(2) == c.k.size(3), "the head size of q must be the cache's");
  require(q.size(1) >= 1 && q.size(1) % c.k.size(1) == 0, "#heads in key/value must divide #heads in query");
  require(q.size(0) <= INT32_MAX && q.size(1) <= 65535 && q.size(0) * q.size(1) <= INT32_MAX && f.max_q >= 0 && f.max_q <= INT32_MAX && f.max_k >= 0 && f.max_k <= INT32_MAX,
          "max_seqlen or the number of rows is out of range");
  require(f.topk >= 1 && f.topk <= 64, "moba_topk must be in [1, 64]");
  require(!f.add_weight || c.weight.defined(), "the cache keeps no weight");
}

// A call that has passed every check, with all that it needs: nothing is refused any more when it is launched.
struct AttnCall {
  fmoba_cache_attn_args a{};
  Tensor q, out, lse, ws;
};
AttnCall attn_call(const Tensor &q_in, const Cache &c, const Tensor &cu, const Tensor &seqlens_k, const Tensor &table, const AttnForm &f) {
  AttnCall call;
  fmoba_cache_attn_args &a = call.a;
  a.cache = cache_view(c);
  const at::Device dev = c.k.device();
  check_attn(q_in, c, f);
  a.batch = check_sequences(cu, seqlens_k, table, dev);
  require(cu.defined(), "cu_seqlens must be given");
  const c10::DeviceGuard guard(dev);
  check_device(dev.index());
  const Tensor q = call.q = as_rows(q_in);
  const Tensor out = call.out = at::empty(q.sizes(), q.options());
  call.lse = at::empty({q.size(1), q.size(0)}, q.options().dtype(at::kFloat));
  a.q = q.data_ptr(), a.out = out.data_ptr(), a.softmax_lse = call.lse.data_ptr<float>();
  a.cu_seqlens_q = cu.data_ptr<int32_t>(), a.seqlens_k = seqlens_k.data_ptr<int32_t>(), a.block_table = table.data_ptr<int32_t>();
  a.q_row_stride = q.stride(0), a.q_head_stride = q.stride(1), a.o_row_stride = out.stride(0), a.o_head_stride = out.stride(1), a.table_stride = table.stride(0);
  a.total_q = q.size(0), a.heads = q.size(1), a.max_seqlen_q = f.max_q, a.max_seqlen_k = f.max_k, a.max_pages = table.size(1), a.topk = f.topk, a.add_weight = f.add_weight;
  a.softmax_scale = static_cast<float>(f.scale ? *f.scale : std::pow(static_cast<double>(q.size(2)), -0.5));
  a.workspace_bytes = fmoba_cache_attn_workspace_bytes(&a);
  call.ws = bytes_like(q, a.workspace_bytes + 255);
  a.workspace = reinterpret_cast<void *>(up256(reinterpret_cast<size_t>(call.ws.data_ptr())));
  check(fmoba_cache_attn_check(&a));
  return call;
}
std::pair<Tensor, Tensor> launch(const AttnCall &call) {
  const c10::DeviceGuard guard(call.q.device());
  check(fmoba_cache_attn(&call.a, current_stream(call.q)));
  return {call.out, call.lse};
}
std::pair<Tensor, Tensor> attn_raw(const Tensor &q, const Cache &c, const Tensor &cu, const Tensor &seqlens_k, const Tensor &table, const AttnForm &f) {
  return launch(attn_call(q, c, cu, seqlens_k, table, f));
}

std::vector<Tensor> evict_raw(const Tensor &weight, const Tensor &seqlens_k, const Tensor &table, int64_t page_size, int64_t keep, int64_t sink, int64_t recent) {
  require(weight.is_cuda() && weight.dim() == 2 && weight.scalar_type() == at::kLong && weight.is_contiguous() && weight.size(0) <= INT32_MAX && weight.size(1) >= 1 && weight.size(1) <= 65535,
          "weight must be dense int64 (pages, heads) on a GPU");
  for (int64_t x : {page_size, keep, sink, recent}) require(x >= INT32_MIN && x <= INT32_MAX, "page_size and numbers of pages must be below 2^31");
  fmoba_cache_evict_args a{};
  a.batch = check_sequences(Tensor(), seqlens_k, table, weight.device());
  const c10::DeviceGuard guard(weight.device());
  check_device(weight.device().index());
  const Tensor new_table = at::empty(table.sizes(), table.options()), freed = at::empty(table.sizes(), table.options());
  const Tensor new_seqlens = at::empty(seqlens_k.sizes(), seqlens_k.options()), num_freed = at::empty(seqlens_k.sizes(), seqlens_k.options());
  a.weight = weight.data_ptr<int64_t>(), a.seqlens_k = seqlens_k.data_ptr<int32_t>(), a.block_table = table.data_ptr<int32_t>();
  a.new_table = new_table.data_ptr<int32_t>(), a.new_seqlens = new_seqlens.data_ptr<int32_t>(), a.freed = freed.data_ptr<int32_t>(), a.num_freed = num_freed.data_ptr<int32_t>();
  a.table_stride = table.stride(0), a.max_pages = table.size(1), a.num_pages = weight.size(0), a.heads_k = weight.size(1);
  a.page_size = page_size, a.keep = keep, a.sink = sink, a.recent = recent;
  a.workspace_bytes = fmoba_cache_evict_workspace_bytes(a.batch, a.max_pages);
  Tensor ws;
  if (a.workspace_bytes) ws = bytes_like(weight, a.workspace_bytes), a.workspace = ws.data_ptr();
  check(fmoba_cache_evict(&a, current_stream(weight)));
  return {new_table, new_seqlens, freed, num_freed};
}

// a tuple of a cache's tensors (the last may be None) as C++ ones; false if one is not an ordinary tensor
bool plain_cache(const py::handle &h, Cache &c) {
  if (!PyTuple_Check(h.ptr()) || PyTuple_GET_SIZE(h.ptr()) != kCacheTensors) throw std::runtime_error("cache must be a MobaKVCache");
  Tensor *to[kCacheTensors] = {&c.k, &c.v, &c.k_scale, &c.v_scale, &c.k_sum, &c.k_mean, &c.weight};
  for (int i = 0; i < kCacheTensors; ++i) {
    PyObject *o = PyTuple_GET_ITEM(h.ptr(), i);
    if (i == kCacheTensors - 1 && o == Py_None) continue;
    if (!plain(o)) return false;
    *to[i] = THPVariable_Unpack(o);
  }
  return true;
}

bool all_plain(std::initializer_list<py::handle> hs) {
  for (const py::handle &h : hs)
    if (!plain(h)) return false;
  return true;
}
const Tensor &unpack(const py::handle &h) { return THPVariable_Unpack(h.ptr()); }

bool cache_append(const py::handle &hc, const py::handle &hk, const py::handle &hv, const py::handle &hcu, int64_t max_seqlen, const py::handle &hlen, const py::handle &htable) {
  Cache c;
  if (!eager() || !plain_cache(hc, c) || !all_plain({hk, hv, hcu, hlen, htable})) return false;
  py::gil_scoped_release nogil;
  at::AutoDispatchBelowADInplaceOrView below;
  append_raw(c, unpack(hk), unpack(hv), unpack(hcu), max_seqlen, unpack(hlen), unpack(htable));
  return true;
}

py::object cache_evict(const py::handle &hw, const py::handle &hlen, const py::handle &htable, int64_t page_size, int64_t keep, int64_t sink, int64_t recent) {
  if (!eager() || !all_plain({hw, hlen, htable})) return none();
  std::vector<Tensor> r;
  {
    py::gil_scoped_release nogil;
    at::AutoDispatchBelowADInplaceOrView below;
    r = evict_raw(unpack(hw), unpack(hlen), unpack(htable), page_size, keep, sink, recent);
  }
  return py::make_tuple(wrap(r[0]), wrap(r[1]), wrap(r[2]), wrap(r[3]));
}

py::object cache_attn(const py::handle &hq, const py::handle &hc, const py::handle &hcu, int64_t max_q, const py::handle &hlen, int64_t max_k, const py::handle &htable, int64_t topk,
                      std::optional<double> scale, bool add_weight) {
  Cache c;
  if (!eager() || !plain_cache(hc, c) || !all_plain({hq, hcu, hlen, htable})) return none();
  std::pair<Tensor, Tensor> r;
  {
    py::gil_scoped_release nogil;
    at::AutoDispatchBelowADInplaceOrView below;
    r = attn_raw(unpack(hq), c, unpack(hcu), unpack(hlen), unpack(htable), AttnForm{max_q, max_k, topk, scale, add_weight});
  }
  return py::make_tuple(wrap(r.first), wrap(r.second));
}

// positions (if there are any), the new keys and values into the cache, attention: one call
py::object cache_step(const py::handle &hq, const py::handle &hk, const py::handle &hv, const py::handle &hc, const py::handle &hcu, int64_t max_q, const py::handle &hlen, int64_t max_k,
                      const py::handle &htable, int64_t topk, const py::handle &hp, std::vector<int64_t> sections, double base, int64_t rotary_dim, bool interleaved, std::optional<double> scale,
                      bool add_weight) {
  Cache c;
  const bool turned = !hp.is_none();
  if (!eager() || !plain_cache(hc, c) || !all_plain({hq, hk, hv, hcu, hlen, htable}) || (turned && !plain(hp))) return none();
  const RotaryForm f = rotary_form(std::move(sections), base, rotary_dim, interleaved, false);
  std::pair<Tensor, Tensor> r;
  {
    py::gil_scoped_release nogil;
    at::AutoDispatchBelowADInplaceOrView below;
    Tensor q = unpack(hq), k = unpack(hk), q_rows;
    const AttnForm attn{max_q, max_k, topk, scale, add_weight};
    cache_view(c);
    check_attn(q, c, attn);
    require(k.dim() == 3 && k.size(0) == q.size(0), "q, k and v must be of the same tokens");
    check_inference({&k});
    if (turned) check_rotary(q, k, unpack(hp), f);
    // (the attention is checked, and has its memory, before the cache changes: a step that is refused can be made again)
    const bool in_append = turned && max_q <= FMOBA_TURN_ROWS;
    Tensor pos;
    fmoba_rotary_args a{};
    if (in_append) {
      a = rotary_args(q, unpack(hp), f, pos);
      q_rows = q, q = rotary_queries(a, q_rows);
    } else if (turned) {
      std::tie(q, k) = turn(q, k, unpack(hp), f);
    }
    const AttnCall call = attn_call(q, c, unpack(hcu), unpack(hlen), unpack(htable), attn);
    append_raw(c, k, unpack(hv), unpack(hcu), max_q, unpack(hlen), unpack(htable), in_append ? &a : nullptr);
    r = launch(call);
  }
  return py::make_tuple(wrap(r.first), wrap(r.second));
}

// the same for the custom ops
using Optional = std::optional<Tensor>;
Cache cache_of(const Tensor &k, const Tensor &v, const Tensor &k_scale, const Tensor &v_scale, const Tensor &k_sum, const Tensor &k_mean, const Optional &weight) {
  return Cache{k, v, k_scale, v_scale, k_sum, k_mean, weight.value_or(Tensor())};
}
void cache_append_op(const Tensor &kc, const Tensor &vc, const Tensor &ks, const Tensor &vs, const Tensor &sum, const Tensor &mean, const Optional &weight, const Tensor &k, const Tensor &v,
                     const Tensor &cu, int64_t max_seqlen, const Tensor &seqlens_k, const Tensor &table) {
  py::gil_scoped_release nogil;
  at::AutoDispatchBelowADInplaceOrView below;
  append_raw(cache_of(kc, vc, ks, vs, sum, mean, weight), k, v, cu, max_seqlen, seqlens_k, table);
}

std::pair<Tensor, Tensor> cache_attn_op(const Tensor &q, const Tensor &kc, const Tensor &vc, const Tensor &ks, const Tensor &vs, const Tensor &sum, const Tensor &mean, const Optional &weight,
                                        const Tensor &cu, int64_t max_q, const Tensor &seqlens_k, int64_t max_k, const Tensor &table, int64_t topk, std::optional<double> scale, bool add_weight) {
  py::gil_scoped_release nogil;
  at::AutoDispatchBelowADInplaceOrView below;
  return attn_raw(q, cache_of(kc, vc, ks, vs, sum, mean, weight), cu, seqlens_k, table, AttnForm{max_q, max_k, topk, scale, add_weight});
}

}  // namespace

void fmoba_host::bind_cache_ops(py::module_ &m) {
  m.def("rotary", &rotary);
  m.def("rotary_raw", &rotary_raw);
  m.def("cache_append", &cache_append);
  m.def("cache_append_op", &cache_append_op);
  m.def("cache_attn", &cache_attn);
  m.def("cache_attn_op", &cache_attn_op);
  m.def("cache_step", &cache_step);
  m.def("cache_evict", &cache_evict);
  m.def("cache_evict_op", &evict_raw);
}
