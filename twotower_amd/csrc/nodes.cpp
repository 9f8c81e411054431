// The eager calls of the token lookup, preference loss and gradient clipping, as a Python module on torch's C++
// interface: argument checks, outputs, autograd nodes, and the calls of the C ABI (twotower_amd.h).
//
// A small batch's forward and backward are bound by the host: autograd runs a GPU node on a thread of its
// own, where a node written in Python costs twice what it does on the caller's, and a list of gradients is
// walked tensor by tensor.  Calls in Python and here (us): lookup of 37 x 29 tokens of 100 with its gradient 78 and
// 43 (a node that does nothing 39; GPU 11), preference loss of 64 x 128 with its gradients 103 and 50-67 (GPU 9),
// clipping of 150 tensors 120 and 42 (GPU 43; 30 since a launch takes them all).
//
// The C ABI comes as addresses from the loaded library (bind), so the module has no second copy of it.  Calls are
// made directly unless someone times or records them (_lib.TIMER, record_calls); then through _lib.call.
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/extension.h>

#include <algorithm>
#include <optional>
#include <string>
#include <typeindex>
#include <unordered_map>
#include <unordered_set>

#include "twotower_amd.h"

namespace py = pybind11;
using at::ScalarType;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

namespace {

// ---- the C ABI
struct Abi {
  decltype(&tt_last_error) last_error;
  decltype(&tt_lookup_fwd) lookup_fwd;
  decltype(&tt_lookup_plan_size) lookup_plan_size;
  decltype(&tt_lookup_plan) lookup_plan;
  decltype(&tt_lookup_bwd_ws_size) lookup_bwd_ws_size;
  decltype(&tt_lookup_bwd) lookup_bwd;
  decltype(&tt_preference_fwd) preference_fwd;
  decltype(&tt_preference_bwd) preference_bwd;
  decltype(&tt_clip_ws_size) clip_ws_size;
  decltype(&tt_clip_grads) clip_grads;
} abi;
PyObject *py_calls, *py_timer, *py_call;  // _lib._CALLS, _lib.TIMER, _lib.call: kept for the process's life

void bind(const py::dict& address, const py::list& calls, const py::object& timer, const py::object& call) {
  auto set = [&](auto& fn, const char* name) {
    fn = reinterpret_cast<std::decay_t<decltype(fn)>>(address[name].cast<size_t>());
  };
  set(abi.last_error, "tt_last_error");
  set(abi.lookup_fwd, "tt_lookup_fwd");
  set(abi.lookup_plan_size, "tt_lookup_plan_size");
  set(abi.lookup_plan, "tt_lookup_plan");
  set(abi.lookup_bwd_ws_size, "tt_lookup_bwd_ws_size");
  set(abi.lookup_bwd, "tt_lookup_bwd");
  set(abi.preference_fwd, "tt_preference_fwd");
  set(abi.preference_bwd, "tt_preference_bwd");
  set(abi.clip_ws_size, "tt_clip_ws_size");
  set(abi.clip_grads, "tt_clip_grads");
  py_calls = py::object(calls).release().ptr();
  py_timer = py::object(timer).release().ptr();
  py_call = py::object(call).release().ptr();
}

bool truth(PyObject* o, const char* name) { return py::handle(o).attr(name).cast<bool>(); }
bool observed() { return PyList_GET_SIZE(py_calls) > 0 || truth(py_timer, "enabled") || truth(py_timer, "stamping"); }

template <typename T>
py::object as_py(T v) {
  if constexpr (std::is_pointer_v<T>) return py::int_(reinterpret_cast<size_t>(v));
  else return py::cast(v);
}

// fn(args..., stream) on t's GPU and its current stream, whichever GPU is current.
template <typename F, typename... A>
void launch(const Tensor& t, const char* name, F fn, A... args) {
  const c10::DeviceGuard guard(t.device());
  tt_stream_t stream = reinterpret_cast<tt_stream_t>(c10::hip::getCurrentHIPStream(t.get_device()).stream());
  py::gil_scoped_acquire gil;
  if (observed()) {
    try {
      py::reinterpret_borrow<py::object>(py_call)(name, as_py(args)..., as_py(stream));
    } catch (py::error_already_set& e) {  // (the backward's thread hands on torch's errors, not Python's)
      TORCH_CHECK(false, e.what());
    }
    return;
  }
  if (const int rc = fn(args..., stream)) {
    const char* why = abi.last_error();
    TORCH_CHECK(false, "twotower_amd: ", name, " failed (code ", rc, "): ", why ? why : "");
  }
}

// ---- arguments
int elem_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case ScalarType::Float: return TT_E_F32;
    case ScalarType::BFloat16: return TT_E_BF16;
    case ScalarType::Half: return TT_E_F16;
    default: return -1;
  }
}
int ids_code(const Tensor& ids) { return ids.scalar_type() == ScalarType::Long ? TT_IDS_I64 : TT_IDS_I32; }

void check_elem(const Tensor& t, const char* name) {
  TORCH_CHECK_TYPE(elem_code(t) >= 0, name, " must be float32, bfloat16 or float16, got ", t.scalar_type());
}

// Every tensor on the first one's GPU: a kernel gets raw pointers, so a mixed call would fault.
void check_gpu(const Tensor& first, std::initializer_list<const Tensor*> others) {
  auto on_gpu = [](const Tensor& t) {
    TORCH_CHECK(t.is_cuda(), "twotower_amd: the HIP kernels need GPU tensors (no CPU fallback); got a tensor on ",
                t.device());
  };
  on_gpu(first);
  for (const Tensor* t : others)
    if (t->defined()) {
      on_gpu(*t);
      TORCH_CHECK(t->device() == first.device(), "twotower_amd: tensors on different devices (", first.device(), " and ",
                  t->device(), ")");
    }
}

Tensor bytes_like(const Tensor& t, size_t n) { return at::empty({(int64_t)n}, t.options().dtype(at::kByte)); }
template <typename T>
T* as(const Tensor& t) {
  return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}

void no_second_derivative(const char* what) {  // (create_graph: it would be dropped without a word)
  TORCH_CHECK(!at::GradMode::is_enabled(), what,
              " has no second derivative: backward with create_graph=True is not supported");
}

// ---- token lookup
struct LookupArgs {
  int64_t V, E, pad;
  double scale;
  ScalarType table, rows;
  bool strict = false;  // of the call's own rows alone: NaN for an id outside the table
  void save(AutogradContext* ctx) const {
    ctx->saved_data["lookup"] = std::make_tuple(V, E, pad, scale, (int64_t)table, (int64_t)rows);
  }
  static LookupArgs load(AutogradContext* ctx) {
    const auto [V, E, pad, scale, table, rows] =
        ctx->saved_data["lookup"].to<std::tuple<int64_t, int64_t, int64_t, double, int64_t, int64_t>>();
    return {V, E, pad, scale, (ScalarType)table, (ScalarType)rows};
  }
};

Tensor lookup_rows(const Tensor& weight, const Tensor& ids, const LookupArgs& a) {
  auto shape = ids.sizes().vec();
  shape.push_back(a.E);
  const Tensor out = at::empty(shape, weight.options().dtype(a.rows));
  if (ids.numel())
    launch(weight, "tt_lookup_fwd", abi.lookup_fwd, as<const void>(weight), elem_code(weight), a.V, (int)a.E,
           a.V > 1 ? weight.stride(0) : a.E, as<const void>(ids),
           ids_code(ids) | (a.strict ? TT_LOOKUP_NAN_OUTSIDE : 0), ids.numel(), (float)a.scale, as<void>(out), elem_code(out));
  return out;
}

Tensor lookup_grad(const Tensor& grad_rows, const Tensor& ids, const LookupArgs& a) {
  const Tensor dout = grad_rows.contiguous();
  const int64_t n = ids.numel();
  const Tensor grad = at::empty({a.V, a.E}, dout.options().dtype(a.table));
  Tensor plan, ws;
  const size_t plan_bytes = abi.lookup_plan_size(n, a.V, (int)a.E, elem_code(dout));
  const size_t ws_bytes = abi.lookup_bwd_ws_size(n, (int)a.E, elem_code(dout));
  if (plan_bytes) {  // (a short call takes neither)
    // Sorted here, not beside the forward on a side stream: the gather fills the memory system and every CU,
    // and the sort beside it ended no sooner (forward and backward back to back 352 against 344 us at
    // 8192 x 64 tokens).  Buffers per call, not shared: two captured graphs, or streams, may run their
    // backwards at once.
    plan = bytes_like(dout, plan_bytes);
    ws = bytes_like(dout, ws_bytes);
    launch(dout, "tt_lookup_plan", abi.lookup_plan, as<const void>(ids), ids_code(ids), n, a.V, a.pad, as<void>(plan),
           plan_bytes);
  }
  launch(dout, "tt_lookup_bwd", abi.lookup_bwd, as<const void>(dout), elem_code(dout), as<const void>(ids), ids_code(ids),
         n, a.V, (int)a.E, a.pad, (float)a.scale, as<void>(grad), elem_code(grad), as<const void>(plan), plan_bytes,
         as<void>(ws), ws_bytes);
  return grad;
}

struct LookupGrad;

struct Lookup : Function<Lookup> {
  static Tensor forward(AutogradContext* ctx, const Tensor& weight, const Tensor& ids, const LookupArgs& a) {
    ctx->save_for_backward({ids});
    a.save(ctx);
    return lookup_rows(weight, ids, a);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g);
};

// The gradient is linear in dout, so its own derivative is a lookup again (without padding_idx's rows).
struct LookupGrad : Function<LookupGrad> {
  static Tensor forward(AutogradContext* ctx, const Tensor& dout, const Tensor& ids, const LookupArgs& a) {
    ctx->save_for_backward({ids});
    a.save(ctx);
    return lookup_grad(dout, ids, a);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    Tensor ids = ctx->get_saved_variables()[0];
    LookupArgs a = LookupArgs::load(ctx);
    if (a.pad >= 0) ids = ids.masked_fill(ids.eq(a.pad), -1);
    a.pad = -1;
    return {Lookup::apply(g[0].contiguous(), ids, a), Tensor(), Tensor()};
  }
};

variable_list Lookup::backward(AutogradContext* ctx, variable_list g) {
  const Tensor ids = ctx->get_saved_variables()[0];
  const LookupArgs a = LookupArgs::load(ctx);
  return {at::GradMode::is_enabled() ? LookupGrad::apply(g[0], ids, a) : lookup_grad(g[0], ids, a), Tensor(), Tensor()};
}

Tensor embedding_lookup(const Tensor& weight, const Tensor& ids, double scale, std::optional<int64_t> padding_idx,
                        std::optional<ScalarType> out_dtype, bool strict) {
  TORCH_CHECK_VALUE(weight.dim() == 2 && weight.numel() > 0, "weight must be a non-empty (V, E) table, got shape ",
                    weight.sizes());
  check_elem(weight, "weight");
  TORCH_CHECK_TYPE(ids.scalar_type() == ScalarType::Int || ids.scalar_type() == ScalarType::Long,
                   "token ids must be int32 or int64, got ", ids.scalar_type());
  const int64_t V = weight.size(0), E = weight.size(1);
  TORCH_CHECK_VALUE((weight.stride(1) == 1 || E == 1) && (weight.stride(0) >= E || V == 1),
                    "weight rows must be contiguous and must not overlap, got strides ", weight.strides());
  const ScalarType table = weight.scalar_type(), rows = out_dtype.value_or(table);
  TORCH_CHECK_TYPE(rows == table || (table == ScalarType::Float &&
                                     (rows == ScalarType::BFloat16 || rows == ScalarType::Half)),
                   "out_dtype ", rows, " from a ", table, " table is not supported");
  TORCH_CHECK_VALUE(V < TT_LOOKUP_MAX && E < TT_LOOKUP_MAX && ids.numel() < TT_LOOKUP_MAX, "at most ", TT_LOOKUP_MAX - 1,
                    " ids, rows and columns, got ", ids.numel(), " ids for shape ", weight.sizes());
  int64_t pad = -1;
  if (padding_idx) {
    pad = *padding_idx;
    TORCH_CHECK_VALUE(-V <= pad && pad < V, "padding_idx ", pad, " outside a table of ", V, " rows");
    pad += pad < 0 ? V : 0;
  }
  check_gpu(weight, {&ids});
  const LookupArgs a{V, E, pad, scale, table, rows, strict};
  const Tensor i = ids.contiguous();
  return weight.requires_grad() && at::GradMode::is_enabled() ? Lookup::apply(weight, i, a) : lookup_rows(weight, i, a);
}

// ---- preference loss
struct PrefArgs {
  Tensor ref, mask;  // undefined: none (constants, so no inputs of the nodes)
  int64_t kind;
  double beta, inv_tau, smooth;
};

// dl/dh (B K), 1 / pairs, then 2 B words of scratch
Tensor pref_loss(const Tensor& q, const Tensor& p, const Tensor& n, const PrefArgs& a, const Tensor& loss) {
  const int64_t B = n.size(0), K = n.size(1);
  const Tensor side = at::empty({B * K + 1 + 2 * B}, loss.options());
  float* s = as<float>(side);
  launch(q, "tt_preference_fwd", abi.preference_fwd, as<const void>(q), q.stride(0), as<const void>(p), p.stride(0),
         as<const void>(n), n.stride(0), n.stride(1), elem_code(q), B, (int)K, (int)n.size(2), as<const float>(a.ref),
         as<const uint8_t>(a.mask), (int)a.kind, (float)a.beta, (float)a.inv_tau, (float)a.smooth, s, (float*)nullptr,
         as<float>(loss), s + B * K, (void*)(s + B * K + 1), (size_t)(8 * B));
  return side;
}

void pref_grad(const Tensor& q, const Tensor& p, const Tensor& n, const Tensor& mask, double inv_tau, const Tensor& side,
               const Tensor& grad_loss, const Tensor& dq, const Tensor& dp, const Tensor& dn) {
  const int64_t B = n.size(0), K = n.size(1);
  const float* s = as<const float>(side);
  const Tensor g = grad_loss.to(at::kFloat);
  launch(q, "tt_preference_bwd", abi.preference_bwd, as<const void>(q), q.stride(0), as<const void>(p), p.stride(0),
         as<const void>(n), n.stride(0), n.stride(1), elem_code(q), B, (int)K, (int)n.size(2), as<const uint8_t>(mask),
         (float)inv_tau, s, s + B * K, as<const float>(g), as<void>(dq), as<void>(dp), as<void>(dn));
}

// t[0], t[1], ... are contiguous and follow each other in one storage
bool consecutive(at::ArrayRef<Tensor> t) {
  for (size_t i = 0; i < t.size(); ++i) {
    if (!t[i].is_contiguous()) return false;
    if (i && (t[i].scalar_type() != t[0].scalar_type() || !t[i].is_alias_of(t[0]) ||
              t[i].storage_offset() != t[i - 1].storage_offset() + t[i - 1].numel()))
      return false;
  }
  return true;
}

Tensor pref_forward(AutogradContext* ctx, const Tensor& q, const Tensor& p, const Tensor& n, const PrefArgs& a) {
  const Tensor loss = at::empty({}, q.options().dtype(at::kFloat));
  ctx->save_for_backward({q, p, n, a.mask, pref_loss(q, p, n, a, loss)});
  ctx->saved_data["inv_tau"] = a.inv_tau;
  return loss;
}

variable_list pref_backward(AutogradContext* ctx, const variable_list& g, bool one_buffer) {
  no_second_derivative("preference_loss");
  const auto s = ctx->get_saved_variables();
  const Tensor &q = s[0], &p = s[1], &n = s[2];
  Tensor dq, dp, dn;
  if (one_buffer) {
    const int64_t B = q.size(0);
    const Tensor all = at::empty({B * (2 + n.size(1)), q.size(1)}, q.options());
    dq = all.narrow(0, 0, B);
    dp = all.narrow(0, B, B);
    dn = all.narrow(0, 2 * B, B * n.size(1)).view(n.sizes());
  } else {
    auto like = [](const Tensor& t) { return at::empty_like(t, {}, at::MemoryFormat::Contiguous); };
    dq = like(q);
    dp = like(p);
    dn = like(n);
  }
  pref_grad(q, p, n, s[3], ctx->saved_data["inv_tau"].toDouble(), s[4], g[0], dq, dp, dn);
  return {dq, dp, dn, Tensor()};
}

struct PreferenceLoss : Function<PreferenceLoss> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& p, const Tensor& n, const PrefArgs& a) {
    return pref_forward(ctx, q, p, n, a);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) { return pref_backward(ctx, g, false); }
};

// The same loss of consecutive row blocks of one tensor (TwoTower's fused output): the three gradients are
// written as consecutive blocks too, which SplitRows hands on whole.
struct PreferenceLossPacked : Function<PreferenceLossPacked> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& p, const Tensor& n, const PrefArgs& a) {
    return pref_forward(ctx, q, p, n, a);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) { return pref_backward(ctx, g, true); }
};

// x cut into consecutive row blocks, as torch.split does, but gradients that are consecutive blocks of one buffer
// again (PreferenceLossPacked's) are that buffer: no launch and no copy (torch.split joins them by a cat: 25 MB read
// and written for 3 x 8192 x 256 floats).  Whatever autograd has between the blocks and the loss -- a hook, a retained
// gradient, a function of the caller's -- sees its own block's gradient.
struct SplitRows : Function<SplitRows> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, std::vector<int64_t> sizes) {
    ctx->set_materialize_grads(false);
    variable_list blocks;
    int64_t at = 0;
    for (const int64_t n : sizes) {
      blocks.push_back(x.narrow(0, at, n));
      at += n;
    }
    ctx->saved_data["sizes"] = sizes;
    return blocks;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto sizes = ctx->saved_data["sizes"].toIntVector();
    int64_t rows = 0;
    size_t defined = 0, one = 0;
    for (size_t i = 0; i < g.size(); ++i) {
      rows += sizes[i];
      if (g[i].defined()) {
        ++defined;
        one = i;
      }
    }
    if (!defined) return {Tensor(), Tensor()};
    auto shape = g[one].sizes().vec();
    if (defined == g.size() && !at::GradMode::is_enabled() && consecutive(g)) {
      shape[0] = rows;
      return {g[0].as_strided(shape, at::detail::defaultStrides(shape), g[0].storage_offset()), Tensor()};
    }
    for (size_t i = 0; i < g.size(); ++i)
      if (!g[i].defined()) {
        shape[0] = sizes[i];
        g[i] = at::zeros(shape, g[one].options());
      }
    return {at::cat(g, 0), Tensor()};
  }
};

// The first of some leaves that an autograd graph lives of (-1: none does).
int64_t live_leaf(const std::vector<Tensor>& leaves) {
  for (size_t i = 0; i < leaves.size(); ++i)
    if (torch::autograd::impl::try_get_grad_accumulator(leaves[i])) return (int64_t)i;
  return -1;
}

variable_list split_rows(const Tensor& x, std::vector<int64_t> sizes) {
  int64_t rows = 0;
  for (const int64_t n : sizes) {
    TORCH_CHECK_VALUE(n >= 0, "split_rows: a block of ", n, " rows");
    rows += n;
  }
  TORCH_CHECK_VALUE(x.dim() >= 1 && !sizes.empty() && rows == x.size(0), "split_rows: blocks of ", rows,
                    " rows for shape ", x.sizes());
  return SplitRows::apply(x, std::move(sizes));
}

bool is_slice(torch::autograd::Node& node) {  // (under the GIL)
  static const std::unordered_set<std::string> names = {
      "SplitBackward0", "SplitWithSizesBackward0", "UnsafeSplitBackward0", "UnsafeSplitWithSizesBackward0",
      "SliceBackward0", "ViewBackward0", "UnsafeViewBackward0", "ReshapeAliasBackward0", "AliasBackward0",
      "UnsqueezeBackward0"};
  static std::unordered_map<std::type_index, bool> known;
  const auto [at, is_new] = known.try_emplace(typeid(node), false);
  if (is_new)
    at->second = names.count(node.name()) || dynamic_cast<torch::autograd::CppNode<SplitRows>*>(&node);
  return at->second;
}

// Whether all of autograd between base and each view are torch's own slices and reshapes (or split_rows): a gradient
// of base then stands for the views'.  Not with a hook or a retained gradient on the way, nor a function of the
// caller's that returns a view, nor for a view that is a leaf of its own or was taken under no_grad.  kRows: and the
// last of them is split_rows for all, so that gradients in one buffer reach the base as that buffer.
enum Views { kOther = 0, kDirect = 1, kRows = 2 };
Views views_of(const Tensor& base, const std::vector<Tensor>& views) {
  using torch::autograd::Node;
  for (const Tensor& v : views)
    if (v.requires_grad() != base.requires_grad()) return kOther;
  if (!base.requires_grad()) return kRows;
  const auto to = torch::autograd::impl::gradient_edge(base);
  Views kind = kRows;
  for (const Tensor& v : views) {
    auto at = torch::autograd::impl::gradient_edge(v);
    while (!(at == to)) {
      Node* const node = at.function.get();
      if (!node || node->num_outputs() != 1 || !node->tensor_pre_hooks().empty() || !node->pre_hooks().empty() ||
          !node->post_hooks().empty() || !node->retains_grad_hooks().empty() || !is_slice(*node))
        return kOther;
      at = node->next_edge(0);
      if (at == to && !dynamic_cast<torch::autograd::CppNode<SplitRows>*>(node)) kind = kDirect;
    }
  }
  return kind;
}
bool direct_views(const Tensor& base, const std::vector<Tensor>& views, bool rows) {
  return views_of(base, views) >= (rows ? kRows : kDirect);
}

// The contiguous matrix whose consecutive row blocks, all of them and in order, are the views, where it stands for
// them (views_of); and whether the blocks are split_rows'.
std::pair<std::optional<Tensor>, bool> packed_base(const std::vector<Tensor>& views) {
  const std::pair<std::optional<Tensor>, bool> none{std::nullopt, false};
  if (!views[0].is_view()) return none;
  const Tensor base(views[0]._base());
  if (base.dim() != 2 || !base.is_contiguous()) return none;
  int64_t at = base.storage_offset();
  for (const Tensor& v : views) {
    if (!v.is_view() || v._base().unsafeGetTensorImpl() != base.unsafeGetTensorImpl() || v.dim() != 2 ||
        !v.is_contiguous() || v.size(1) != base.size(1) || v.scalar_type() != base.scalar_type() ||
        v.storage_offset() != at)
      return none;
    at += v.numel();
  }
  if (at != base.storage_offset() + base.numel()) return none;
  const Views kind = views_of(base, views);
  if (kind == kOther) return none;
  return {base, kind == kRows};
}

// (q, p, n with a pair axis) of a checked call, rows of contiguous elements
std::array<Tensor, 3> pref_args(const Tensor& q, const Tensor& p, const Tensor& n) {
  TORCH_CHECK_VALUE(q.dim() == 2 && p.sizes() == q.sizes(), "q and p must both be (B, H), got ", q.sizes(), " and ",
                    p.sizes());
  const Tensor n3 = n.dim() == 2 ? n.unsqueeze(1) : n;
  TORCH_CHECK_VALUE(n3.dim() == 3 && n3.size(0) == q.size(0) && n3.size(2) == q.size(1) && n3.size(1) >= 1,
                    "n must be (B, H) or (B, K, H) with K >= 1 beside q ", q.sizes(), ", got ", n.sizes());
  TORCH_CHECK_VALUE(q.size(1) >= 1, "H must be at least 1");
  check_elem(q, "q");
  TORCH_CHECK_TYPE(p.scalar_type() == q.scalar_type() && n.scalar_type() == q.scalar_type(),
                   "q, p and n must have one type, got ", q.scalar_type(), ", ", p.scalar_type(), ", ", n.scalar_type());
  TORCH_CHECK_VALUE(q.size(0) * n3.size(1) < (int64_t(1) << 31) && q.size(1) < (int64_t(1) << 31), "too many pairs: ",
                    n3.sizes());
  auto rows = [](const Tensor& t) { return t.size(-1) == 1 || t.stride(-1) == 1 ? t : t.contiguous(); };
  return {rows(q), rows(p), rows(n3)};
}

// a contiguous (B, K) side input (ref_margin, mask); (B) is taken where K = 1
Tensor pref_pairs(const std::optional<Tensor>& t, const char* name, ScalarType type, const Tensor& n) {
  if (!t) return {};
  const int64_t B = n.size(0), K = n.size(1);
  TORCH_CHECK_VALUE(t->sizes().equals({B, K}) || (K == 1 && t->sizes().equals({B})), name, " must be (", B, ", ", K,
                    "), got ", t->sizes());
  TORCH_CHECK(t->device() == n.device(), "twotower_amd: ", name, " is on ", t->device(), ", the embeddings on ",
              n.device());
  const bool bools = type == ScalarType::Bool;
  TORCH_CHECK_TYPE(bools ? t->scalar_type() == type : t->is_floating_point(), name, " must be ",
                   bools ? "bool" : "a floating-point tensor", ", got ", t->scalar_type());
  return t->detach().to(type).contiguous();
}

Tensor preference_loss(const Tensor& q_, const Tensor& p_, const Tensor& n_, const std::optional<Tensor>& ref_margin,
                       const std::optional<Tensor>& mask_, int64_t kind, double beta, double inv_tau, double smooth) {
  const auto [q, p, n] = pref_args(q_, p_, n_);
  const Tensor ref = pref_pairs(ref_margin, "ref_margin", ScalarType::Float, n);
  const Tensor mask = pref_pairs(mask_, "mask", ScalarType::Bool, n);
  check_gpu(q, {&p, &n});
  const PrefArgs a{ref, mask, kind, beta, inv_tau, smooth};
  // (leaves keep gradients of their own memory)
  const bool packed = !q.is_leaf() && !p.is_leaf() && !n.is_leaf() && consecutive({q, p, n});
  return packed ? PreferenceLossPacked::apply(q, p, n, a) : PreferenceLoss::apply(q, p, n, a);
}

Tensor preference_margin(const Tensor& q_, const Tensor& p_, const Tensor& n_, double inv_tau) {
  const auto [q, p, n] = pref_args(q_.detach(), p_.detach(), n_.detach());
  check_gpu(q, {&p, &n});
  const int64_t B = n.size(0), K = n.size(1);
  const Tensor margins = at::empty({B, K}, q.options().dtype(at::kFloat));
  launch(q, "tt_preference_fwd", abi.preference_fwd, as<const void>(q), q.stride(0), as<const void>(p), p.stride(0),
         as<const void>(n), n.stride(0), n.stride(1), elem_code(q), B, (int)K, (int)n.size(2), (const float*)nullptr,
         (const uint8_t*)nullptr, 0, 1.f, (float)inv_tau, 0.f, (float*)nullptr, as<float>(margins), (float*)nullptr,
         (float*)nullptr, (void*)nullptr, (size_t)0);
  return margins;
}

// ---- gradient norm and clipping
// t's elements fill one block of memory, in any order (a norm and a product need no more)
bool dense(const Tensor& t) { return t.is_contiguous() || t.is_non_overlapping_and_dense(); }

Tensor clip_grad_norm(const std::vector<Tensor>& grads, std::optional<double> max_norm, bool inf_norm,
                      const std::optional<std::vector<Tensor>>& out) {
  const bool scale = max_norm.has_value();
  const std::vector<Tensor>& outs = out ? *out : grads;
  const size_t count = grads.size();
  TORCH_CHECK_VALUE(outs.size() == count, outs.size(), " out tensors for ", count, " gradients");
  std::vector<uint8_t> type(count), otype(count);
  for (size_t i = 0; i < count; ++i) {
    const int s = elem_code(grads[i]), d = elem_code(outs[i]);
    TORCH_CHECK_TYPE(s >= 0 && (d == s || d == TT_E_F32), "gradient ", i, " of ", grads[i].scalar_type(), " into ",
                     outs[i].scalar_type(), ": float32, bfloat16 or float16, into its own type or float32");
    TORCH_CHECK(grads[i].layout() == at::kStrided && outs[i].layout() == at::kStrided,
                "clip_grad_norm does not support sparse gradients");
    type[i] = (uint8_t)s;
    otype[i] = (uint8_t)d;
  }
  // what the kernels read and write: the tensors themselves where their elements lie in one block
  std::vector<Tensor> kept;
  std::vector<std::pair<Tensor, Tensor>> copies;  // (tensor, its result elsewhere)
  kept.reserve(2 * count);
  std::vector<const void*> src(count);
  std::vector<void*> dst(count);
  std::vector<int64_t> n(count);
  for (size_t i = 0; i < count; ++i) {
    const Tensor &g = grads[i], &o = outs[i];
    n[i] = g.numel();
    if (!out) {
      const Tensor t = dense(g) ? g : g.contiguous();
      src[i] = dst[i] = t.data_ptr();
      if (!t.is_same(g)) {
        TORCH_CHECK_VALUE(!scale || at::has_internal_overlap(g) != at::MemOverlap::Yes, "a gradient of shape ", g.sizes(),
                          " has elements that share memory (an expanded tensor): clip a copy");
        kept.push_back(t);
        if (scale) copies.emplace_back(g, t);
      }
      continue;
    }
    TORCH_CHECK_VALUE(g.sizes() == o.sizes(), "out ", i, " has shape ", o.sizes(), ", the gradient ", g.sizes());
    const Tensor s = g.contiguous();
    const Tensor d = o.is_contiguous() ? o : at::empty_like(o, {}, at::MemoryFormat::Contiguous);
    src[i] = s.data_ptr();
    dst[i] = d.data_ptr();
    if (!s.is_same(g)) kept.push_back(s);
    if (!d.is_same(o)) copies.emplace_back(o, d);
  }
  if (scale) {  // what is written lies apart, and apart from what is read elsewhere
    auto bytes = [](int code) { return code == TT_E_F32 ? 4 : 2; };
    std::vector<std::pair<const char*, const char*>> written;
    written.reserve(count);
    for (size_t i = 0; i < count; ++i)
      if (n[i]) {
        const char* at = static_cast<const char*>(dst[i]);
        written.emplace_back(at, at + n[i] * bytes(otype[i]));
      }
    std::sort(written.begin(), written.end());
    for (size_t k = 1; k < written.size(); ++k)
      TORCH_CHECK_VALUE(written[k - 1].second <= written[k].first,
                        "a gradient is written twice: the same memory is listed more than once");
    if (out)
      for (size_t i = 0; i < count; ++i) {
        if (!n[i] || (src[i] == dst[i] && type[i] == otype[i])) continue;
        const char* at = static_cast<const char*>(src[i]);
        const auto next = std::upper_bound(written.begin(), written.end(), at,
                                           [](const char* x, const auto& r) { return x < r.second; });
        TORCH_CHECK_VALUE(next == written.end() || next->first >= at + n[i] * bytes(type[i]),
                          "an out tensor is the memory of another gradient, or of its own in another type or place");
      }
  }
  const Tensor& first = grads[0];
  for (size_t i = 0; i < count; ++i) check_gpu(first, {&grads[i], &outs[i]});
  const Tensor norm = at::empty({}, first.options().dtype(at::kFloat));
  const size_t ws_bytes = abi.clip_ws_size((int)count);
  const Tensor ws = bytes_like(first, ws_bytes);
  launch(first, "tt_clip_grads", abi.clip_grads, (const void* const*)src.data(), (void* const*)dst.data(),
         (const int64_t*)n.data(), (const uint8_t*)type.data(), (const uint8_t*)otype.data(), (int)count, (int)inf_norm,
         max_norm.value_or(0.0), (int)scale, as<float>(norm), as<void>(ws), ws_bytes);
  if (scale)  // written past autograd's eyes: what was saved of them is not what they hold
    for (const Tensor& o : outs)
      if (!o.is_inference()) o.unsafeGetTensorImpl()->bump_version();
  for (const auto& [o, t] : copies) o.copy_(t);
  return norm;
}

}  // namespace

PYBIND11_MODULE(_nodes, m) {
  const py::call_guard<py::gil_scoped_release> unlocked;  // (an allocation may wait for the GPU)
  m.def("bind", &bind);
  m.def("embedding_lookup", &embedding_lookup, unlocked);
  m.def("preference_loss", &preference_loss, unlocked);
  m.def("preference_margin", &preference_margin, unlocked);
  m.def("split_rows", &split_rows, unlocked);
  m.def("direct_views", &direct_views);
  m.def("packed_base", &packed_base);
  m.def("live_leaf", &live_leaf);
  m.def("clip_grad_norm", &clip_grad_norm, unlocked);
}
