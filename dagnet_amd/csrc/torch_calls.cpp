// The attention and rotary entries of include/dagnet_hip.h called on torch tensors, with their autograd nodes (dagnet_amd._ops binds this module;
// argument checks and public names: dagnet_amd/attention.py).  Host code only: it allocates, fills the argument structs and calls the entries by the
// addresses that bind() got from the loaded libdagnet_hip.so.
//
// Why not ctypes and a Python autograd.Function, like the other operators: a training call of a small batch spent 128 us on the host (a third of
// it Python in autograd's own thread, on a cold core) for 35 us on the GPU; these nodes take 55.
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>

#include "../../include/dagnet_hip.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

struct Entries {
    decltype(&dagnet_last_error) last_error = nullptr;
    decltype(&dagnet_op_attn_fwd_workspace) fwd_workspace = nullptr;
    decltype(&dagnet_op_attn_fwd) fwd = nullptr;
    decltype(&dagnet_op_attn_bwd_workspace) bwd_workspace = nullptr;
    decltype(&dagnet_op_attn_bwd) bwd = nullptr;
    decltype(&dagnet_op_attn_step_workspace) step_workspace = nullptr;
    decltype(&dagnet_op_attn_step) step = nullptr;
    decltype(&dagnet_op_rotary) rotary = nullptr;
} E;

struct Refused : std::runtime_error {
    using std::runtime_error::runtime_error;
};

void check(int rc) {
    if (rc) throw Refused(std::string("libdagnet_hip: ") + E.last_error() + " (status " + std::to_string(rc) + ")");
}

// host tensors (no stream) reach only entries that a test has bound: dagnet_amd/attention.py refuses them
void *stream_of(const Tensor &t) { return t.is_cuda() ? c10::hip::getCurrentHIPStream(t.get_device()).stream() : nullptr; }
template <typename T> T *ptr(const Tensor &t) { return t.defined() ? static_cast<T *>(t.data_ptr()) : nullptr; }
Tensor floats(const Tensor &like, int64_t n) { return at::empty({n}, like.options().dtype(at::kFloat)); }
Tensor dense(const Tensor &like) { return at::empty_like(like, like.options(), at::MemoryFormat::Contiguous); }
// a gradient, or what a hook returned, as autograd hands it over -> memory that holds its values, unit column stride
Tensor columns(const Tensor &t) {
    if (t._is_zerotensor()) return at::zeros(t.sizes(), t.options());
    if (t.is_neg()) return t.resolve_neg();
    return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous();
}

// The entries write through addresses: what records, replays or replaces torch's operations does not see it.  A traced program would return the memory
// that was allocated for the output as it found it.
void eager() {
    using c10::impl::TorchDispatchModeKey;
    using Modes = c10::impl::TorchDispatchModeTLS;
    if (torch::jit::tracer::isTracing() || (Modes::any_modes_set() && (Modes::get_mode(TorchDispatchModeKey::FAKE) || Modes::get_mode(TorchDispatchModeKey::PROXY) ||
                                                                       Modes::get_mode(TorchDispatchModeKey::FUNCTIONAL))))
        throw Refused("the attention and rotary calls cannot be traced (torch.jit.trace, make_fx, export, fake tensors): call them eagerly, or capture a graph");
}
// and what is more than its memory: its tangent would be lost, its values are elsewhere
void plain(std::initializer_list<const Tensor *> tensors, bool gradients = false) {
    eager();
    using c10::DispatchKey;
    static constexpr c10::DispatchKeySet other({DispatchKey::Python, DispatchKey::Functionalize, DispatchKey::Batched, DispatchKey::FuncTorchBatched,
                                                DispatchKey::FuncTorchGradWrapper}), lazy({DispatchKey::Negative, DispatchKey::ZeroTensor});
    for (const Tensor *p : tensors) {
        if (!p || !p->defined()) continue;
        const Tensor &t = *p;
        if (t._fw_grad(0).defined()) throw Refused("the attention and rotary calls have no forward-mode derivative: an argument carries a tangent");
        if (t.key_set().has_any(gradients ? other : other | lazy))       // columns() makes lazy gradients plain
            throw Refused("the attention and rotary calls take plain tensors: no subclass with its own dispatch, no function transform's, no lazily negated view (resolve_neg())");
    }
}

Tensor given(const std::optional<Tensor> &t) { return t ? *t : Tensor(); }

// What a node saved comes back from autograd as whatever the saved-tensor hooks made of it: activation checkpointing computes it again, offloading
// copies it back.  Addresses and strides are therefore taken from what comes back and never kept from the forward call, and a tensor of another
// shape, type or device than the saved one is refused before a kernel reads it.
void unpacked(const Tensor &t, at::IntArrayRef sizes, at::ScalarType type, const at::Device &device, const char *what) {
    if (t.defined() && t.sizes() == sizes && t.scalar_type() == type && t.device() == device) return;
    throw Refused(std::string("a saved-tensor hook returned ") + what + " with another shape, type or device than was saved");
}
// small plain values of a call, kept with its node
template <typename V> void keep(AutogradContext *ctx, const char *name, const V &v) {
    ctx->saved_data[name] = std::string(reinterpret_cast<const char *>(&v), sizeof(V));
}
template <typename V> V kept(AutogradContext *ctx, const char *name) {
    V v;
    memcpy(&v, ctx->saved_data[name].toStringRef().data(), sizeof(V));
    return v;
}

// addresses of a layout's tables on the device, and how many keys its rows see
struct Tables {
    int64_t row_lo, row_hi, key_lo, key_hi, ptr;
    int32_t max_keys, mean_keys;
};
template <typename T> const T *at_address(int64_t a) { return reinterpret_cast<const T *>(a); }

// what the backward pass needs of the forward call beside its tensors; axes 0: no distance
struct Call {
    Tables t;
    double scale, softcap;
    int64_t nk, kv, axes;
};

// q [nq, H, D], k and v [..., KV, D]: their row and head strides are those of the last three dimensions
dagnet_attn arguments(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &slopes, const Tensor &pos, const Tensor &k_pos, int64_t nk, double scale,
                      double softcap) {
    dagnet_attn a = {};
    a.q = q.data_ptr(); a.k = k.data_ptr(); a.v = v.data_ptr();
    a.slopes = ptr<float>(slopes); a.q_pos = ptr<float>(pos); a.k_pos = ptr<float>(k_pos);
    a.q_row = q.stride(0); a.q_head = q.stride(1);
    a.k_row = k.stride(-3); a.k_head = k.stride(-2);
    a.v_row = v.stride(-3); a.v_head = v.stride(-2);
    a.nq = (int32_t)q.size(0); a.nk = (int32_t)nk;
    a.n_heads = (int32_t)q.size(1); a.n_kv_heads = (int32_t)k.size(-2); a.head_dim = (int32_t)q.size(2);
    a.axes = slopes.defined() ? (int32_t)pos.size(-1) : 0;
    a.dtype = q.scalar_type() == at::kBFloat16;
    a.scale = (float)scale; a.softcap = (float)softcap;
    return a;
}

// -> out, and with grad the rows' statistics and the unrounded output (bf16; fp32: out itself)
std::tuple<Tensor, Tensor, Tensor> attend(dagnet_attn &a, const Tensor &q, const Tables &t, bool grad) {
    const c10::DeviceGuard guard(q.device());
    Tensor out = dense(q), lse, o;
    if (grad) {
        lse = floats(q, q.size(0) * q.size(1));
        o = a.dtype ? at::empty(q.sizes(), q.options().dtype(at::kFloat)) : out;
    }
    const int64_t n = E.fwd_workspace(&a);
    const Tensor ws = n ? floats(q, n) : Tensor();          // of its own: captured calls must not share one
    check(E.fwd(&a, at_address<int32_t>(t.row_lo), at_address<int32_t>(t.row_hi), out.data_ptr(), ptr<float>(lse), a.dtype ? ptr<float>(o) : nullptr,
                ptr<float>(ws), stream_of(q)));
    return {out, lse, o};
}

// gradients that have none of their own: a second derivative through them raises (the error's node is attached to tensors that require a gradient only)
variable_list once(variable_list grads, const char *what) {
    if (!at::GradMode::is_enabled()) return grads;
    for (Tensor &g : grads)
        if (g.defined()) g.set_requires_grad(true);
    return torch::autograd::DelayedError(std::string(what) + " has no second derivative", (int64_t)grads.size())(std::move(grads));
}

struct SceneAttn : torch::autograd::Function<SceneAttn> {
    static Tensor forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v, const std::optional<Tensor> &slopes_,
                          const std::optional<Tensor> &pos_, const std::optional<Tensor> &k_pos_, const Tables &t, double scale, double softcap, const Tensor &held) {
        const Tensor slopes = given(slopes_), pos = given(pos_), k_pos = given(k_pos_);
        dagnet_attn a = arguments(q, k, v, slopes, pos, k_pos, k.size(0), scale, softcap);
        a.max_keys = t.max_keys;
        a.mean_keys = t.mean_keys;
        auto [out, lse, o] = attend(a, q, t, true);
        ctx->save_for_backward({q, k, v, slopes, pos, k_pos, lse, o});
        ctx->saved_data["held"] = held;                     // no saved variable: a hook would put a copy in its place, and the addresses are held's own
        keep(ctx, "call", Call{t, scale, softcap, k.size(0), k.size(1), a.axes});
        return out;
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        plain({&grads[0]}, true);
        const Call call = kept<Call>(ctx, "call");
        const Tables &t = call.t;
        const variable_list saved = ctx->get_saved_variables();
        const Tensor dout = columns(grads[0]);
        const int64_t rows = dout.size(0), heads = dout.size(1), D = dout.size(2);
        const at::ScalarType type = dout.scalar_type();
        unpacked(saved[0], {rows, heads, D}, type, dout.device(), "q");
        unpacked(saved[1], {call.nk, call.kv, D}, type, dout.device(), "k");
        unpacked(saved[2], {call.nk, call.kv, D}, type, dout.device(), "v");
        Tensor slopes, pos, k_pos;
        if (call.axes) {
            unpacked(saved[3], {heads}, at::kFloat, dout.device(), "slopes");
            unpacked(saved[4], {rows, call.axes}, at::kFloat, dout.device(), "pos");
            unpacked(saved[5], {call.nk, call.axes}, at::kFloat, dout.device(), "k_pos");
            slopes = columns(saved[3]).contiguous();
            pos = columns(saved[4]).contiguous();
            k_pos = columns(saved[5]).contiguous();
        }
        unpacked(saved[6], {rows * heads}, at::kFloat, dout.device(), "the rows' statistics");
        unpacked(saved[7], {rows, heads, D}, at::kFloat, dout.device(), "the output");
        const Tensor q = columns(saved[0]), k = columns(saved[1]), v = columns(saved[2]), lse = columns(saved[6]).contiguous(), o = columns(saved[7]).contiguous();
        dagnet_attn a = arguments(q, k, v, slopes, pos, k_pos, call.nk, call.scale, call.softcap);
        a.max_keys = t.max_keys;
        a.mean_keys = t.mean_keys;
        const bool nq = ctx->needs_input_grad(0), nk = ctx->needs_input_grad(1), nv = ctx->needs_input_grad(2), ns = slopes.defined() && ctx->needs_input_grad(3);
        const c10::DeviceGuard guard(q.device());
        Tensor dq, dk, dv, ds;
        if (nq || ns) dq = dense(q);
        if (nk || nv) {
            dk = dense(k);
            dv = dense(v);
        }
        if (ns) ds = dense(slopes);
        const Tensor ws = floats(q, E.bwd_workspace(&a));
        check(E.bwd(&a, at_address<int32_t>(t.row_lo), at_address<int32_t>(t.row_hi), at_address<int32_t>(t.key_lo), at_address<int32_t>(t.key_hi), dout.data_ptr(),
                    dout.stride(0), dout.stride(1), ptr<float>(lse), ptr<float>(o), ptr<float>(ws), ptr<void>(dq), ptr<void>(dk), ptr<void>(dv), ptr<float>(ds),
                    stream_of(q)));
        return once({nq ? dq : Tensor(), nk ? dk : Tensor(), nv ? dv : Tensor(), ds, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()}, "scene_attention");
    }
};

// tables: (row_lo, row_hi, key_lo, key_hi, ptr, (max, mean), the tensor that holds them)
Tables tables_of(const py::tuple &t) {
    const py::tuple span = t[5];
    return {t[0].cast<int64_t>(), t[1].cast<int64_t>(), t[2].cast<int64_t>(), t[3].cast<int64_t>(), t[4].cast<int64_t>(), span[0].cast<int32_t>(), span[1].cast<int32_t>()};
}

Tensor scene_attn(const Tensor &q, const Tensor &k, const Tensor &v, const std::optional<Tensor> &slopes_, const py::tuple &tables, double scale, double softcap,
                  const std::optional<Tensor> &pos_, const std::optional<Tensor> &k_pos_) {
    const Tensor slopes = given(slopes_), pos = given(pos_), k_pos = given(k_pos_);
    plain({&q, &k, &v, &slopes, &pos, &k_pos});
    const Tables t = tables_of(tables);
    if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad() || (slopes.defined() && slopes.requires_grad()))) {
        const Tensor held = tables[6].cast<Tensor>();       // the tables live as long as a backward pass may read them
        py::gil_scoped_release release;
        return SceneAttn::apply(q, k, v, slopes_, pos_, k_pos_, t, scale, softcap, held);
    }
    py::gil_scoped_release release;
    dagnet_attn a = arguments(q, k, v, slopes, pos, k_pos, k.size(0), scale, softcap);
    a.max_keys = t.max_keys;
    a.mean_keys = t.mean_keys;
    return std::get<0>(attend(a, q, t, false));
}

Tensor scene_attn_step(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &k_len, int64_t q_ptr, int64_t max_rows, const std::optional<Tensor> &slopes_,
                       const std::optional<Tensor> &pos_, const std::optional<Tensor> &k_pos_, double scale, double softcap) {
    py::gil_scoped_release release;
    const Tensor slopes = given(slopes_), pos = given(pos_), k_pos = given(k_pos_);
    plain({&q, &k, &v, &k_len, &slopes, &pos, &k_pos});
    dagnet_attn a = arguments(q, k, v, slopes, pos, k_pos, 0, scale, softcap);
    const c10::DeviceGuard guard(q.device());
    const int32_t scenes = (int32_t)k.size(0), room = (int32_t)k.size(1);
    Tensor out = dense(q);
    const int64_t n = E.step_workspace(&a, scenes, room, (int32_t)max_rows);
    const Tensor ws = n ? floats(q, n) : Tensor();
    check(E.step(&a, at_address<int32_t>(q_ptr), ptr<int32_t>(k_len), scenes, room, (int32_t)max_rows, k.stride(0), v.stride(0), out.data_ptr(), ptr<float>(ws),
                 stream_of(q)));
    return out;
}

// what a RotaryAxes holds on the device
struct Axes {
    int64_t turns, axis;
    int32_t pairs;
    bool interleaved;
};

void turn(const Tensor &q, const Tensor &k, const Tensor &pos, const Axes &x, bool inverse, const Tensor &qo, const Tensor &ko) {
    const c10::DeviceGuard guard(q.device());
    const bool two = k.defined();
    const int type = pos.scalar_type() == at::kFloat ? 0 : pos.scalar_type() == at::kInt ? 1 : 2;
    check(E.rotary(q.size(0), (int32_t)q.size(1), two ? (int32_t)k.size(1) : 0, (int32_t)q.size(2), q.scalar_type() == at::kBFloat16, q.data_ptr(), q.stride(0),
                   q.stride(1), ptr<void>(k), two ? k.stride(0) : 0, two ? k.stride(1) : 0, pos.data_ptr(), type, (int32_t)pos.size(1), at_address<double>(x.turns),
                   at_address<int32_t>(x.axis), x.pairs, x.interleaved, inverse, qo.data_ptr(), qo.stride(0), qo.stride(1), ptr<void>(ko), two ? ko.stride(0) : 0,
                   two ? ko.stride(1) : 0, stream_of(q)));
}

struct Rotary : torch::autograd::Function<Rotary> {
    static variable_list forward(AutogradContext *ctx, const Tensor &q, const std::optional<Tensor> &k_, const Tensor &pos, const Axes &x, const Tensor &held) {
        const Tensor k = given(k_);
        const Tensor qo = dense(q), ko = k.defined() ? dense(k) : Tensor();
        turn(q, k, pos, x, false, qo, ko);
        ctx->save_for_backward({pos});
        ctx->saved_data["held"] = held;                     // as in SceneAttn
        keep(ctx, "axes", x);
        keep(ctx, "pos", std::array<int64_t, 2>{pos.size(1), (int64_t)pos.scalar_type()});
        return k.defined() ? variable_list{qo, ko} : variable_list{qo};
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        plain({&grads[0], grads.size() > 1 ? &grads[1] : nullptr}, true);
        const Axes x = kept<Axes>(ctx, "axes");
        const auto was = kept<std::array<int64_t, 2>>(ctx, "pos");
        const Tensor gq = columns(grads[0]), gk = grads.size() > 1 ? columns(grads[1]) : Tensor(), back = ctx->get_saved_variables()[0];
        unpacked(back, {gq.size(0), was[0]}, (at::ScalarType)was[1], gq.device(), "pos");
        const Tensor pos = columns(back).contiguous();
        const Tensor dq = dense(gq), dk = gk.defined() ? dense(gk) : Tensor();
        turn(gq, gk, pos, x, true, dq, dk);
        return once({dq, dk, Tensor(), Tensor(), Tensor()}, "rotary");
    }
};

py::tuple rotary(const Tensor &q, const std::optional<Tensor> &k_, const Tensor &pos, const py::tuple &tables, int64_t pairs, bool interleaved, bool inplace) {
    const Axes x = {tables[0].cast<int64_t>(), tables[1].cast<int64_t>(), (int32_t)pairs, interleaved};
    const Tensor k = given(k_), held = tables[2].cast<Tensor>();
    plain({&q, &k, &pos});
    variable_list out;
    {
        py::gil_scoped_release release;
        if (!inplace && at::GradMode::is_enabled() && (q.requires_grad() || (k.defined() && k.requires_grad()))) out = Rotary::apply(q, k_, pos, x, held);
        else {
            out = {inplace ? q : dense(q), !k.defined() || inplace ? k : dense(k)};
            if (inplace)                                    // what autograd saved of them is no longer what it was
                for (const Tensor &t : out)
                    if (t.defined()) t.unsafeGetTensorImpl()->bump_version();
            turn(q, k, pos, x, false, out[0], out[1]);
        }
    }
    return py::make_tuple(out[0], k.defined() ? py::cast(out[1]) : py::none());
}

void bind(const py::dict &addresses, py::object error) {
    auto get = [&](auto &entry, const char *name) { entry = reinterpret_cast<std::decay_t<decltype(entry)>>(addresses[name].cast<uintptr_t>()); };
    get(E.last_error, "dagnet_last_error");
    get(E.fwd_workspace, "dagnet_op_attn_fwd_workspace");
    get(E.fwd, "dagnet_op_attn_fwd");
    get(E.bwd_workspace, "dagnet_op_attn_bwd_workspace");
    get(E.bwd, "dagnet_op_attn_bwd");
    get(E.step_workspace, "dagnet_op_attn_step_workspace");
    get(E.step, "dagnet_op_attn_step");
    get(E.rotary, "dagnet_op_rotary");
    static py::object *raised = new py::object(std::move(error));        // outlives the interpreter's shutdown order
    py::register_local_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const Refused &e) {
            PyErr_SetString(raised->ptr(), e.what());
        }
    });
}

}  // namespace

PYBIND11_MODULE(_dagnet_torch, m) {
    m.def("bind", &bind);
    m.def("eager", &eager);
    m.def("scene_attn", &scene_attn);
    m.def("scene_attn_step", &scene_attn_step);
    m.def("rotary", &rotary);
}
