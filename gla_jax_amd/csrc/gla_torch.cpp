// The host side of the Python entry points for arrays that are already as the kernels take them (on the GPU, dense, one
// element type): argument checks, buffers, launches and the autograd rules in one native call.  The same path in Python
// took 23 us for a forward and 105 to 210 us for a forward and backward, more than the kernels of a small call; here it
// is about a third of that.  Everything else (other layouts and types, function transforms, error messages) stays in
// gla.py, which calls this again once the arrays are converted, and whose backward rules are called where a transform is active.
#include <ATen/TracerMode.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <ATen/ops/zeros.h>
#include <ATen/ops/zeros_like.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/utils/pybind.h>

#include <array>
#include <optional>

#include "../../include/gla_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// A status of the library as gla_jax_amd._lib.GlaError.  The Python error itself is thrown: out of a backward the autograd
// engine carries it to the caller as it is, while any exception of this file's own would arrive as a plain RuntimeError.
PyObject *gla_error = nullptr;
void check(const char *fn, int status)
{
    if (status == 0) return;
    const py::gil_scoped_acquire gil;
    PyErr_SetObject(gla_error, py::handle(gla_error)(fn, status, gla_status_string(status)).ptr());
    throw py::error_already_set();
}

void *stream_of(const Tensor &t)
{
    return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

bool known(at::ScalarType s) { return s == at::kFloat || s == at::kBFloat16; }
gla_dtype code(const Tensor &t) { return t.scalar_type() == at::kFloat ? GLA_F32 : GLA_BF16; }
bool dense_on_gpu(const Tensor &t) { return t.defined() && t.is_cuda() && t.layout() == at::kStrided && t.is_contiguous(); }

struct Dims {
    int64_t B, T, H, D;
};
Dims dims_of(const Tensor &k)
{
    const auto s = k.sizes();
    const size_t n = s.size();
    int64_t B = 1;
    for (size_t i = 0; i + 3 < n; ++i) B *= s[i];
    return {B, s[n - 3], s[n - 2], s[n - 1]};
}

// The arrays can go to the kernels as they are: see gla.py's _prep for the contract.
bool canonical_rows(const Tensor &g, const Tensor &v, const Tensor &k, const Tensor &q)
{
    for (const Tensor *t : {&g, &v, &k, &q})
        if (!dense_on_gpu(*t) || t->device() != k.device()) return false;
    const auto s = k.sizes();
    if (s.size() < 3 || q.sizes() != s || g.sizes() != s || v.sizes() != s) return false;
    return g.scalar_type() == at::kFloat && known(v.scalar_type()) && k.scalar_type() == v.scalar_type() &&
           q.scalar_type() == v.scalar_type();
}
std::vector<int64_t> state_sizes(const Tensor &k)
{
    std::vector<int64_t> s = k.sizes().vec();
    const size_t n = s.size();
    s[n - 3] = s[n - 2];
    s[n - 2] = s[n - 1];
    return s;
}
bool canonical(const Tensor &h0, const Tensor &g, const Tensor &v, const Tensor &k, const Tensor &q)
{
    return canonical_rows(g, v, k, q) && dense_on_gpu(h0) && h0.device() == k.device() && known(h0.scalar_type()) &&
           h0.sizes() == at::IntArrayRef(state_sizes(k));
}

Tensor bytes_like(size_t n, const Tensor &t) { return at::empty({(int64_t)n}, t.options().dtype(at::kByte)); }

[[noreturn]] void no_double_backward(const char *name)
{
    TORCH_CHECK_NOT_IMPLEMENTED(false, name, ": second-order gradients are not provided (the reference defines first-order "
                                             "custom_vjp rules only)");
    std::abort();
}

// The call goes through the autograd function: a gradient may be asked for, or an array carries a forward-mode tangent,
// which the function refuses (a call past it would drop the tangent without a word).
bool wants_grad(const Tensor &h0, const Tensor &g, const Tensor &v, const Tensor &k, const Tensor &q)
{
    for (const Tensor *t : {&h0, &g, &v, &k, &q})
        if ((at::GradMode::is_enabled() && t->requires_grad()) || t->_fw_grad(/*level=*/0).defined()) return true;
    return false;
}

// ---- chunk_gla ----------------------------------------------------------------------------------
struct ChunkOut {
    Tensor hT, out, states;
};
ChunkOut chunk_forward(const Tensor &h0, const Tensor &g, const Tensor &v, const Tensor &k, const Tensor &q, int64_t chunk,
                       bool residual)
{
    const c10::DeviceGuard guard(k.device());
    const Dims d = dims_of(k);
    const gla_dtype dt = code(v);
    const size_t nws = gla_chunk_fwd_workspace_bytes(d.B, d.T, d.H, d.D, d.D, chunk, dt);
    const size_t nst = residual ? gla_chunk_states_bytes(d.B, d.T, d.H, d.D, d.D, chunk, dt) : 0;
    if (nws == 0) check("gla_chunk_fwd", GLA_ERR_UNSUPPORTED);
    ChunkOut r{at::empty_like(h0), at::empty_like(v), Tensor()};
    // as B rows of bytes, which is how gla.py's rules map them
    if (residual) r.states = at::empty({d.B, (int64_t)(nst + d.B - 1) / d.B}, v.options().dtype(at::kByte));
    const Tensor ws = bytes_like(nws, v);
    check("gla_chunk_fwd",
          gla_chunk_fwd(stream_of(k), d.B, d.T, d.H, d.D, d.D, chunk, dt, code(h0), h0.data_ptr(), (const float *)g.data_ptr(),
                        v.data_ptr(), k.data_ptr(), q.data_ptr(), r.hT.data_ptr(), r.out.data_ptr(),
                        residual ? r.states.data_ptr() : nullptr, ws.data_ptr(), nws));
    return r;
}

variable_list chunk_backward(const Tensor &states, const Tensor &g, const Tensor &v, const Tensor &k, const Tensor &q,
                             const Tensor &dhT, const Tensor &dout, int64_t chunk)
{
    const c10::DeviceGuard guard(k.device());
    const Dims d = dims_of(k);
    const gla_dtype dt = code(v);
    const size_t nws = gla_chunk_bwd_workspace_bytes(d.B, d.T, d.H, d.D, d.D, chunk, dt);
    const Tensor ws = bytes_like(nws, v);
    Tensor dh0 = at::empty_like(dhT), dg = at::empty_like(g), dv = at::empty_like(v), dk = at::empty_like(k),
           dq = at::empty_like(q);
    check("gla_chunk_bwd",
          gla_chunk_bwd(stream_of(k), d.B, d.T, d.H, d.D, d.D, chunk, dt, code(dhT), (const float *)g.data_ptr(), v.data_ptr(),
                        k.data_ptr(), q.data_ptr(), states.data_ptr(), dhT.data_ptr(), dout.data_ptr(), dh0.data_ptr(),
                        (float *)dg.data_ptr(), dv.data_ptr(), dk.data_ptr(), dq.data_ptr(), ws.data_ptr(), nws));
    return {dh0, dg, dv, dk, dq};
}

// What autograd saved: a saved-tensor hook may hand it back in another layout (taken as it is, the kernels would read other
// values), or as another array altogether (refused).
void check_saved(bool as_saved)
{
    TORCH_CHECK(as_saved, "a saved-tensor hook handed back an array of another type, shape or device");
}
variable_list saved_dense(AutogradContext *ctx)
{
    variable_list s = ctx->get_saved_variables();
    for (Tensor &t : s)
        if (t.defined() && !t.is_contiguous()) t = t.contiguous();
    return s;
}
bool holds(const Tensor &bytes, size_t n, const Tensor &like)
{
    return bytes.scalar_type() == at::kByte && bytes.device() == like.device() && (size_t)bytes.numel() >= n;
}
// A function transform can be active in the backward alone (torch.func.vmap over torch.autograd.grad): the cotangents then
// are wrappers without memory of their own, and the rules of gla.py, which know how to map, take over.  The older mapping
// behind is_grads_batched reaches no rule of a custom function.
bool transforms_active()
{
    return c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode);
}
// a cotangent as the kernels take it: zeros where autograd has none, dense, in the type of what it belongs to
Tensor cotangent(const Tensor &d, at::IntArrayRef sizes, at::ScalarType type, const Tensor &like)
{
    if (!d.defined()) return at::zeros(sizes, like.options().dtype(type));
    check_saved(d.sizes() == sizes && d.device() == like.device());
    TORCH_CHECK_NOT_IMPLEMENTED(d.has_storage() || transforms_active(), "batched cotangents (is_grads_batched, jacobian with "
                                "vectorize=True) are not provided: map torch.autograd.grad by torch.func.vmap");
    // (each operation on a tensor that changes nothing costs a microsecond of a small step's hundred)
    return d.scalar_type() == type && d.is_contiguous() ? d : d.to(type).contiguous();
}

template <typename... Args> variable_list python_rule(const char *module, const char *name, Args &&...args)
{
    const py::gil_scoped_acquire gil;
    const py::object r = py::module_::import(module).attr(name).attr("apply")(std::forward<Args>(args)...);
    return r.cast<variable_list>();
}

// The backward rules as functions of their own, used where a graph of the gradients is asked for: what they return can
// be differentiated no further, and says so.
struct ChunkBackward : torch::autograd::Function<ChunkBackward> {
    static variable_list forward(AutogradContext *, const Tensor &states, const Tensor &g, const Tensor &v, const Tensor &k,
                                 const Tensor &q, const Tensor &dhT, const Tensor &dout, int64_t chunk)
    {
        return chunk_backward(states, g, v, k, q, dhT, dout, chunk);
    }
    static variable_list backward(AutogradContext *, variable_list) { no_double_backward("chunk_gla"); }
};

struct Chunk : torch::autograd::Function<Chunk> {      // gla.py:483-550, 552-625
    static variable_list forward(AutogradContext *ctx, const Tensor &h0, const Tensor &g, const Tensor &v, const Tensor &k,
                                 const Tensor &q, int64_t chunk)
    {
        ChunkOut r = chunk_forward(h0, g, v, k, q, chunk, true);
        ctx->save_for_backward({r.states, g, v, k, q});      // residuals of gla.py:542-549
        ctx->saved_data["chunk"] = chunk;
        ctx->saved_data["hidden"] = (int64_t)h0.scalar_type();
        ctx->set_materialize_grads(false);
        return {r.hT, r.out};
    }
    static variable_list backward(AutogradContext *ctx, variable_list d)
    {
        const variable_list s = saved_dense(ctx);
        const int64_t chunk = ctx->saved_data["chunk"].toInt();
        check_saved(canonical_rows(s[1], s[2], s[3], s[4]));
        const Dims n = dims_of(s[3]);
        check_saved(holds(s[0], gla_chunk_states_bytes(n.B, n.T, n.H, n.D, n.D, chunk, code(s[2])), s[3]));
        const Tensor dhT = cotangent(d[0], state_sizes(s[3]), (at::ScalarType)ctx->saved_data["hidden"].toInt(), s[3]);
        const Tensor dout = cotangent(d[1], s[2].sizes(), s[2].scalar_type(), s[2]);
        variable_list r = transforms_active() ? python_rule("gla_jax_amd.gla", "_ChunkGLABwd", s[0], s[1], s[2], s[3], s[4], dhT, dout, chunk)
                          : at::GradMode::is_enabled() ? ChunkBackward::apply(s[0], s[1], s[2], s[3], s[4], dhT, dout, chunk)
                                                       : chunk_backward(s[0], s[1], s[2], s[3], s[4], dhT, dout, chunk);
        r.emplace_back();
        return r;
    }
};

// ---- recurrent_gla ------------------------------------------------------------------------------
// residual: what the forward can leave for the backward (undefined where sequences run whole), if that is wanted
std::pair<Tensor, Tensor> recurrent_forward(const Tensor &h0, const Tensor &g, const Tensor &v, const Tensor &k,
                                            const Tensor &q, bool reverse, bool out_fp32, Tensor *residual = nullptr)
{
    const c10::DeviceGuard guard(k.device());
    const Dims d = dims_of(k);
    const gla_dtype dt = code(v);
    Tensor hT = at::empty_like(h0), out = out_fp32 ? at::empty_like(v, v.options().dtype(at::kFloat)) : at::empty_like(v), ws;
    // a workspace where the library can use one (head dimension 256, few sequences)
    const size_t nws = gla_recurrent_fwd_workspace_bytes(d.B, d.T, d.H, d.D, d.D, dt);
    if (nws) ws = bytes_like(nws, v);
    const size_t nres = residual ? gla_recurrent_residual_bytes(d.B, d.T, d.H, d.D, d.D, dt) : 0;
    if (nres) *residual = bytes_like(nres, v);
    check("gla_recurrent_fwd_res",
          gla_recurrent_fwd_res(stream_of(k), d.B, d.T, d.H, d.D, d.D, dt, code(h0), out_fp32 ? GLA_F32 : dt, reverse,
                               h0.data_ptr(), (const float *)g.data_ptr(), v.data_ptr(), k.data_ptr(), q.data_ptr(),
                               hT.data_ptr(), out.data_ptr(), nres ? residual->data_ptr() : nullptr,
                               nws ? ws.data_ptr() : nullptr, nws));
    return {hT, out};
}

variable_list recurrent_backward(const Tensor &h0, const Tensor &g, const Tensor &v, const Tensor &k, const Tensor &q,
                                 const Tensor &hT, const Tensor &residual, const Tensor &dhT, const Tensor &dout, bool reverse,
                                 bool out_fp32)
{
    const c10::DeviceGuard guard(k.device());
    const Dims d = dims_of(k);
    const gla_dtype dt = code(v);
    Tensor dh0 = at::empty_like(h0), dg = at::empty_like(g), dv = at::empty_like(v), dk = at::empty_like(k),
           dq = at::empty_like(q), ws;
    const size_t nws = gla_recurrent_bwd_workspace_bytes(d.B, d.T, d.H, d.D, d.D, dt);
    if (nws) ws = bytes_like(nws, v);
    check("gla_recurrent_bwd_res",
          gla_recurrent_bwd_res(stream_of(k), d.B, d.T, d.H, d.D, d.D, dt, code(h0), out_fp32 ? GLA_F32 : dt, reverse,
                               h0.data_ptr(), (const float *)g.data_ptr(), v.data_ptr(), k.data_ptr(), q.data_ptr(),
                               hT.data_ptr(), dhT.data_ptr(), dout.data_ptr(), dh0.data_ptr(), (float *)dg.data_ptr(),
                               dv.data_ptr(), dk.data_ptr(), dq.data_ptr(), residual.defined() ? residual.data_ptr() : nullptr,
                               nws ? ws.data_ptr() : nullptr, nws));
    return {dh0, dg, dv, dk, dq};
}

struct RecurrentBackward : torch::autograd::Function<RecurrentBackward> {
    static variable_list forward(AutogradContext *, const Tensor &h0, const Tensor &g, const Tensor &v, const Tensor &k,
                                 const Tensor &q, const Tensor &hT, const std::optional<Tensor> &residual, const Tensor &dhT,
                                 const Tensor &dout, bool reverse, bool out_fp32)
    {
        return recurrent_backward(h0, g, v, k, q, hT, residual.value_or(Tensor()), dhT, dout, reverse, out_fp32);
    }
    static variable_list backward(AutogradContext *, variable_list) { no_double_backward("recurrent_gla"); }
};

struct Recurrent : torch::autograd::Function<Recurrent> {      // gla.py:99-170, 172-269
    static variable_list forward(AutogradContext *ctx, const Tensor &h0, const Tensor &g, const Tensor &v, const Tensor &k,
                                 const Tensor &q, bool reverse, bool out_fp32)
    {
        Tensor residual;
        auto [hT, out] = recurrent_forward(h0, g, v, k, q, reverse, out_fp32, &residual);
        ctx->save_for_backward({h0, g, v, k, q, hT, residual});          // residuals of gla.py:169, and the segments' states
        ctx->saved_data["reverse"] = reverse;
        ctx->saved_data["out_fp32"] = out_fp32;
        ctx->set_materialize_grads(false);
        return {hT, out};
    }
    static variable_list backward(AutogradContext *ctx, variable_list d)
    {
        const variable_list s = saved_dense(ctx);
        check_saved(canonical(s[0], s[1], s[2], s[3], s[4]) && dense_on_gpu(s[5]) && s[5].sizes() == s[0].sizes());
        const Dims n = dims_of(s[3]);
        check_saved(!s[6].defined() || holds(s[6], gla_recurrent_residual_bytes(n.B, n.T, n.H, n.D, n.D, code(s[2])), s[3]));
        const bool reverse = ctx->saved_data["reverse"].toBool(), out_fp32 = ctx->saved_data["out_fp32"].toBool();
        const Tensor dhT = cotangent(d[0], s[0].sizes(), s[0].scalar_type(), s[0]);
        const Tensor dout = cotangent(d[1], s[2].sizes(), out_fp32 ? at::kFloat : s[2].scalar_type(), s[2]);
        variable_list r = transforms_active()
                              ? python_rule("gla_jax_amd.gla", "_RecurrentGLABwd", s[0], s[1], s[2], s[3], s[4], s[5], dhT, dout, reverse, out_fp32)
                          : at::GradMode::is_enabled()
                              ? RecurrentBackward::apply(s[0], s[1], s[2], s[3], s[4], s[5], std::optional<Tensor>(s[6]), dhT, dout, reverse, out_fp32)
                              : recurrent_backward(s[0], s[1], s[2], s[3], s[4], s[5], s[6], dhT, dout, reverse, out_fp32);
        r.resize(7);
        return r;
    }
};

// ---- linear attention with one decay a head -------------------------------------------------------
bool on_16_bytes(const Tensor &t) { return t.numel() == 0 || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }
// Rows [B,T,heads,features] (or [T,heads,features]) that the kernels take where they lie: see decay.py's _rows.
bool rows_on_gpu(const Tensor &t)
{
    if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || t.dim() < 3 || t.dim() > 4 || t.stride(-1) != 1) return false;
    const int64_t piece = 16 / (int64_t)t.element_size();
    for (int64_t i = 0; i + 1 < t.dim(); ++i)
        if (t.size(i) > 1 && t.stride(i) % piece) return false;
    if (t.size(-3) > 1 && t.stride(-3) >= 1 << 23) return false;
    return on_16_bytes(t);
}
struct DecayDims {
    int64_t B, T, H, HK, DK, DV;
};
DecayDims decay_dims(const Tensor &v, const Tensor &k)
{
    return {v.dim() == 4 ? v.size(0) : 1, v.size(-3), v.size(-2), k.size(-2), k.size(-1), v.size(-1)};
}
bool decay_rows(const Tensor &a, const Tensor &v, const Tensor &k, const Tensor &q, const std::optional<Tensor> &lengths)
{
    if (!rows_on_gpu(v) || !rows_on_gpu(k) || !rows_on_gpu(q) || !a.defined() || !a.is_cuda() || a.layout() != at::kStrided) return false;
    const DecayDims n = decay_dims(v, k);
    if (k.dim() != v.dim() || q.sizes() != k.sizes() || k.size(-3) != n.T || (v.dim() == 4 && k.size(0) != n.B)) return false;
    if (n.B < 1 || n.H < 1 || n.HK < 1 || n.H % n.HK || n.DK % 16 || n.DV % 16 || n.DK < 16 || n.DV < 16 || n.DK > 256 || n.DV > 256) return false;
    if (!known(v.scalar_type()) || k.scalar_type() != v.scalar_type() || q.scalar_type() != v.scalar_type()) return false;
    if (a.scalar_type() != at::kFloat || a.size(-1) != n.H) return false;
    if (a.dim() != 1 && (a.dim() != v.dim() - 1 || a.size(-2) != n.T || (v.dim() == 4 && a.size(0) != n.B))) return false;
    for (const Tensor *t : {&a, &k, &q})
        if (t->device() != v.device()) return false;
    if (lengths && (!dense_on_gpu(*lengths) || lengths->scalar_type() != at::kInt || lengths->dim() != v.dim() - 3 ||
                    lengths->numel() != n.B || lengths->device() != v.device()))
        return false;
    return true;
}
std::vector<int64_t> decay_state_sizes(const Tensor &v, const Tensor &k)
{
    const DecayDims n = decay_dims(v, k);
    return v.dim() == 4 ? std::vector<int64_t>{n.B, n.H, n.DK, n.DV} : std::vector<int64_t>{n.H, n.DK, n.DV};
}
std::array<int64_t, 12> decay_strides(const Tensor &a, const Tensor &v, const Tensor &k, const Tensor &q)
{
    std::array<int64_t, 12> s{};
    int64_t i = 0;
    const bool batch = v.dim() == 4;
    s[i++] = a.dim() == 3 ? a.stride(0) : 0;
    s[i++] = a.dim() == 1 ? 0 : a.stride(-2);
    s[i++] = a.stride(-1);
    for (const Tensor *t : {&v, &k, &q}) {
        s[i++] = batch && t->size(0) > 1 ? t->stride(0) : 0;
        s[i++] = t->size(-3) > 1 ? t->stride(-3) : 0;
        s[i++] = t->size(-2) > 1 ? t->stride(-2) : 0;
    }
    return s;
}
const int32_t *lengths_of(const std::optional<Tensor> &lengths)
{
    return lengths ? (const int32_t *)lengths->data_ptr() : nullptr;
}
// a new dense array like `t`
Tensor dense_like(const Tensor &t) { return at::empty(t.sizes(), t.options()); }

ChunkOut decay_forward(const Tensor &h0, const Tensor &a, const Tensor &v, const Tensor &k, const Tensor &q,
                       const std::optional<Tensor> &lengths, bool residual)
{
    const c10::DeviceGuard guard(v.device());
    const DecayDims n = decay_dims(v, k);
    const gla_dtype dt = code(v);
    const size_t nws = gla_decay_fwd_workspace_bytes(n.B, n.T, n.H, n.HK, n.DK, n.DV, dt, (bool)lengths);
    const size_t nst = residual ? gla_decay_states_bytes(n.B, n.T, n.H, n.HK, n.DK, n.DV, dt) : 0;
    ChunkOut r{at::empty_like(h0), dense_like(v), Tensor()};
    if (residual) r.states = at::empty({n.B, (int64_t)nst / n.B}, v.options().dtype(at::kByte));
    Tensor ws;
    if (nws) ws = bytes_like(nws, v);
    const auto strides = decay_strides(a, v, k, q);
    check("gla_decay_fwd",
          gla_decay_fwd(stream_of(v), n.B, n.T, n.H, n.HK, n.DK, n.DV, dt, code(h0), strides.data(), h0.data_ptr(),
                        (const float *)a.data_ptr(), v.data_ptr(), k.data_ptr(), q.data_ptr(), lengths_of(lengths), r.hT.data_ptr(),
                        r.out.data_ptr(), nst ? r.states.data_ptr() : nullptr, nws ? ws.data_ptr() : nullptr, nws));
    return r;
}

variable_list decay_backward(const Tensor &states, const Tensor &a, const Tensor &v, const Tensor &k, const Tensor &q,
                             const std::optional<Tensor> &lengths, const Tensor &dhT, const Tensor &dout)
{
    const c10::DeviceGuard guard(v.device());
    const DecayDims n = decay_dims(v, k);
    const gla_dtype dt = code(v);
    const bool constant = a.dim() == 1;
    const size_t nws = gla_decay_bwd_workspace_bytes(n.B, n.T, n.H, n.HK, n.DK, n.DV, dt, constant, (bool)lengths);
    Tensor ws;
    if (nws) ws = bytes_like(nws, v);
    Tensor dh0 = at::empty_like(dhT), da = dense_like(a), dv = dense_like(v), dk = dense_like(k), dq = dense_like(q);
    const auto strides = decay_strides(a, v, k, q);
    check("gla_decay_bwd",
          gla_decay_bwd(stream_of(v), n.B, n.T, n.H, n.HK, n.DK, n.DV, dt, code(dhT), constant, strides.data(), (const float *)a.data_ptr(),
                        v.data_ptr(), k.data_ptr(), q.data_ptr(), lengths_of(lengths), states.data_ptr(), dhT.data_ptr(),
                        dout.data_ptr(), dh0.data_ptr(), (float *)da.data_ptr(), dv.data_ptr(), dk.data_ptr(), dq.data_ptr(),
                        nws ? ws.data_ptr() : nullptr, nws));
    return {dh0, da, dv, dk, dq};
}

struct DecayBackward : torch::autograd::Function<DecayBackward> {
    static variable_list forward(AutogradContext *, const Tensor &states, const Tensor &a, const Tensor &v, const Tensor &k,
                                 const Tensor &q, const std::optional<Tensor> &lengths, const Tensor &dhT, const Tensor &dout)
    {
        return decay_backward(states, a, v, k, q, lengths, dhT, dout);
    }
    static variable_list backward(AutogradContext *, variable_list) { no_double_backward("chunk_decay"); }
};

struct Decay : torch::autograd::Function<Decay> {
    static variable_list forward(AutogradContext *ctx, const Tensor &h0, const Tensor &a, const Tensor &v, const Tensor &k,
                                 const Tensor &q, const std::optional<Tensor> &lengths)
    {
        ChunkOut r = decay_forward(h0, a, v, k, q, lengths, true);
        ctx->save_for_backward({r.states, a, v, k, q, lengths.value_or(Tensor())});
        ctx->saved_data["hidden"] = (int64_t)h0.scalar_type();
        ctx->set_materialize_grads(false);
        return {r.hT, r.out};
    }
    static variable_list backward(AutogradContext *ctx, variable_list d)
    {
        variable_list s = ctx->get_saved_variables();
        // rows keep their strides; what a saved-tensor hook hands back in a layout that the kernels do not take is copied
        for (size_t i = 2; i < 5; ++i)
            if (s[i].defined() && !rows_on_gpu(s[i])) s[i] = s[i].clone(at::MemoryFormat::Contiguous);
        if (!s[0].is_contiguous() || !on_16_bytes(s[0])) s[0] = s[0].clone(at::MemoryFormat::Contiguous);
        if (s[5].defined() && !s[5].is_contiguous()) s[5] = s[5].contiguous();
        const std::optional<Tensor> lengths = s[5].defined() ? std::optional<Tensor>(s[5]) : std::nullopt;
        check_saved(decay_rows(s[1], s[2], s[3], s[4], lengths));
        const DecayDims n = decay_dims(s[2], s[3]);
        check_saved(holds(s[0], gla_decay_states_bytes(n.B, n.T, n.H, n.HK, n.DK, n.DV, code(s[2])), s[2]));
        Tensor dhT = cotangent(d[0], decay_state_sizes(s[2], s[3]), (at::ScalarType)ctx->saved_data["hidden"].toInt(), s[2]);
        Tensor dout = cotangent(d[1], s[2].sizes(), s[2].scalar_type(), s[2]);
        if (!transforms_active())
            for (Tensor *t : {&dhT, &dout})
                if (!on_16_bytes(*t)) *t = t->clone();
        variable_list r =
            transforms_active() ? python_rule("gla_jax_amd.decay", "_ChunkDecayBwd", s[0], s[1], s[2], s[3], s[4], lengths, dhT, dout)
            : at::GradMode::is_enabled() ? DecayBackward::apply(s[0], s[1], s[2], s[3], s[4], lengths, dhT, dout)
                                         : decay_backward(s[0], s[1], s[2], s[3], s[4], lengths, dhT, dout);
        r.emplace_back();
        return r;
    }
};

// ---- module -------------------------------------------------------------------------------------
typedef std::optional<std::vector<Tensor>> Result;       // none: not for this path

// A tracer records an autograd function of Python's as a call of it; of a native call it would record the buffers that are
// allocated here, and replay those.
bool traced() { return at::tracer::impl::is_dispatch_enabled(); }

Result chunk(const Tensor &h0, const Tensor &g, const Tensor &v, const Tensor &k, const Tensor &q, int64_t size)
{
    if (traced() || !canonical(h0, g, v, k, q) || size <= 0 || (size & (size - 1)) || dims_of(k).T % size) return std::nullopt;
    if (wants_grad(h0, g, v, k, q)) return Chunk::apply(h0, g, v, k, q, size);
    ChunkOut r = chunk_forward(h0, g, v, k, q, size, false);
    return std::vector<Tensor>{r.hT, r.out};
}

Result recurrent(const Tensor &h0, const Tensor &g, const Tensor &v, const Tensor &k, const Tensor &q, bool reverse,
                 bool out_fp32)
{
    if (traced() || !canonical(h0, g, v, k, q) || k.size(-1) < 16) return std::nullopt;
    if (wants_grad(h0, g, v, k, q)) return Recurrent::apply(h0, g, v, k, q, reverse, out_fp32);
    auto [hT, out] = recurrent_forward(h0, g, v, k, q, reverse, out_fp32);
    return std::vector<Tensor>{hT, out};
}

bool plain_f32(const Tensor &t) { return dense_on_gpu(t) && t.scalar_type() == at::kFloat; }

std::optional<Tensor> cumsum(const Tensor &src, int64_t axis, const std::optional<Tensor> &init, bool reverse)
{
    const int64_t n = src.dim();
    if (!plain_f32(src) || axis < 0 || axis >= n) return std::nullopt;
    int64_t outer = 1, inner = 1;
    for (int64_t i = 0; i < axis; ++i) outer *= src.size(i);
    for (int64_t i = axis + 1; i < n; ++i) inner *= src.size(i);
    if (outer < 1 || outer > 65535) return std::nullopt;
    if (init) {
        if (!plain_f32(*init) || init->dim() != n - 1 || init->device() != src.device()) return std::nullopt;
        for (int64_t i = 0; i < n - 1; ++i)
            if (init->size(i) != src.size(i < axis ? i : i + 1)) return std::nullopt;
    }
    const c10::DeviceGuard guard(src.device());
    Tensor dst = at::empty_like(src), ws;
    const size_t nws = gla_cumsum_workspace_bytes(outer, src.size(axis), inner);
    if (nws) ws = bytes_like(nws, src);
    check("gla_cumsum_f32", gla_cumsum_f32_ws(stream_of(src), (const float *)src.data_ptr(),
                                              init ? (const float *)init->data_ptr() : nullptr, (float *)dst.data_ptr(), outer,
                                              src.size(axis), inner, reverse, nws ? ws.data_ptr() : nullptr, nws));
    return dst;
}

std::optional<std::pair<Tensor, Tensor>> rnn(const Tensor &a, const Tensor &b, const std::optional<Tensor> &ia,
                                             const std::optional<Tensor> &ib, bool reverse)
{
    const int64_t n = b.dim();
    if (!plain_f32(a) || !plain_f32(b) || (n != 3 && n != 4) || a.dim() != n - 1 || a.device() != b.device()) return std::nullopt;
    for (int64_t i = 0; i < n - 1; ++i)
        if (a.size(i) != b.size(i)) return std::nullopt;
    if ((bool)ia != (bool)ib) return std::nullopt;
    const int64_t B = n == 4 ? b.size(0) : 1, T = b.size(n - 3), K = b.size(n - 2), V = b.size(n - 1);
    // the initial pair is read as B rows of K (and K x V) whatever its shape: the number of values is what has to fit
    if (ia && (!plain_f32(*ia) || !plain_f32(*ib) || ia->numel() != B * K || ib->numel() != B * K * V ||
               ia->device() != b.device() || ib->device() != b.device()))
        return std::nullopt;
    const c10::DeviceGuard guard(b.device());
    Tensor oa = at::empty_like(a), ox = at::empty_like(b);
    check("gla_rnn_scan_f32",
          gla_rnn_scan_f32(stream_of(b), (const float *)a.data_ptr(), (const float *)b.data_ptr(),
                           ia ? (const float *)ia->data_ptr() : nullptr, ib ? (const float *)ib->data_ptr() : nullptr,
                           (float *)oa.data_ptr(), (float *)ox.data_ptr(), B, T, K, V, reverse));
    return std::make_pair(oa, ox);
}

// [B,T,..] rows, or [T,..] as those of one sequence
Result decay(const Tensor &h0, const Tensor &a, const Tensor &v, const Tensor &k, const Tensor &q, const std::optional<Tensor> &lengths)
{
    if (traced() || !decay_rows(a, v, k, q, lengths) || !dense_on_gpu(h0) || !on_16_bytes(h0) || h0.device() != v.device() || !known(h0.scalar_type()) ||
        h0.sizes() != at::IntArrayRef(decay_state_sizes(v, k)))
        return std::nullopt;
    if (wants_grad(h0, a, v, k, q)) return Decay::apply(h0, a, v, k, q, lengths);
    ChunkOut r = decay_forward(h0, a, v, k, q, lengths, false);
    return std::vector<Tensor>{r.hT, r.out};
}

bool index_array(const std::optional<Tensor> &t, at::IntArrayRef sizes, const Tensor &like, at::ScalarType type)
{
    return !t || (dense_on_gpu(*t) && t->sizes() == sizes && t->device() == like.device() && t->scalar_type() == type);
}
at::ScalarType index_type(const std::optional<Tensor> &x, const std::optional<Tensor> &y)
{
    const at::ScalarType t = x ? x->scalar_type() : y ? y->scalar_type() : at::kLong;
    return t == at::kInt ? at::kInt : at::kLong;
}
bool has_tangent(at::ArrayRef<Tensor> arrays)
{
    for (const Tensor &t : arrays)
        if (t._fw_grad(/*level=*/0).defined()) return true;
    return false;
}
bool takes_gradient(at::ArrayRef<Tensor> arrays)
{
    for (const Tensor &t : arrays)
        if (at::GradMode::is_enabled() && t.requires_grad()) return true;
    return has_tangent(arrays);
}

// States that a call has updated in place count as a new version: autograd then refuses to use what it saved of the old one.  (What
// inference mode makes has no version.)
void updated(const Tensor &states)
{
    if (!states.is_inference()) states.unsafeGetTensorImpl()->bump_version();
}

std::optional<Tensor> decay_step(const Tensor &states, const Tensor &a, const Tensor &v, const Tensor &k, const Tensor &q,
                                 const std::optional<Tensor> &slots, const std::optional<Tensor> &parents)
{
    if (traced() || !dense_on_gpu(states) || states.dim() != 4 || !known(states.scalar_type()) || takes_gradient({states, a, v, k, q}))
        return std::nullopt;
    if (!rows_on_gpu(v) || !rows_on_gpu(k) || !rows_on_gpu(q) || v.dim() != 3 || k.dim() != 3 || q.sizes() != k.sizes()) return std::nullopt;
    const int64_t B = v.size(0), H = v.size(1), DV = v.size(2), HK = k.size(1), DK = k.size(2), N = states.size(0);
    if (B < 1 || H < 1 || N < 1 || HK < 1 || H % HK || k.size(0) != B || states.size(1) != H || states.size(2) != DK || states.size(3) != DV)
        return std::nullopt;
    if (!known(v.scalar_type()) || k.scalar_type() != v.scalar_type() || q.scalar_type() != v.scalar_type()) return std::nullopt;
    if (!a.is_cuda() || a.layout() != at::kStrided || a.scalar_type() != at::kFloat || a.size(-1) != H || a.dim() > 2 || (a.dim() == 2 && a.size(0) != B))
        return std::nullopt;
    for (const Tensor *t : {&a, &v, &k, &q})
        if (t->device() != states.device()) return std::nullopt;
    const at::ScalarType type = index_type(slots, parents);
    const int64_t W = parents && parents->dim() == 2 ? parents->size(1) : 0;
    if (!index_array(slots, {B}, states, type) || (parents && (W < 1 || !index_array(parents, {B / W, W}, states, type) || B % W)) ||
        (!slots && N < B) || W > GLA_MOST_BEAMS || DK % 16 || DV % 16 || DK > 256 || DV > 256 || !on_16_bytes(states))
        return std::nullopt;
    const c10::DeviceGuard guard(states.device());
    Tensor out = dense_like(v);
    const int64_t strides[8] = {a.dim() == 2 ? a.stride(0) : 0, a.stride(-1), B > 1 ? v.stride(0) : 0, H > 1 ? v.stride(1) : 0,
                                B > 1 ? k.stride(0) : 0, HK > 1 ? k.stride(1) : 0, B > 1 ? q.stride(0) : 0, HK > 1 ? q.stride(1) : 0};
    const int rc = gla_decay_step(stream_of(states), N, B, H, HK, DK, DV, W, code(v), code(states), type == at::kLong, strides,
                                  (const float *)a.data_ptr(), v.data_ptr(), k.data_ptr(), q.data_ptr(), slots ? slots->data_ptr() : nullptr,
                                  parents ? parents->data_ptr() : nullptr, states.data_ptr(), out.data_ptr());
    check("gla_decay_step", rc);
    updated(states);
    return out;
}

// ---- beam search ----------------------------------------------------------------------------------
Result beam_select(const Tensor &logits, const Tensor &scores, const std::optional<int64_t> &wanted, const std::optional<Tensor> &finished, int64_t eos)
{
    const int64_t n = logits.dim();
    if (traced() || n < 2 || !logits.is_cuda() || logits.layout() != at::kStrided || logits.stride(-1) != 1 || !known(logits.scalar_type()) ||
        !plain_f32(scores) || scores.dim() != n - 1 || scores.device() != logits.device() || has_tangent({logits, scores}))
        return std::nullopt;
    const int64_t W = logits.size(-2), V = logits.size(-1), row = W > 1 ? logits.stride(-2) : V;
    int64_t G = 1;
    std::vector<int64_t> sizes;
    // rows one distance apart from each other, whatever axes lie in front
    int64_t step = W * row;
    for (int64_t i = n - 3; i >= 0; --i) {
        if (logits.size(i) > 1 && logits.stride(i) != step) return std::nullopt;
        step *= logits.size(i);
        G *= logits.size(i);
    }
    for (int64_t i = 0; i + 2 < n; ++i) sizes.push_back(logits.size(i));
    for (int64_t i = 0; i + 1 < n; ++i)
        if (scores.size(i) != logits.size(i)) return std::nullopt;
    if (finished && (!dense_on_gpu(*finished) || finished->scalar_type() != at::kBool || finished->sizes() != scores.sizes() ||
                     finished->device() != logits.device()))
        return std::nullopt;
    const int64_t num = wanted.value_or(W);
    if (finished && (eos < 0 || eos >= V)) return std::nullopt;
    const size_t nws = row < V ? 0 : gla_beam_select_workspace_bytes(G, W, V, num);
    if (nws == 0) return std::nullopt;
    const c10::DeviceGuard guard(logits.device());
    sizes.push_back(num);
    Tensor best = at::empty(sizes, scores.options()), parents = at::empty(sizes, scores.options().dtype(at::kLong)),
           tokens = at::empty(sizes, scores.options().dtype(at::kLong)), ws = bytes_like(nws, logits);
    const int rc = gla_beam_select(stream_of(logits), G, W, V, num, code(logits), row, logits.data_ptr(), (const float *)scores.data_ptr(),
                                   finished ? finished->data_ptr() : nullptr, eos, (float *)best.data_ptr(), (int64_t *)parents.data_ptr(),
                                   (int64_t *)tokens.data_ptr(), ws.data_ptr(), nws);
    check("gla_beam_select", rc);
    return std::vector<Tensor>{best, parents, tokens};
}

bool reorder(const Tensor &states, const Tensor &parents, const std::optional<Tensor> &slots)
{
    if (traced() || !dense_on_gpu(states) || states.dim() < 1 || states.numel() == 0 || takes_gradient({states}) || parents.dim() != 2)
        return false;
    const at::ScalarType type = index_type(slots, parents);
    const int64_t G = parents.size(0), W = parents.size(1), N = states.size(0);
    if (!index_array(parents, parents.sizes(), states, type) || !index_array(slots, parents.sizes(), states, type) || G * W == 0 ||
        W > GLA_MOST_BEAMS || (!slots && N < G * W))
        return false;
    const c10::DeviceGuard guard(states.device());
    const int rc = gla_reorder_states(stream_of(states), N, G, W, states.numel() / N * (int64_t)states.element_size(), type == at::kLong,
                                      parents.data_ptr(), slots ? slots->data_ptr() : nullptr, states.data_ptr());
    check("gla_reorder_states", rc);
    updated(states);
    return true;
}

}  // namespace

PYBIND11_MODULE(_gla_torch, m)
{
    gla_error = py::object(py::module_::import("gla_jax_amd._lib").attr("GlaError")).release().ptr();
    typedef py::call_guard<py::gil_scoped_release> NoGil;
    m.def("chunk", &chunk, NoGil());
    m.def("recurrent", &recurrent, NoGil());
    m.def("cumsum", &cumsum, NoGil());
    m.def("rnn", &rnn, NoGil());
    m.def("decay", &decay, NoGil());
    m.def("decay_step", &decay_step, NoGil());
    m.def("beam_select", &beam_select, NoGil());
    m.def("reorder", &reorder, NoGil());
}
