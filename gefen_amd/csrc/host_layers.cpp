// Host side of a layer's training operators: attention, the norm of the residual stream and
// dropout, each with its autograd function.  The kernels are reached through the C ABI, as in
// host_training.cpp.

#include <cmath>
#include <cstring>
#include <functional>
#include <initializer_list>
#include <optional>
#include <vector>

#include <c10/hip/HIPGraphsC10Utils.h>

#include "host_common.h"

namespace {

using namespace gefen_host;

struct Library {
    decltype(&gefen_attention_forward_workspace_size) attention_forward_workspace;
    decltype(&gefen_attention_forward) attention_forward;
    decltype(&gefen_attention_backward_workspace_size) attention_workspace;
    decltype(&gefen_attention_backward) attention_backward;
    decltype(&gefen_rms_norm_forward) rms_forward;
    decltype(&gefen_rms_norm_backward_workspace_size) rms_workspace;
    decltype(&gefen_rms_norm_backward) rms_backward;
    decltype(&gefen_dropout) dropout;
};
Library lib{};

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

const at::Tensor kNone;
// An undefined tensor as autograd functions take it, and back.
using Maybe = std::optional<at::Tensor>;
Maybe maybe(const at::Tensor& t) { return t.defined() ? Maybe(t) : std::nullopt; }
const at::Tensor& given(const Maybe& t) { return t ? *t : kNone; }

// An optional tensor argument.
const at::Tensor& optional_tensor(py::handle o, const char* name) {
    return o.is_none() ? kNone : tensor_of(o, name);
}

void floating(const at::Tensor& t, const char* name) {
    if (dtype_code(t) < 0)
        throw py::value_error(std::string("Expected ") + name + " to be float32, float16 or bfloat16, got " +
                              c10::toString(t.scalar_type()));
}
void same_dtype(const at::Tensor& t, const char* name, const at::Tensor& first, const char* of) {
    if (t.scalar_type() != first.scalar_type())
        throw py::value_error(std::string("Expected ") + name + " of " + of + "'s dtype " +
                              c10::toString(first.scalar_type()) + ", got " + c10::toString(t.scalar_type()));
}
// An operand that autograd follows.
void operand(const at::Tensor& t, const char* name, const at::Tensor& first, const char* of) {
    plain_on(t, name, first);
    no_tangent(t, name);
    floating(t, name);
    same_dtype(t, name, first, of);
}
// Whole numbers on the device.
void indices(const at::Tensor& t, const char* name, const at::Tensor& first) {
    plain_on(t, name, first);
    if (t.scalar_type() != at::kInt && t.scalar_type() != at::kLong)
        throw py::value_error(std::string("Expected ") + name + " to be int32 or int64, got " +
                              c10::toString(t.scalar_type()));
    if (t.dim() != 1) throw py::value_error(std::string("Expected ") + name + " to be 1D, got dim=" + std::to_string(t.dim()));
}

bool wants(const at::Tensor& t) { return t.defined() && t.requires_grad(); }

// Raises where a call under graph capture would join a graph of autograd that was recorded outside,
// on the default stream: the backward pass waits for the stream of each node that it reaches, a
// captured one cannot wait for that one, and torch's engine then ends the process.
void no_eager_graph(std::initializer_list<std::reference_wrapper<const at::Tensor>> operands) {
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    for (const at::Tensor& t : operands) {
        if (!wants(t)) continue;
        const auto node = t.grad_fn() ? t.grad_fn() : torch::autograd::impl::try_get_grad_accumulator(t);
        if (!node) continue;
        const auto stream = node->stream();
        if (stream && stream->id() == c10::hip::getDefaultHIPStream(t.device().index()).id())
            throw std::runtime_error(
                "Expected no autograd graph from outside the capture: drop what was computed from these tensors on the "
                "default stream, or warm up on another one.");
    }
}

// A tensor as a backward pass finds it, which hooks of saved tensors may have replaced.
at::Tensor found(const at::Tensor& t, c10::IntArrayRef sizes, at::ScalarType type, const at::Tensor& first) {
    TORCH_CHECK(t.defined() && t.sizes() == sizes && t.scalar_type() == type && t.device() == first.device(),
                "Expected a saved tensor to come back with its shape, dtype and device.");
    return t;
}

// What the last dimension holds, one after the other.
at::Tensor rows_dense(const at::Tensor& t) {
    const at::Tensor s = as_stored(t);
    return s.size(-1) <= 1 || s.stride(-1) == 1 ? s : s.contiguous();
}

int64_t bits_of(double v) {
    int64_t b;
    std::memcpy(&b, &v, 8);
    return b;
}
double double_of(int64_t b) {
    double v;
    std::memcpy(&v, &b, 8);
    return v;
}

// ------------------------------------------------------------------ attention

struct AttentionCall {
    at::Tensor q, k, v, go;
    gefen_attention_task t{};

    AttentionCall(const at::Tensor& query, const at::Tensor& key, const at::Tensor& value, const at::Tensor& lengths,
                  const at::Tensor& offsets, bool causal, double scale)
        : q(rows_dense(query)), k(rows_dense(key)), v(rows_dense(value)) {
        t.query = q.data_ptr();
        t.key = k.data_ptr();
        t.value = v.data_ptr();
        const bool packed = offsets.defined();
        t.batch = packed ? 1 : q.size(0);
        t.queries = q.size(-3);
        t.keys = k.size(-3);
        t.heads = q.size(-2);
        t.kv_heads = k.size(-2);
        t.width = q.size(-1);
        strides(q, t.query_strides);
        strides(k, t.key_strides);
        strides(v, t.value_strides);
        if (lengths.defined()) {
            t.key_lengths = lengths.data_ptr();
            t.lengths_int64 = lengths.scalar_type() == at::kLong;
        }
        if (packed) {
            t.offsets = offsets.data_ptr();
            t.offsets_int64 = offsets.scalar_type() == at::kLong;
            t.sequences = offsets.size(0) - 1;
        }
        t.scale = scale;
        t.dtype = dtype_code(q);
        t.causal = causal;
    }
    static void strides(const at::Tensor& x, int64_t* out) {
        out[0] = x.dim() == 4 ? x.stride(0) : 0;
        out[1] = x.stride(-3);
        out[2] = x.stride(-2);
    }
};

at::Tensor attention_forward(const at::Tensor& query, const at::Tensor& key, const at::Tensor& value,
                             const at::Tensor& lengths, const at::Tensor& offsets, bool causal, double scale,
                             at::Tensor* lse) {
    c10::DeviceGuard guard(query.device());
    AttentionCall c(query, key, value, lengths, offsets, causal, scale);
    at::Tensor out = at::empty(query.sizes(), query.options().requires_grad(false));
    c.t.out = out.data_ptr();
    if (lse) {
        *lse = at::empty({c.t.batch * c.t.queries * c.t.heads}, query.options().dtype(at::kFloat).requires_grad(false));
        c.t.lse = floats(*lse);
    }
    at::Tensor ws;
    const size_t bytes = lib.attention_forward_workspace(&c.t);
    if (bytes) ws = bytes_on(query, bytes);
    check(lib.attention_forward(&c.t, data(ws), bytes, stream_of(query)));
    return out;
}

class Attention : public torch::autograd::Function<Attention> {
   public:
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& query, const at::Tensor& key,
                              const at::Tensor& value, const Maybe& lengths_, const Maybe& offsets_, bool causal,
                              double scale, bool need_q, bool need_kv) {
        ctx->set_materialize_grads(false);
        const at::Tensor &lengths = given(lengths_), &offsets = given(offsets_);
        at::Tensor lse;
        at::Tensor out = attention_forward(query, key, value, lengths, offsets, causal, scale, &lse);
        ctx->save_for_backward({query, key, value, lengths, offsets, out, lse});
        ctx->saved_data["options"] =
            std::vector<int64_t>{causal,         bits_of(scale), need_q,
                                 need_kv,        key.size(-3),   key.size(-2),
                                 lengths.defined() ? static_cast<int64_t>(lengths.scalar_type()) : 0,
                                 offsets.defined() ? static_cast<int64_t>(offsets.scalar_type()) : 0,
                                 offsets.defined() ? offsets.size(0) : 0};
        return out;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        TORCH_CHECK(!c10::GradMode::is_enabled(), "attention can be differentiated once only");
        at::Tensor gq, gk, gv;
        if (grads[0].defined()) {
            const std::vector<int64_t> o = ctx->saved_data["options"].toIntVector();
            const auto saved = ctx->get_saved_variables();
            const at::Tensor& go = grads[0];
            const at::ScalarType type = go.scalar_type();
            auto sizes = go.sizes().vec();
            const at::Tensor query = found(saved[0], sizes, type, go), out = found(saved[5], sizes, type, go).contiguous();
            const at::Tensor lse = found(saved[6], {query.numel() / query.size(-1)}, at::kFloat, go).contiguous();
            sizes[sizes.size() - 3] = o[4];
            sizes[sizes.size() - 2] = o[5];
            const at::Tensor key = found(saved[1], sizes, type, go), value = found(saved[2], sizes, type, go);
            at::Tensor lengths, offsets;
            if (o[6]) lengths = found(saved[3], {query.size(0)}, static_cast<at::ScalarType>(o[6]), go).contiguous();
            if (o[7]) offsets = found(saved[4], {o[8]}, static_cast<at::ScalarType>(o[7]), go).contiguous();
            c10::DeviceGuard guard(query.device());
            AttentionCall c(query, key, value, lengths, offsets, o[0], double_of(o[1]));
            c.go = rows_dense(go);
            c.t.grad_out = c.go.data_ptr();
            AttentionCall::strides(c.go, c.t.grad_out_strides);
            c.t.out = out.data_ptr();
            c.t.lse = floats(lse);
            gq = empty_grad(query, true, query.scalar_type());  // D is formed with it
            gk = empty_grad(key, o[3], key.scalar_type());
            gv = empty_grad(value, o[3], value.scalar_type());
            c.t.grad_query = data(gq);
            c.t.grad_key = data(gk);
            c.t.grad_value = data(gv);
            at::Tensor ws = bytes_on(query, lib.attention_workspace(&c.t));
            check(lib.attention_backward(&c.t, ws.data_ptr(), ws.numel(), stream_of(query)));
            if (!o[2]) gq = at::Tensor();
        }
        return {gq, gk, gv, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
    }
};

py::object attention(py::handle query_, py::handle key_, py::handle value_, py::handle lengths_, py::handle offsets_,
                     bool causal, py::object scale_) {
    need_library();
    const at::Tensor& query = tensor_of(query_, "query");
    const at::Tensor& key = tensor_of(key_, "key");
    const at::Tensor& value = tensor_of(value_, "value");
    const at::Tensor& lengths_given = optional_tensor(lengths_, "key_lengths");
    const at::Tensor& offsets_given = optional_tensor(offsets_, "offsets");
    const bool packed = offsets_given.defined();
    operand(query, "query", query, "query");
    operand(key, "key", query, "query");
    operand(value, "value", query, "query");
    const int64_t dims = packed ? 3 : 4;
    if (query.dim() != dims || key.dim() != dims || value.dim() != dims)
        throw py::value_error(packed ? "Expected packed query, key and value [tokens, heads, width]."
                                     : "Expected query, key and value [batch, tokens, heads, width].");
    if (key.sizes() != value.sizes())
        throw py::value_error("Expected value of key's shape " + shape_of(key.sizes()) + ", got " + shape_of(value.sizes()));
    if (query.size(-1) != key.size(-1))
        throw py::value_error("Expected key of query's width " + std::to_string(query.size(-1)) + ", got shape " +
                              shape_of(key.sizes()));
    if (packed ? query.size(0) != key.size(0) : query.size(0) != key.size(0))
        throw py::value_error(std::string("Expected key of as many ") + (packed ? "tokens" : "sequences") + " as query, " +
                              std::to_string(query.size(0)) + ", got shape " + shape_of(key.sizes()));
    if (query.size(-2) < 1 || key.size(-2) < 1 || query.size(-2) % key.size(-2))
        throw py::value_error("Expected query's heads to be a multiple of key's, got " + std::to_string(query.size(-2)) +
                              " and " + std::to_string(key.size(-2)));
    at::Tensor lengths, offsets;
    if (packed) {
        if (lengths_given.defined()) throw py::value_error("Expected either offsets or key_lengths.");
        indices(offsets_given, "offsets", query);
        if (offsets_given.size(0) < 1) throw py::value_error("Expected offsets of one element at least.");
        offsets = offsets_given.contiguous();
    } else if (lengths_given.defined()) {
        indices(lengths_given, "key_lengths", query);
        if (lengths_given.size(0) != query.size(0))
            throw py::value_error("Expected key_lengths of " + std::to_string(query.size(0)) + " elements, got " +
                                  std::to_string(lengths_given.size(0)));
        lengths = lengths_given.contiguous();
    }
    if (query.size(-1) < 1 || query.size(-1) > GEFEN_ATTENTION_MAX_WIDTH)
        throw py::value_error("Expected heads of width 1 to " + std::to_string(GEFEN_ATTENTION_MAX_WIDTH) + ", got " +
                              std::to_string(query.size(-1)));
    const double scale = scale_.is_none() ? 1.0 / std::sqrt(static_cast<double>(query.size(-1))) : scale_.cast<double>();
    const bool grad = c10::GradMode::is_enabled();
    const bool need_q = grad && wants(query), need_kv = grad && (wants(key) || wants(value));
    if (need_q || need_kv) {
        no_eager_graph({query, key, value});
        return wrap(Attention::apply(query, key, value, maybe(lengths), maybe(offsets), causal, scale, need_q, need_kv));
    }
    return wrap(attention_forward(query.detach(), key.detach(), value.detach(), lengths, offsets, causal, scale, nullptr));
}

// ------------------------------------------------------------------ dropout's seed

// The seed of a call: a tensor on the device, which the kernels read, or a number.
struct Seed {
    at::Tensor at;
    int64_t value = 0;
    const int64_t* pointer() const { return at.defined() ? at.data_ptr<int64_t>() : nullptr; }
};
Seed seed_of(py::handle tensor, int64_t value, const at::Tensor& first) {
    Seed s;
    s.value = value;
    if (tensor.is_none()) return s;
    s.at = tensor_of(tensor, "seed");
    plain_on(s.at, "seed", first);
    if (s.at.scalar_type() != at::kLong || s.at.numel() != 1)
        throw py::value_error("Expected seed to be an int or an int64 tensor of one element.");
    if (s.at.dim()) s.at = s.at.reshape({});
    return s;
}

// ------------------------------------------------------------------ norm of the residual stream

// A tensor [..., width] as rows with one stride.
at::Tensor as_rows(const at::Tensor& t) {
    const at::Tensor r = rows_dense(t);
    return r.dim() == 2 ? r : r.reshape({-1, r.size(-1)});
}

struct RmsOptions {
    double eps, dropout;
    int64_t seed, offset;
};

struct RmsCall {
    at::Tensor x, residual, w;
    gefen_rms_norm_task t{};

    RmsCall(const at::Tensor& x_, const at::Tensor& weight, const at::Tensor& residual_, const at::Tensor& seed,
            const RmsOptions& o)
        : x(as_rows(x_)), w(as_stored(weight).contiguous()) {
        t.x = x.data_ptr();
        t.x_row_stride = x.stride(0);
        t.weight = w.data_ptr();
        if (residual_.defined()) {
            residual = as_rows(residual_);
            t.residual = residual.data_ptr();
            t.residual_row_stride = residual.stride(0);
        }
        t.rows = x.size(0);
        t.width = x.size(1);
        t.eps = o.eps;
        t.dropout = o.dropout;
        t.seed_at = seed.defined() ? seed.data_ptr<int64_t>() : nullptr;
        t.seed = o.seed;
        t.offset = o.offset;
        t.dtype = dtype_code(x);
    }
};

at::Tensor empty_as(const at::Tensor& like, c10::IntArrayRef sizes, at::ScalarType type) {
    return at::empty(sizes, like.options().dtype(type).requires_grad(false));
}

class RmsNorm : public torch::autograd::Function<RmsNorm> {
   public:
    static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& weight,
                                 const Maybe& residual_, const Maybe& seed_, double eps, double dropout,
                                 int64_t seed_value, int64_t offset, bool need_x, bool need_r, bool need_w) {
        ctx->set_materialize_grads(false);
        const at::Tensor &residual = given(residual_), &seed = given(seed_);
        c10::DeviceGuard guard(x.device());
        RmsCall c(x, weight, residual, seed, {eps, dropout, seed_value, offset});
        at::Tensor y = empty_as(x, x.sizes(), x.scalar_type()), s;
        at::Tensor rstd = empty_as(x, {c.t.rows}, at::kFloat);
        c.t.y = y.data_ptr();
        c.t.rstd = floats(rstd);
        if (residual.defined()) {
            s = empty_as(x, x.sizes(), x.scalar_type());
            c.t.sum = s.data_ptr();
        }
        check(lib.rms_forward(&c.t, stream_of(x)));
        ctx->save_for_backward({s.defined() ? s : x, weight, rstd, seed});
        ctx->saved_data["options"] = std::vector<int64_t>{bits_of(eps), bits_of(dropout), seed_value, offset,
                                                          need_x,       need_r,           need_w,     seed.defined()};
        if (s.defined()) return {y, s};
        return {y};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        TORCH_CHECK(!c10::GradMode::is_enabled(), "rms_norm can be differentiated once only");
        at::Tensor gx, gr, gw;
        const bool two = grads.size() > 1;
        if (grads[0].defined() || (two && grads[1].defined())) {
            const std::vector<int64_t> o = ctx->saved_data["options"].toIntVector();
            const bool need_x = o[4], need_r = o[5], need_w = o[6];
            const auto saved = ctx->get_saved_variables();
            const at::Tensor& first = grads[0].defined() ? grads[0] : grads[1];
            const at::ScalarType type = first.scalar_type();
            const at::Tensor s = found(saved[0], first.sizes(), type, first);
            const at::Tensor weight = found(saved[1], {s.size(-1)}, type, first);
            at::Tensor seed;
            if (o[7]) seed = found(saved[3], {}, at::kLong, first);
            const at::Tensor rstd = found(saved[2], {s.numel() / s.size(-1)}, at::kFloat, first).contiguous();
            c10::DeviceGuard guard(s.device());
            RmsCall c(s, weight, at::Tensor(), seed, {double_of(o[0]), double_of(o[1]), o[2], o[3]});
            const at::Tensor gy = as_rows(grads[0].defined() ? grads[0] : at::zeros(s.sizes(), s.options()));
            at::Tensor gs;
            c.t.grad_y = gy.data_ptr();
            c.t.grad_y_row_stride = gy.stride(0);
            if (two && grads[1].defined()) {
                gs = as_rows(grads[1]);
                c.t.grad_sum = gs.data_ptr();
                c.t.grad_sum_row_stride = gs.stride(0);
            }
            c.t.rstd = floats(rstd);
            // without dropout x and the residual have the same gradient
            const bool drop = c.t.dropout > 0.0;
            if (need_x && drop) gx = empty_as(s, s.sizes(), s.scalar_type());
            if (need_r || (need_x && !drop)) gr = empty_as(s, s.sizes(), s.scalar_type());
            at::Tensor ws;
            if (need_w) {
                gw = empty_as(weight, weight.sizes(), weight.scalar_type());
                ws = bytes_on(s, lib.rms_workspace(&c.t));
            }
            c.t.grad_x = data(gx);
            c.t.grad_residual = data(gr);
            c.t.grad_weight = data(gw);
            check(lib.rms_backward(&c.t, data(ws), ws.defined() ? ws.numel() : 0, stream_of(s)));
            if (need_x && !drop) gx = gr;
            if (!need_r) gr = at::Tensor();
        }
        variable_list out(11);
        out[0] = gx;
        out[1] = gw;
        out[2] = gr;
        return out;
    }
};

// The operands of rms_norm and rms_norm_quantized.
void rms_operands(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& residual) {
    operand(x, "x", x, "x");
    operand(weight, "weight", x, "x");
    if (x.dim() < 1) throw py::value_error("Expected x of one dimension at least.");
    if (weight.dim() != 1 || weight.size(0) != x.size(-1))
        throw py::value_error("Expected weight of shape (" + std::to_string(x.size(-1)) + "), got " + shape_of(weight.sizes()));
    if (x.size(-1) < 1 || x.size(-1) > GEFEN_RMS_MAX_WIDTH)
        throw py::value_error("Expected rows of 1 to " + std::to_string(GEFEN_RMS_MAX_WIDTH) + " elements, got shape " +
                              shape_of(x.sizes()));
    if (!residual.defined()) return;
    operand(residual, "residual", x, "x");
    if (residual.sizes() != x.sizes())
        throw py::value_error("Expected residual of x's shape " + shape_of(x.sizes()) + ", got " + shape_of(residual.sizes()));
}

py::object rms_norm(py::handle x_, py::handle weight_, py::handle residual_, double eps, double dropout,
                    py::handle seed_, int64_t seed_value, int64_t offset) {
    need_library();
    const at::Tensor& x = tensor_of(x_, "x");
    const at::Tensor& weight = tensor_of(weight_, "weight");
    const at::Tensor& residual = optional_tensor(residual_, "residual");
    rms_operands(x, weight, residual);
    const Seed seed = seed_of(seed_, seed_value, x);
    const bool grad = c10::GradMode::is_enabled();
    const bool need_x = grad && wants(x), need_w = grad && wants(weight), need_r = grad && wants(residual);
    if (need_x || need_w || need_r) {
        no_eager_graph({x, weight, residual});
        const variable_list out = RmsNorm::apply(x, weight, maybe(residual), maybe(seed.at), eps, dropout, seed.value,
                                                 offset, need_x, need_r, need_w);
        if (out.size() > 1) return py::make_tuple(wrap(out[0]), wrap(out[1]));
        return wrap(out[0]);
    }
    c10::DeviceGuard guard(x.device());
    RmsCall c(x.detach(), weight.detach(), residual.defined() ? residual.detach() : residual, seed.at,
              {eps, dropout, seed.value, offset});
    at::Tensor y = empty_as(x, x.sizes(), x.scalar_type()), s;
    c.t.y = y.data_ptr();
    if (residual.defined()) {
        s = empty_as(x, x.sizes(), x.scalar_type());
        c.t.sum = s.data_ptr();
    }
    check(lib.rms_forward(&c.t, stream_of(x)));
    if (s.defined()) return py::make_tuple(wrap(y), wrap(s));
    return wrap(y);
}

py::object rms_norm_quantized(py::handle x_, py::handle weight_, py::handle residual_, double eps, bool e5m2) {
    need_library();
    const at::Tensor& x = tensor_of(x_, "x");
    const at::Tensor& weight = tensor_of(weight_, "weight");
    const at::Tensor& residual = optional_tensor(residual_, "residual");
    rms_operands(x, weight, residual);
    if (c10::GradMode::is_enabled() && (wants(x) || wants(weight) || wants(residual)))
        throw py::value_error("Expected no gradient to be wanted of an 8-bit output: call it under torch.no_grad().");
    c10::DeviceGuard guard(x.device());
    RmsCall c(x.detach(), weight.detach(), residual.defined() ? residual.detach() : residual, at::Tensor(),
              {eps, 0.0, 0, 0});
    at::Tensor q = empty_as(x, x.sizes(), e5m2 ? at::kFloat8_e5m2 : at::kFloat8_e4m3fn), s;
    at::Tensor scales = empty_as(x, x.sizes().slice(0, x.dim() - 1), at::kFloat);
    c.t.y = q.data_ptr();
    c.t.scales = floats(scales);
    c.t.out = e5m2 ? GEFEN_RMS_E5M2 : GEFEN_RMS_E4M3;
    if (residual.defined()) {
        s = empty_as(x, x.sizes(), x.scalar_type());
        c.t.sum = s.data_ptr();
    }
    check(lib.rms_forward(&c.t, stream_of(x)));
    if (s.defined()) return py::make_tuple(wrap(q), wrap(scales), wrap(s));
    return py::make_tuple(wrap(q), wrap(scales));
}

// ------------------------------------------------------------------ dropout

at::Tensor dropout_run(const at::Tensor& x_, const at::Tensor& residual_, double p, const at::Tensor& seed,
                       int64_t seed_value, int64_t offset) {
    c10::DeviceGuard guard(x_.device());
    const at::Tensor x = as_stored(x_).contiguous();
    const at::Tensor residual = residual_.defined() ? as_stored(residual_).contiguous() : residual_;
    at::Tensor y = empty_as(x, x.sizes(), x.scalar_type());
    check(lib.dropout(x.data_ptr(), data(residual), y.data_ptr(), x.numel(), dtype_code(x), p,
                      seed.defined() ? seed.data_ptr<int64_t>() : nullptr, seed_value, offset, stream_of(x)));
    return y;
}

class DropoutFunction : public torch::autograd::Function<DropoutFunction> {
   public:
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const Maybe& residual_, const Maybe& seed_,
                              double p, int64_t seed_value, int64_t offset, bool need_x, bool need_r) {
        ctx->set_materialize_grads(false);
        const at::Tensor &residual = given(residual_), &seed = given(seed_);
        ctx->save_for_backward({seed});
        ctx->saved_data["options"] = std::vector<int64_t>{bits_of(p), seed_value, offset, need_x, need_r, seed.defined()};
        return dropout_run(x, residual, p, seed, seed_value, offset);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        TORCH_CHECK(!c10::GradMode::is_enabled(), "dropout can be differentiated once only");
        variable_list out(8);
        if (grads[0].defined()) {
            const std::vector<int64_t> o = ctx->saved_data["options"].toIntVector();
            if (o[3]) {
                at::Tensor seed;
                if (o[5]) seed = found(ctx->get_saved_variables()[0], {}, at::kLong, grads[0]);
                out[0] = dropout_run(grads[0], at::Tensor(), double_of(o[0]), seed, o[1], o[2]);
            }
            if (o[4]) out[1] = grads[0];
        }
        return out;
    }
};

py::object dropout(py::handle x_, py::handle residual_, double p, py::handle seed_, int64_t seed_value, int64_t offset) {
    need_library();
    const at::Tensor& x = tensor_of(x_, "x");
    const at::Tensor& residual = optional_tensor(residual_, "residual");
    operand(x, "x", x, "x");
    if (residual.defined()) {
        operand(residual, "residual", x, "x");
        if (residual.sizes() != x.sizes())
            throw py::value_error("Expected residual of x's shape " + shape_of(x.sizes()) + ", got " +
                                  shape_of(residual.sizes()));
    }
    const Seed seed = seed_of(seed_, seed_value, x);
    const bool grad = c10::GradMode::is_enabled();
    const bool need_x = grad && wants(x), need_r = grad && wants(residual);
    if (need_x || need_r) {
        no_eager_graph({x, residual});
        return wrap(DropoutFunction::apply(x, maybe(residual), maybe(seed.at), p, seed.value, offset, need_x, need_r));
    }
    return wrap(dropout_run(x.detach(), residual.defined() ? residual.detach() : residual, p, seed.at, seed.value, offset));
}

}  // namespace

void bind_layers(const py::dict& addresses) {
    auto at = [&](const char* name) { return addresses[name].cast<uintptr_t>(); };
    lib.attention_forward_workspace =
        reinterpret_cast<decltype(lib.attention_forward_workspace)>(at("gefen_attention_forward_workspace_size"));
    lib.attention_forward = reinterpret_cast<decltype(lib.attention_forward)>(at("gefen_attention_forward"));
    lib.attention_workspace =
        reinterpret_cast<decltype(lib.attention_workspace)>(at("gefen_attention_backward_workspace_size"));
    lib.attention_backward = reinterpret_cast<decltype(lib.attention_backward)>(at("gefen_attention_backward"));
    lib.rms_forward = reinterpret_cast<decltype(lib.rms_forward)>(at("gefen_rms_norm_forward"));
    lib.rms_workspace = reinterpret_cast<decltype(lib.rms_workspace)>(at("gefen_rms_norm_backward_workspace_size"));
    lib.rms_backward = reinterpret_cast<decltype(lib.rms_backward)>(at("gefen_rms_norm_backward"));
    lib.dropout = reinterpret_cast<decltype(lib.dropout)>(at("gefen_dropout"));
}

void register_layers(py::module_& m) {
    m.def("attention", &attention);
    m.def("rms_norm", &rms_norm);
    m.def("rms_norm_quantized", &rms_norm_quantized);
    m.def("dropout", &dropout);
}
