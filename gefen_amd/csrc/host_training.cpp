// Host side of the operators around the optimizer: the task tables of the gradient norm
// and clipping, and the linear cross entropy with its autograd function.  In C++ because
// a call on small tensors takes less time on the GPU than its Python form takes to start
// it (a training call of 48 x 1000 x 96: 160 us from Python).
//
// The kernels are reached through the C ABI (include/gefen_hip.h) of the library that
// gefen_amd/_lib.py has loaded: bind_library() receives the functions' addresses.  Built
// with the host compiler against torch's headers (no device code).

#include <Python.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <pybind11/pybind11.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>

#include <ATen/ATen.h>
#include <algorithm>
#include <cstdint>
#include <cstring>
#include <stdexcept>
#include <string>
#include <vector>

#include "gefen_hip.h"

namespace py = pybind11;

namespace {

struct Library {
    decltype(&gefen_last_error) last_error;
    decltype(&gefen_gradient_norm_workspace_size) norm_workspace;
    decltype(&gefen_gradient_norm) norm;
    decltype(&gefen_clip_gradients) clip;
    decltype(&gefen_scale_gradients) scale;
    decltype(&gefen_linear_cross_entropy_workspace_size) lce_workspace;
    decltype(&gefen_linear_cross_entropy) lce;
    decltype(&gefen_scale_by) scale_by;
    decltype(&gefen_scale_from_f32) scale_from_f32;
};
Library lib{};

void bind_library(py::dict addresses) {
    auto at = [&](const char* name) { return addresses[name].cast<uintptr_t>(); };
    lib.norm_workspace = reinterpret_cast<decltype(lib.norm_workspace)>(at("gefen_gradient_norm_workspace_size"));
    lib.norm = reinterpret_cast<decltype(lib.norm)>(at("gefen_gradient_norm"));
    lib.clip = reinterpret_cast<decltype(lib.clip)>(at("gefen_clip_gradients"));
    lib.scale = reinterpret_cast<decltype(lib.scale)>(at("gefen_scale_gradients"));
    lib.lce_workspace =
        reinterpret_cast<decltype(lib.lce_workspace)>(at("gefen_linear_cross_entropy_workspace_size"));
    lib.lce = reinterpret_cast<decltype(lib.lce)>(at("gefen_linear_cross_entropy"));
    lib.scale_by = reinterpret_cast<decltype(lib.scale_by)>(at("gefen_scale_by"));
    lib.scale_from_f32 = reinterpret_cast<decltype(lib.scale_from_f32)>(at("gefen_scale_from_f32"));
    lib.last_error = reinterpret_cast<decltype(lib.last_error)>(at("gefen_last_error"));
}
void need_library() {
    if (!lib.last_error) throw std::runtime_error("bind_library() has not been called");
}

void check(int rc) {
    if (rc == GEFEN_OK) return;
    if (rc == GEFEN_EINVAL) throw py::value_error(lib.last_error());
    throw std::runtime_error(lib.last_error());
}

int32_t dtype_code(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return GEFEN_F32;
        case at::kHalf: return GEFEN_F16;
        case at::kBFloat16: return GEFEN_BF16;
        default: return -1;
    }
}

gefen_stream_t stream_of(const at::Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

at::Tensor bytes_on(const at::Tensor& like, size_t n) {
    return at::empty({static_cast<int64_t>(n)}, like.options().dtype(at::kByte).requires_grad(false));
}

const at::Tensor& tensor_of(py::handle o, const char* name) {
    if (!THPVariable_Check(o.ptr()))
        throw py::type_error(std::string("Expected ") + name + " to be a torch.Tensor, got " + Py_TYPE(o.ptr())->tp_name);
    return THPVariable_Unpack(o.ptr());
}

// Raises for a forward-mode tangent, which a call on addresses would drop.
void no_tangent(const at::Tensor& t, const char* name) {
    const auto* meta = torch::autograd::impl::get_autograd_meta(t);
    if (!meta || !meta->fw_grad(/*level=*/0, t).defined()) return;
    PyErr_Format(PyExc_NotImplementedError, "Expected %s without a forward-mode tangent.", name);
    throw py::error_already_set();
}

// A tensor whose memory holds its values: a view that stands for the negative of its memory
// (the imaginary part of a conjugate) is copied.
at::Tensor as_stored(const at::Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }

py::object wrap(const at::Tensor& t) { return py::reinterpret_steal<py::object>(THPVariable_Wrap(t)); }

// ------------------------------------------------------------------ gradient norm

// The bytes of a tensor's elements: runs of `block` bytes at begin + sum of index x stride.
struct Layout {
    struct Dim {
        int64_t stride, lo, hi;  // bytes; the range of an index (or of the difference of two)
    };
    uint64_t begin;
    int64_t block;
    std::vector<Dim> dims;
    explicit Layout(const at::Tensor& t)
        : begin(reinterpret_cast<uint64_t>(t.data_ptr())), block(static_cast<int64_t>(t.element_size())) {
        for (int64_t i = 0; i < t.dim(); ++i)
            if (t.size(i) > 1) dims.push_back({t.stride(i) * block, 0, t.size(i) - 1});
        std::sort(dims.begin(), dims.end(), [](const Dim& a, const Dim& b) { return a.stride < b.stride; });
        size_t inner = 0;  // dimensions that only continue the run
        while (inner < dims.size() && dims[inner].stride == block) block *= dims[inner++].hi + 1;
        dims.erase(dims.begin(), dims.begin() + inner);
    }
};
// Whether at + sum of stride x index can lie within [least, most], with an index other than 0
// if `apart`.  dims by descending stride: all but a few values of each index are ruled out by
// what the smaller strides reach, so nested layouts take a few steps; one that takes too many
// counts as reaching it.
struct Reach {
    std::vector<Layout::Dim> dims;
    int64_t least, most;
    int steps = 1 << 16;
    std::vector<int64_t> lo, hi;  // reached by dims from k on
    Reach(std::vector<Layout::Dim> all, int64_t least, int64_t most) : least(least), most(most) {
        std::sort(all.begin(), all.end(),
                  [](const Layout::Dim& a, const Layout::Dim& b) { return a.stride > b.stride; });
        for (const Layout::Dim& d : all) {
            if (!dims.empty() && dims.back().stride == d.stride) {
                dims.back().lo += d.lo;
                dims.back().hi += d.hi;
            } else {
                dims.push_back(d);
            }
        }
        lo.assign(dims.size() + 1, 0);
        hi = lo;
        for (size_t k = dims.size(); k-- > 0;) {
            lo[k] = lo[k + 1] + dims[k].stride * dims[k].lo;
            hi[k] = hi[k + 1] + dims[k].stride * dims[k].hi;
        }
    }
    static int64_t floor_div(int64_t a, int64_t b) { return a / b - (a % b < 0); }
    bool from(size_t k, int64_t at, bool apart) {
        if (k == dims.size()) return !apart && at >= least && at <= most;
        const Layout::Dim& d = dims[k];
        const int64_t first = std::max(d.lo, -floor_div(at + hi[k + 1] - least, d.stride));
        const int64_t last = std::min(d.hi, floor_div(most - at - lo[k + 1], d.stride));
        for (int64_t c = first; c <= last; ++c) {
            if (--steps < 0) return true;
            if (from(k + 1, at + c * d.stride, apart && c == 0)) return true;
        }
        return false;
    }
};
bool share_memory(const Layout& a, const Layout& b) {
    std::vector<Layout::Dim> dims;  // an expanded dimension adds no memory
    for (const Layout::Dim& d : a.dims)
        if (d.stride) dims.push_back(d);
    for (const Layout::Dim& d : b.dims)
        if (d.stride) dims.push_back({d.stride, -d.hi, 0});
    const int64_t apart = static_cast<int64_t>(a.begin - b.begin);
    return Reach(std::move(dims), 1 - a.block, b.block - 1).from(0, apart, false);
}
// Whether two elements of a tensor lie in the same memory.
bool overlaps_itself(const at::Tensor& t) {
    if (t.is_non_overlapping_and_dense()) return false;
    Layout l(t);
    std::vector<Layout::Dim> dims;
    for (size_t k = 0; k < l.dims.size(); ++k) {
        const Layout::Dim& d = l.dims[k];
        if (d.stride == 0 || (k > 0 && d.stride == l.dims[k - 1].stride)) return true;
        dims.push_back({d.stride, -d.hi, d.hi});
    }
    return Reach(std::move(dims), 1 - l.block, l.block - 1).from(0, 0, true);
}

// What a call reads and writes: raises where something written shares memory with anything
// else, before anything is launched.
class Accesses {
   public:
    explicit Accesses(size_t most) { spans_.reserve(most); }
    void add(const at::Tensor& t, bool write) {
        if (t.numel() == 0) return;
        const int64_t size = static_cast<int64_t>(t.itemsize());
        int64_t extent = t.numel() * size;
        if (!t.is_contiguous()) {
            if (write && overlaps_itself(t))
                throw py::value_error("Expected gradients to write whose elements do not overlap.");
            extent = size;
            for (int64_t i = 0; i < t.dim(); ++i) extent += (t.size(i) - 1) * t.stride(i) * size;
        }
        const uint64_t begin = reinterpret_cast<uint64_t>(t.data_ptr());
        spans_.push_back({begin, begin + extent, write, &t});
    }
    void check() {
        std::sort(spans_.begin(), spans_.end(), [](const Span& a, const Span& b) { return a.begin < b.begin; });
        std::vector<const Span*> open;  // those that reach past the current one's begin
        uint64_t reach = 0;
        for (const Span& s : spans_) {
            if (s.begin >= reach) open.clear();
            for (const Span* o : open)
                if ((s.write || o->write) && s.begin < o->end && share_memory(Layout(*o->t), Layout(*s.t)))
                    throw py::value_error("Expected gradients that share no memory with what is written.");
            open.push_back(&s);
            reach = std::max(reach, s.end);
        }
    }

   private:
    struct Span {
        uint64_t begin, end;
        bool write;
        const at::Tensor* t;
    };
    std::vector<Span> spans_;
};

// The tasks of a list of gradients (and the list that receives them scaled; None: in
// place).  bad: the first tensor whose elements are not one dense run, in the same order
// in both, or not what its memory holds, or -1.  Raises for what no call takes, and, with `writes`, where what is
// written overlaps anything else of the call (total_norm, if given, among it).
struct Tasks {
    std::vector<gefen_gradient_task> rows;
    std::vector<const at::Tensor*> written;
    at::Tensor first;
    int64_t bad = -1;
    // Autograd's count of in-place writes, for what it has saved; the kernels write through
    // addresses, which it does not see.
    void count_writes() const {
        for (const at::Tensor* t : written)
            if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
    }
};
Tasks tasks_of(const py::list& tensors, const py::object& outs, bool writes, const at::Tensor* total_norm = nullptr) {
    Tasks out;
    const size_t n = tensors.size();
    const bool in_place = outs.is_none();
    py::list out_list = in_place ? py::list() : py::reinterpret_borrow<py::list>(outs);
    if (!in_place && out_list.size() != n) throw py::value_error("Expected as many output tensors as gradients.");
    auto tensor_at = [&](const py::list& l, size_t k) -> const at::Tensor& {
        const at::Tensor& t = tensor_of(PyList_GET_ITEM(l.ptr(), static_cast<Py_ssize_t>(k)), "gradients");
        if (t.unsafeGetTensorImpl()->is_python_dispatch())
            throw py::type_error("Expected plain tensors; give the local shards and the norm over all of them.");
        if (!t.is_cuda()) throw py::value_error("Expected gradients on CUDA, got device " + t.device().str());
        if (!out.first.defined()) out.first = t;
        if (t.device() != out.first.device()) throw py::value_error("Expected all gradients on one device.");
        if (t.layout() != at::kStrided) throw py::value_error("Expected strided gradients.");
        if (dtype_code(t) < 0) throw py::value_error("Expected float32, float16 or bfloat16 gradients.");
        no_tangent(t, "gradients");
        return t;
    };
    Accesses accesses(writes ? 2 * n + 1 : 0);
    out.rows.resize(n);
    for (size_t k = 0; k < n; ++k) {
        const at::Tensor& t = tensor_at(tensors, k);
        gefen_gradient_task& r = out.rows[k];
        r.src = r.dst = t.data_ptr();
        r.numel = t.numel();
        r.src_dtype = r.dst_dtype = dtype_code(t);
        bool dense = !t.is_neg() && (t.is_contiguous() || t.is_non_overlapping_and_dense());
        if (in_place && writes) {
            accesses.add(t, true);
            out.written.push_back(&t);
        }
        if (!in_place) {
            const at::Tensor& o = tensor_at(out_list, k);
            out.written.push_back(&o);
            if (o.sizes() != t.sizes()) throw py::value_error("Expected outputs of the gradients' shapes.");
            r.dst = o.data_ptr();
            r.dst_dtype = dtype_code(o);
            const bool same_order = o.strides() == t.strides() || (o.is_contiguous() && t.is_contiguous());
            dense = dense && same_order && !o.is_neg();
            accesses.add(o, true);
            if (r.dst != r.src || r.dst_dtype != r.src_dtype || !same_order) accesses.add(t, false);
        }
        if (!dense && r.numel && out.bad < 0) out.bad = static_cast<int64_t>(k);
    }
    if (total_norm) accesses.add(*total_norm, false);
    accesses.check();
    return out;
}

// The norm, or None where a tensor is not one dense run of elements.
py::object gradient_norm(py::list tensors, double norm_type) {
    need_library();
    Tasks t = tasks_of(tensors, py::none(), false);
    if (t.bad >= 0) return py::none();
    const int n = static_cast<int>(t.rows.size());
    c10::DeviceGuard guard(t.first.device());
    at::Tensor norm = at::empty({}, t.first.options().dtype(at::kFloat).requires_grad(false));
    at::Tensor ws = bytes_on(t.first, lib.norm_workspace(t.rows.data(), n));
    check(lib.norm(t.rows.data(), n, norm_type, norm.data_ptr<float>(), ws.data_ptr(), stream_of(norm)));
    return wrap(norm);
}

// Clips (by total_norm, or the norm of these gradients) and returns the norm; None as above.
py::object clip_gradients(py::list tensors, py::object outs, double max_norm, double norm_type, py::object total_norm) {
    need_library();
    const at::Tensor* given = total_norm.is_none() ? nullptr : &tensor_of(total_norm, "total_norm");
    Tasks t = tasks_of(tensors, outs, true, given);
    if (t.bad >= 0) return py::none();
    const int n = static_cast<int>(t.rows.size());
    c10::DeviceGuard guard(t.first.device());
    if (given) {
        const at::Tensor norm = as_stored(*given);
        check(lib.scale(t.rows.data(), n, norm.data_ptr<float>(), max_norm, stream_of(t.first)));
        t.count_writes();
        return total_norm;
    }
    at::Tensor norm = at::empty({}, t.first.options().dtype(at::kFloat).requires_grad(false));
    at::Tensor ws = bytes_on(t.first, lib.norm_workspace(t.rows.data(), n));
    check(lib.clip(t.rows.data(), n, norm_type, max_norm, norm.data_ptr<float>(), ws.data_ptr(), stream_of(norm)));
    t.count_writes();
    return wrap(norm);
}

// ------------------------------------------------------------------ linear cross entropy

struct LceOptions {
    int64_t ignore_index, workspace_limit;
    double label_smoothing;
    int64_t reduction;
};

float* floats(const at::Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
void* data(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// One library call, to be made on the current stream: the task, and what its addresses
// belong to.
struct LceCall {
    at::Tensor h, w, y;
    gefen_linear_cross_entropy_task t{};

    LceCall(const at::Tensor& hidden, const at::Tensor& weight, const at::Tensor& targets, const LceOptions& o)
        : h(as_stored(hidden.dim() == 2 ? hidden : hidden.reshape({-1, hidden.size(-1)}))),
          w(as_stored(weight)),
          y(targets.contiguous()) {
        t.hidden = h.data_ptr();
        t.weight = w.data_ptr();
        t.targets = y.data_ptr();
        t.n = h.size(0);
        t.v = w.size(0);
        t.d = w.size(1);
        t.hidden_row_stride = h.stride(0);
        t.hidden_col_stride = h.stride(1);
        t.weight_row_stride = w.stride(0);
        t.weight_col_stride = w.stride(1);
        t.ignore_index = o.ignore_index;
        t.workspace_limit = o.workspace_limit;
        t.label_smoothing = o.label_smoothing;
        t.dtype = dtype_code(h);
        t.targets_int32 = y.scalar_type() == at::kInt;
        t.reduction = static_cast<int32_t>(o.reduction);
    }
    int grads = 0;  // GEFEN_LCE_GRADS_F32 or nothing
    // The bytes that the stage needs; 0 where it cannot be made.
    size_t bytes(int stage) {
        t.stage = stage | grads;
        return lib.lce_workspace(&t);
    }
    void form(void* grad_hidden, void* grad_weight, bool f32) {
        t.grad_hidden = grad_hidden;
        t.grad_weight = grad_weight;
        grads = f32 ? GEFEN_LCE_GRADS_F32 : 0;
    }
    // The stage of the last bytes(), or (ws defined) a backward stage on what a forward one left.
    at::Tensor run(size_t nbytes, at::Tensor ws = {}) {
        if (nbytes == 0) check(GEFEN_EINVAL);
        if (!ws.defined()) ws = bytes_on(h, nbytes);
        check(lib.lce(&t, ws.data_ptr(), ws.numel(), stream_of(h)));
        return ws;
    }
};

at::Tensor empty_grad(const at::Tensor& like, bool wanted, at::ScalarType type) {
    return wanted ? at::empty(like.sizes(), like.options().dtype(type).requires_grad(false)) : at::Tensor();
}

// The loss, and for its backward pass one of
//   * kept: what the gradients are formed from, where all rows fit the workspace limit
//     together.  16-bit gradients wait, so that the loss's own gradient reaches them before
//     they are rounded, and so do those of losses that are not reduced;
//   * gh, gw: the gradients of a reduced loss of float32 operands;
//   * formed: those of bfloat16 ones in pieces or small (kFormSmall), in float32, hidden's
//     first (Formed);
//   * nothing: they are formed from the operands.
// Elements of bfloat16 gradients up to which they are formed in the forward call: rounding
// them from float32 moves 8 bytes an element more, and keeping values takes a launch more and
// the row losses a pass of their own (48 x 1000 x 96: 36 us on the device against 40 to 44).
constexpr int64_t kFormSmall = 4 << 20;
struct Formed {
    int64_t nh, nw, at_w, numel;
    Formed(const at::Tensor& hidden, const at::Tensor& weight, bool need_h, bool need_w)
        : nh(need_h ? hidden.numel() : 0), nw(need_w ? weight.numel() : 0), at_w((nh + 63) / 64 * 64), numel(at_w + nw) {}
    float* hidden(const at::Tensor& t) const { return nh ? t.data_ptr<float>() : nullptr; }
    float* weight(const at::Tensor& t) const { return nw ? t.data_ptr<float>() + at_w : nullptr; }
};
at::Tensor lce_forward(const at::Tensor& hidden, const at::Tensor& weight, const at::Tensor& targets,
                       const LceOptions& o, bool need_h, bool need_w, at::Tensor* gh, at::Tensor* gw,
                       at::Tensor* formed, at::Tensor* kept) {
    c10::DeviceGuard guard(hidden.device());
    const auto f32 = hidden.options().dtype(at::kFloat).requires_grad(false);
    const bool reduced = o.reduction != GEFEN_REDUCE_NONE, need = need_h || need_w;
    const at::ScalarType type = hidden.scalar_type();
    LceCall c(hidden, weight, targets, o);
    at::Tensor result = reduced ? at::empty({}, f32) : at::empty(targets.sizes(), f32);
    (reduced ? c.t.loss : c.t.losses) = floats(result);
    const bool small = type == at::kBFloat16 && hidden.numel() + weight.numel() <= kFormSmall;
    if (need && !(reduced && (type == at::kFloat || small))) {
        if (const size_t nbytes = c.bytes(GEFEN_LCE_FORWARD)) {
            *kept = c.run(nbytes);
            return result;
        }
    }
    if (need && reduced && type == at::kFloat) {
        *gh = empty_grad(hidden, need_h, type);
        *gw = empty_grad(weight, need_w, type);
        c.form(data(*gh), data(*gw), true);
    } else if (need && reduced && type == at::kBFloat16) {
        const Formed f(hidden, weight, need_h, need_w);
        *formed = at::empty({f.numel}, f32);
        c.form(f.hidden(*formed), f.weight(*formed), true);
    }
    c.run(c.bytes(GEFEN_LCE_WHOLE));
    return result;
}

class LinearCrossEntropy : public torch::autograd::Function<LinearCrossEntropy> {
   public:
    static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& hidden, const at::Tensor& weight,
                              const at::Tensor& targets, int64_t ignore_index, int64_t workspace_limit,
                              double label_smoothing, int64_t reduction, bool need_h, bool need_w) {
        at::Tensor gh, gw, formed, kept;
        at::Tensor result = lce_forward(hidden, weight, targets, {ignore_index, workspace_limit, label_smoothing, reduction},
                                        need_h, need_w, &gh, &gw, &formed, &kept);
        // what waits for backward is saved as the operands are: hooks of saved tensors see it
        ctx->save_for_backward({hidden, weight, targets, gh, gw, formed, kept});
        int64_t smoothing;
        std::memcpy(&smoothing, &label_smoothing, 8);
        ctx->saved_data["options"] =
            std::vector<int64_t>{ignore_index, workspace_limit, smoothing, reduction, need_h, need_w};
        return result;
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                   torch::autograd::variable_list grads) {
        TORCH_CHECK(!c10::GradMode::is_enabled(), "linear_cross_entropy can be differentiated once only");
        at::Tensor gh, gw;
        if (grads[0].defined()) {
            const std::vector<int64_t> o = ctx->saved_data["options"].toIntVector();
            const bool need_h = o[4], need_w = o[5];
            const auto saved = ctx->get_saved_variables();
            const at::Tensor &hidden = saved[0], &weight = saved[1], &formed = saved[5];
            const at::ScalarType type = hidden.scalar_type();
            c10::DeviceGuard guard(hidden.device());
            const at::Tensor grad = grads[0].to(at::kFloat).contiguous();
            const float* factor = grad.data_ptr<float>();
            // kept values are used up by the call and float32 gradients handed over: a second
            // backward of a retained graph starts from the operands
            const bool used = ctx->saved_data.count("used");
            if (type == at::kFloat && !used && (saved[3].defined() || saved[4].defined())) {
                ctx->saved_data["used"] = true;
                gh = saved[3];
                gw = saved[4];
                check(lib.scale_by(data(gh), need_h ? gh.numel() : 0, data(gw), need_w ? gw.numel() : 0, GEFEN_F32, factor,
                                   stream_of(hidden)));
            } else {
                gh = empty_grad(hidden, need_h, type);
                gw = empty_grad(weight, need_w, type);
                if (formed.defined()) {
                    const Formed f(hidden, weight, need_h, need_w);
                    check(lib.scale_from_f32(f.hidden(formed), data(gh), f.nh, f.weight(formed), data(gw), f.nw,
                                             dtype_code(hidden), factor, stream_of(hidden)));
                } else {
                    at::Tensor kept;
                    if (!used && saved[6].defined()) {
                        ctx->saved_data["used"] = true;
                        kept = saved[6];
                    }
                    double smoothing;
                    std::memcpy(&smoothing, &o[2], 8);
                    LceCall c(hidden, weight, saved[2], {o[0], o[1], smoothing, o[3]});
                    c.form(data(gh), data(gw), false);
                    c.t.grad = factor;
                    c.run(c.bytes(kept.defined() ? GEFEN_LCE_BACKWARD : GEFEN_LCE_WHOLE), kept);
                }
            }
        }
        return {gh, gw, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
    }
};

std::string shape_of(c10::IntArrayRef s) {
    std::string out = "(";
    for (size_t i = 0; i < s.size(); ++i) out += (i ? ", " : "") + std::to_string(s[i]);
    return out + ")";
}

py::object linear_cross_entropy(py::handle hidden_, py::handle weight_, py::handle targets_, int64_t ignore_index,
                                double label_smoothing, int64_t reduction, int64_t workspace_limit) {
    need_library();
    const at::Tensor& hidden = tensor_of(hidden_, "hidden");
    const at::Tensor& weight = tensor_of(weight_, "weight");
    const at::Tensor& targets = tensor_of(targets_, "targets");
    auto on_device = [&](const at::Tensor& t, const char* name) {
        if (!t.is_cuda())
            throw py::value_error(std::string("Expected ") + name + " to be on CUDA, got device " + t.device().str() + ".");
        if (t.device() != hidden.device())
            throw py::value_error(std::string("Expected ") + name + " on " + hidden.device().str() + ", got " +
                                  t.device().str() + ".");
        if (t.unsafeGetTensorImpl()->is_python_dispatch() || t.layout() != at::kStrided)
            throw py::type_error(std::string("Expected ") + name + " to be a plain strided tensor.");
    };
    on_device(hidden, "hidden");
    on_device(weight, "weight");
    on_device(targets, "targets");
    no_tangent(hidden, "hidden");
    no_tangent(weight, "weight");
    if (dtype_code(hidden) < 0)
        throw py::value_error(std::string("Expected hidden to be float32, float16 or bfloat16, got ") +
                              c10::toString(hidden.scalar_type()));
    if (weight.scalar_type() != hidden.scalar_type())
        throw py::value_error(std::string("Expected weight of hidden's dtype ") + c10::toString(hidden.scalar_type()) +
                              ", got " + c10::toString(weight.scalar_type()));
    if (targets.scalar_type() != at::kLong && targets.scalar_type() != at::kInt)
        throw py::value_error(std::string("Expected targets to be int64 or int32, got ") +
                              c10::toString(targets.scalar_type()));
    if (weight.dim() != 2) throw py::value_error("Expected weight to be 2D, got dim=" + std::to_string(weight.dim()));
    if (hidden.dim() < 1 || hidden.size(-1) != weight.size(1))
        throw py::value_error("Expected hidden of width " + std::to_string(weight.size(1)) + ", got shape " +
                              shape_of(hidden.sizes()));
    if (targets.sizes() != hidden.sizes().slice(0, hidden.dim() - 1))
        throw py::value_error("Expected targets of shape " + shape_of(hidden.sizes().slice(0, hidden.dim() - 1)) +
                              ", got " + shape_of(targets.sizes()));
    if (weight.numel() == 0)
        throw py::value_error("Expected a non-empty weight, got shape " + shape_of(weight.sizes()));
    const bool grad = c10::GradMode::is_enabled();
    const bool need_h = grad && hidden.requires_grad(), need_w = grad && weight.requires_grad();
    if (need_h || need_w)
        return wrap(LinearCrossEntropy::apply(hidden, weight, targets, ignore_index, workspace_limit, label_smoothing,
                                              reduction, need_h, need_w));
    return wrap(lce_forward(hidden.detach(), weight.detach(), targets,
                            {ignore_index, workspace_limit, label_smoothing, reduction}, false, false, nullptr, nullptr,
                            nullptr, nullptr));
}

}  // namespace

void register_training(py::module_& m) {
    m.def("bind_library", &bind_library);
    m.def("gradient_norm", &gradient_norm);
    m.def("clip_gradients", &clip_gradients);
    m.def("linear_cross_entropy", &linear_cross_entropy);
}
