// The torch side of multigrid_amd/policy.py: checks of arguments, output and workspace tensors, autograd nodes, and the calls of
// the C entry points (include/mgrid.h), whose addresses the Python side hands over.  Native because of what surrounds a launch
// of a few microseconds: a differentiable call and its backward pass took 110 us of Python, most of it in handing the
// interpreter's lock to the autograd thread and back.
//
// Nothing here launches a kernel or touches memory on the GPU by itself.

#include <pybind11/stl.h>
#include <torch/extension.h>

#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>

#include <optional>
#include <stdexcept>
#include <string>
#include <unordered_set>
#include <variant>
#include <vector>

#include "mgrid.h"

namespace {

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Fields = std::optional<std::vector<int64_t>>;
using Number = std::variant<Tensor, double>;  // one for all rows, or a tensor of one per row
using Maybe = std::optional<Tensor>;

struct Entry {
    decltype(&mg_last_error) last_error;
    decltype(&mg_embed) embed;
    decltype(&mg_embed_grad_workspace) embed_grad_workspace;
    decltype(&mg_embed_grad) embed_grad;
    decltype(&mg_adjust_logits) adjust;
    decltype(&mg_adjust_logits_grad) adjust_grad;
    decltype(&mg_draw_workspace) draw_workspace;
    decltype(&mg_draw) draw;
    decltype(&mg_token_logprobs_workspace) logprobs_workspace;
    decltype(&mg_token_logprobs) logprobs;
    decltype(&mg_token_logprobs_grad) logprobs_grad;
} entry;

py::object error_type;  // multigrid_amd._lib.MgError

struct Failure : std::runtime_error {
    using std::runtime_error::runtime_error;
};

void check(int64_t rc) {
    if (rc >= 0) return;
    const char *text = entry.last_error(nullptr);
    throw Failure("libmgrid_hip error " + std::to_string(rc) + ": " + (text && *text ? text : "?"));
}

// The device made the current one, and its current stream.
struct On {
    c10::DeviceGuard guard;
    void *stream;
    explicit On(const Tensor &t) : guard(t.device()), stream(c10::hip::getCurrentHIPStream(t.device().index()).stream()) {}
};

const Tensor &on_gpu(const char *name, const Tensor &t) {
    TORCH_CHECK_VALUE(t.is_cuda(), name, " must be a tensor on a GPU (there is no CPU fallback)");
    return t;
}
const Tensor &beside(const char *name, const Tensor &t, const Tensor &other) {
    on_gpu(name, t);
    TORCH_CHECK_VALUE(t.device() == other.device(), name, " is on ", t.device(), ", the other tensors are on ", other.device());
    return t;
}

int floating(const char *name, const Tensor &t) {
    switch (t.scalar_type()) {
        case at::kFloat: return MG_F32;
        case at::kBFloat16: return MG_BF16;
        case at::kHalf: return MG_F16;
        default: TORCH_CHECK_VALUE(false, name, " must be float32, bfloat16 or float16, got ", t.scalar_type());
    }
}
int whole(const char *name, at::ScalarType t) {
    switch (t) {
        case at::kByte: return MG_U8;
        case at::kInt: return MG_I32;
        case at::kLong: return MG_I64;
        default: TORCH_CHECK_VALUE(false, name, " must be uint8, int32 or int64, got ", t);
    }
}

bool wants_grad(const Tensor &t) { return at::GradMode::is_enabled() && t.requires_grad(); }

// Forward-mode differentiation (which torch.no_grad() does not switch off): a tangent is refused, as its loss would read as a derivative of 0.
bool has_tangent(const Tensor &t) { return c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(/*level=*/0).defined(); }
void no_tangent(const char *name, const Tensor &t) { TORCH_CHECK_NOT_IMPLEMENTED(!has_tangent(t), name, " has a tangent: forward-mode derivatives are not supported"); }

void no_gradient(const char *name, const Maybe &t, const char *instead) {
    if (!t) return;
    TORCH_CHECK_VALUE(!wants_grad(*t), name, " passes no gradient: ", instead);
    no_tangent(name, *t);
}
void no_gradient(const char *name, const Number &v) {
    if (const Tensor *t = std::get_if<Tensor>(&v)) no_gradient(name, Maybe(*t), "detach it");
}

// Before a differentiable call of `t`, while a stream is captured: a leaf's gradient is accumulated on the stream that was
// current when the first graph that holds the leaf was built.  Where that is the default stream, the captured backward pass
// would order work behind it, which no capture allows and no one catches.
void no_leaf_of_the_default_stream(const Tensor &t) {
    const auto current = c10::hip::getCurrentHIPStream(t.device().index());
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    if (current.id() == 0 || hipStreamIsCapturing(current.stream(), &status) != hipSuccess || status == hipStreamCaptureStatusNone) return;  // (the default stream is never captured)
    std::vector<std::shared_ptr<torch::autograd::Node>> rest;
    std::unordered_set<torch::autograd::Node *> seen;
    if (auto first = t.grad_fn() ? t.grad_fn() : torch::autograd::impl::try_get_grad_accumulator(t)) rest.push_back(std::move(first));
    while (!rest.empty()) {
        const auto node = std::move(rest.back());
        rest.pop_back();
        if (!seen.insert(node.get()).second) continue;
        const auto stream = node->stream();
        TORCH_CHECK(!stream || stream->id() != 0, "a differentiable call is captured, but what it depends on belongs to an eager graph of the default stream as well (", node->name(),
                    "): let that graph go first (del its outputs)");
        for (const auto &edge : node->next_edges())
            if (edge.function) rest.push_back(edge.function);
    }
}

// of a backward pass, with the gradients that come in
void once(const variable_list &grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "the operators of multigrid_amd.policy are differentiable once (create_graph is not supported)");
    for (const Tensor &g : grads) TORCH_CHECK_NOT_IMPLEMENTED(!g.defined() || !has_tangent(g), "the operators of multigrid_amd.policy are differentiable once (the gradient has a tangent)");
}

// [..., k] as [n, k] with adjacent elements in a row; a view wherever there is one
Tensor rows_of(const Tensor &t) {
    const int64_t k = t.size(-1);
    Tensor r = t;
    if (t.dim() != 2) {
        int64_t n = 1;
        for (int64_t d = 0; d + 1 < t.dim(); ++d) n *= t.size(d);
        r = t.reshape({n, k});
    }
    return k == 1 || r.stride(1) == 1 ? r : r.contiguous();
}
int64_t row_stride(const Tensor &t) { return t.size(0) > 1 ? t.stride(0) : 0; }

Tensor workspace(int64_t bytes, const Tensor &like) {
    check(bytes);
    return bytes ? at::empty({bytes}, like.options().dtype(at::kByte)) : Tensor();
}
void *address(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
int64_t bytes_of(const Tensor &t) { return t.defined() ? t.numel() : 0; }

// ---- embedding

struct Lookup {
    MgEmbed e{};
    Tensor ids;                  // [n, fields]
    std::vector<int64_t> shape;  // of the tokens
};

Lookup lookup(const Tensor &ids, const Fields &fields, int64_t rows, int64_t dim, int dtype, double scale) {
    Lookup l;
    MgEmbed &e = l.e;
    int64_t count = 1;
    TORCH_CHECK_VALUE(rows <= (1 << 30) && dim <= (1 << 20), "a table of ", rows, " x ", dim, " is not supported");
    if (!fields) {
        l.shape = ids.sizes().vec();
        e.sizes[0] = static_cast<int32_t>(rows);
    } else {
        count = static_cast<int64_t>(fields->size());
        int64_t sum = 0;
        bool ok = count >= 1 && count <= MG_MAX_FIELDS;
        for (int64_t f = 0; ok && f < count; ++f) {
            ok = (*fields)[f] >= 1 && (*fields)[f] <= rows;
            sum += (*fields)[f];
            e.sizes[f] = static_cast<int32_t>((*fields)[f]);
        }
        TORCH_CHECK_VALUE(ok && sum == rows, "fields ", *fields, " must be 1 to ", MG_MAX_FIELDS, " positive numbers that add up to the ", rows, " rows of the table");
        TORCH_CHECK_VALUE(ids.dim() >= 1 && ids.size(-1) == count, "ids of shape ", ids.sizes(), " must have ", count, " fields in their last dimension");
        l.shape.assign(ids.sizes().begin(), ids.sizes().end() - 1);
    }
    int64_t n = 1;
    for (int64_t s : l.shape) n *= s;
    l.ids = ids.reshape({n, count});
    e.n = n;
    e.fields = static_cast<int32_t>(count);
    e.dim = static_cast<int32_t>(dim);
    e.ids_type = whole("ids", ids.scalar_type());
    e.dtype = dtype;
    e.ids_stride = row_stride(l.ids);
    e.field_stride = l.ids.stride(1);
    e.scale = static_cast<float>(scale);
    return l;
}

// `copy`: set to a copy of the ids, written by the same launch
Tensor embed_forward(const Tensor &ids, const Tensor &given, const Fields &fields, double scale, Tensor *copy = nullptr) {
    const Tensor table = given.stride(1) == 1 || given.size(1) == 1 ? given : given.contiguous();
    Lookup l = lookup(ids, fields, table.size(0), table.size(1), floating("table", table), scale);
    l.e.row_stride = row_stride(table);
    l.shape.push_back(table.size(1));
    Tensor out = at::empty(l.shape, table.options());
    if (copy) {
        *copy = at::empty(ids.sizes(), ids.options());
        l.e.ids_copy_dev = address(*copy);
    }
    if (out.numel()) {
        On on(table);
        check(entry.embed(&l.e, address(l.ids), address(table), address(out), on.stream));
    }
    return out;
}

Tensor embed_grad(const Tensor &grad, const Tensor &ids, int64_t rows, const Fields &fields, double scale) {
    on_gpu("grad", grad);
    beside("ids", ids, grad);
    TORCH_CHECK_VALUE(grad.dim() >= 1 && grad.size(-1) >= 1 && rows >= 1, "grad of shape ", grad.sizes(), " and ", rows, " rows: both must hold something");
    Lookup l = lookup(ids, fields, rows, grad.size(-1), floating("grad", grad), scale);
    TORCH_CHECK_VALUE(grad.sizes().slice(0, grad.dim() - 1) == at::IntArrayRef(l.shape), "grad has shape ", grad.sizes(), ", the ids are of shape ", l.shape);
    const Tensor g = rows_of(grad);
    l.e.row_stride = row_stride(g);
    Tensor out = at::empty({rows, grad.size(-1)}, grad.options());
    On on(grad);
    const Tensor ws = workspace(entry.embed_grad_workspace(&l.e), grad);
    check(entry.embed_grad(&l.e, address(l.ids), address(g), address(out), address(ws), bytes_of(ws), on.stream));
    return out;
}

struct Embed : torch::autograd::Function<Embed> {
    static Tensor forward(AutogradContext *ctx, const Tensor &ids, const Tensor &table, const Fields &fields, double scale) {
        // a copy of the ids is kept: the simulator writes its images in place, where no version is counted
        Tensor copy;
        Tensor out = embed_forward(ids, table, fields, scale, &copy);
        ctx->save_for_backward({copy});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["rows"] = table.size(0);
        ctx->saved_data["fields"] = fields ? c10::IValue(*fields) : c10::IValue();
        return out;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        once(grads);
        const auto &f = ctx->saved_data["fields"];
        const Fields fields = f.isNone() ? Fields() : Fields(f.toIntVector());
        return {Tensor(), embed_grad(grads[0], ctx->get_saved_variables()[0], ctx->saved_data["rows"].toInt(), fields, ctx->saved_data["scale"].toDouble()), Tensor(), Tensor()};
    }
};

Tensor embed(const Tensor &ids, const Tensor &table, const Fields &fields, double scale) {
    on_gpu("table", table);
    beside("ids", ids, table);
    TORCH_CHECK_VALUE(table.dim() == 2 && table.size(0) && table.size(1), "table must be [rows, dim] and hold something, got ", table.sizes());
    no_tangent("table", table);
    if (!wants_grad(table)) return embed_forward(ids, table, fields, scale);
    no_leaf_of_the_default_stream(table);
    return Embed::apply(ids, table, fields, scale);
}

// ---- adjustment of logits

at::IntArrayRef lead_of(const Tensor &logits) {
    on_gpu("logits", logits);
    TORCH_CHECK_VALUE(logits.dim() >= 1 && logits.size(-1) >= 1, "logits must be [..., k], got ", logits.sizes());
    return logits.sizes().slice(0, logits.dim() - 1);
}

// a number, or float32 [n]: the tensor (undefined for a number) and the number
std::pair<Tensor, float> per_row(const char *name, const Number &v, const Tensor &logits) {
    if (const double *d = std::get_if<double>(&v)) return {Tensor(), static_cast<float>(*d)};
    Tensor t = std::get<Tensor>(v);
    beside(name, t, logits);
    const auto lead = lead_of(logits);
    if (t.dim() == 0) t = t.expand(lead);
    TORCH_CHECK_VALUE(t.sizes() == lead, name, " must be a number or of shape ", lead, ", got ", t.sizes());
    return {t.to(at::kFloat).reshape({-1}).contiguous(), 0.f};
}

// [width] for every row, or [..., width]
Tensor table_of(const char *name, const Tensor &t, const Tensor &logits, int64_t width) {
    beside(name, t, logits);
    if (t.dim() == 1 && t.size(0) == width) return t.contiguous();
    const auto lead = lead_of(logits);
    TORCH_CHECK_VALUE(t.dim() == logits.dim() && t.size(-1) == width && t.sizes().slice(0, t.dim() - 1) == lead, name, " must be of shape [", width, "] or ", lead, " + [", width,
                      "], got ", t.sizes());
    return width ? rows_of(t) : t;
}
int64_t table_stride(const Tensor &t) { return t.dim() == 1 || t.size(0) <= 1 ? 0 : t.stride(0); }

// whether two tensors may share memory, by their first and last element
bool overlap(const Tensor &a, const Tensor &b) {
    if (!a.numel() || !b.numel()) return false;
    auto end = [](const Tensor &t) {
        int64_t last = 1;
        for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
        return static_cast<const char *>(t.data_ptr()) + last * t.element_size();
    };
    return static_cast<const char *>(a.data_ptr()) < end(b) && static_cast<const char *>(b.data_ptr()) < end(a);
}

struct Adjustment {
    MgAdjust a{};
    std::vector<Tensor> keep;  // whose memory it names
};

Adjustment adjustment(const Tensor &logits, const Maybe &history, const Maybe &lengths, const Number &repetition, const Number &presence, const Number &frequency,
                      const Maybe &bias, const Maybe &mask) {
    const auto lead = lead_of(logits);
    Adjustment d;
    MgAdjust &a = d.a;
    const int64_t k = logits.size(-1);
    TORCH_CHECK_VALUE(k <= (1 << 24), "rows of ", k, " tokens are not supported (at most 2^24)");
    a.n = logits.numel() / k;
    a.k = static_cast<int32_t>(k);
    a.dtype = floating("logits", logits);
    d.keep.reserve(8);
    if (history) {
        a.history_type = whole("history", beside("history", *history, logits).scalar_type());
        TORCH_CHECK_VALUE(history->dim() >= 1 && history->size(-1) <= (1 << 24), "history must be [t] or [..., t], got ", history->sizes());
        const Tensor h = table_of("history", *history, logits, history->size(-1));
        a.t = static_cast<int32_t>(h.size(-1));
        a.history_dev = a.t ? address(h) : nullptr;
        a.history_stride = a.t ? table_stride(h) : 0;
        d.keep.push_back(h);
        if (lengths) {
            beside("lengths", *lengths, logits);
            TORCH_CHECK_VALUE((lengths->scalar_type() == at::kInt || lengths->scalar_type() == at::kLong) && lengths->sizes() == lead, "lengths must be int32 or int64 of shape ", lead,
                              ", got ", lengths->scalar_type(), " ", lengths->sizes());
            Tensor n = lengths->scalar_type() == at::kLong ? lengths->clamp(0, a.t).to(at::kInt) : *lengths;
            n = n.reshape({-1}).contiguous();
            a.lengths_dev = static_cast<const int32_t *>(address(n));
            d.keep.push_back(n);
        }
    } else {
        TORCH_CHECK_VALUE(!lengths, "lengths without a history");
    }
    auto row = [&](const char *name, const Number &v, const float *&dev, float &number) {
        auto [t, value] = per_row(name, v, logits);
        number = value;
        if (t.defined()) {
            dev = static_cast<const float *>(address(t));
            d.keep.push_back(std::move(t));
        }
    };
    row("repetition", repetition, a.repetition_dev, a.repetition);
    row("presence", presence, a.presence_dev, a.presence);
    row("frequency", frequency, a.frequency_dev, a.frequency);
    if (bias) {
        Tensor b = table_of("bias", *bias, logits, k);
        if (b.scalar_type() != at::kFloat) b = b.to(at::kFloat);
        a.bias_dev = static_cast<const float *>(address(b));
        a.bias_stride = table_stride(b);
        d.keep.push_back(std::move(b));
    }
    if (mask) {
        const auto type = mask->scalar_type();
        TORCH_CHECK_VALUE(type == at::kBool || type == at::kByte || type == at::kInt, "mask must be bool or uint8 (one for each token) or int32 (one bit for each token), got ", type);
        a.mask_kind = type == at::kInt ? MG_MASK_BITS : MG_MASK_BYTES;
        Tensor m = table_of("mask", *mask, logits, type == at::kInt ? (k + 31) / 32 : k);
        a.mask_dev = address(m);
        a.mask_stride = table_stride(m);
        d.keep.push_back(std::move(m));
    }
    return d;
}

Tensor adjust_forward(const Tensor &logits, const Maybe &into, const Maybe &history, const Maybe &lengths, const Number &repetition, const Number &presence,
                      const Number &frequency, const Maybe &bias, const Maybe &mask) {
    Adjustment d = adjustment(logits, history, lengths, repetition, presence, frequency, bias, mask);
    const Tensor x = rows_of(logits), out = into ? *into : at::empty(logits.sizes(), logits.options());
    d.a.logits_stride = row_stride(x);
    d.a.out_stride = d.a.k;
    if (into)
        for (const Tensor &t : d.keep) TORCH_CHECK_VALUE(!overlap(out, t), "out must not lie across history, lengths, penalties, bias or mask");
    if (d.a.n) {
        On on(logits);
        check(entry.adjust(&d.a, address(x), address(out), on.stream));
    }
    // a write that autograd counts: a graph that has kept the tensor raises instead of using the new values (inference tensors count none)
    if (into && !out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
    return out;
}

struct Adjust : torch::autograd::Function<Adjust> {
    static Tensor forward(AutogradContext *ctx, const Tensor &logits, const Maybe &history, const Maybe &lengths, const Number &repetition, const Number &presence,
                          const Number &frequency, const Maybe &bias, const Maybe &mask) {
        const Tensor *of_rows = std::get_if<Tensor>(&repetition);
        ctx->save_for_backward({logits, history.value_or(Tensor()), lengths.value_or(Tensor()), of_rows ? *of_rows : Tensor(), mask.value_or(Tensor())});
        ctx->saved_data["repetition"] = of_rows ? 0.0 : std::get<double>(repetition);
        return adjust_forward(logits, Maybe(), history, lengths, repetition, presence, frequency, bias, mask);
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        once(grads);
        const auto saved = ctx->get_saved_variables();
        const Tensor &logits = saved[0];
        auto maybe = [](const Tensor &t) { return t.defined() ? Maybe(t) : Maybe(); };
        const Number repetition = saved[3].defined() ? Number(saved[3]) : Number(ctx->saved_data["repetition"].toDouble());
        Adjustment d = adjustment(logits, maybe(saved[1]), maybe(saved[2]), repetition, 0.0, 0.0, Maybe(), maybe(saved[4]));
        const Tensor x = rows_of(logits), g = rows_of(grads[0]), out = at::empty(logits.sizes(), logits.options());
        d.a.logits_stride = row_stride(x);
        d.a.grad_stride = row_stride(g);
        d.a.out_stride = d.a.k;
        if (d.a.n) {
            On on(logits);
            check(entry.adjust_grad(&d.a, address(x), address(g), address(out), on.stream));
        }
        return {out, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

Tensor adjust_logits(const Tensor &logits, const Maybe &history, const Maybe &lengths, const Number &repetition, const Number &presence, const Number &frequency,
                     const Maybe &bias, const Maybe &mask, const Maybe &out) {
    on_gpu("logits", logits);
    no_tangent("logits", logits);
    no_gradient("repetition", repetition);
    no_gradient("presence", presence);
    no_gradient("frequency", frequency);
    no_gradient("bias", bias, "add one that is trained to the logits");
    if (out) {
        TORCH_CHECK_VALUE(!wants_grad(logits) && !wants_grad(*out), "out is not differentiable: leave it out, or call under torch.no_grad()");
        beside("out", *out, logits);
        no_tangent("out", *out);
        TORCH_CHECK_VALUE(out->sizes() == logits.sizes() && out->scalar_type() == logits.scalar_type() && out->is_contiguous(), "out must be contiguous, ", logits.scalar_type(),
                          " and of shape ", logits.sizes());
        TORCH_CHECK_VALUE(!overlap(*out, logits) || (out->data_ptr() == logits.data_ptr() && logits.is_contiguous()), "out may be the logits or lie beside them, not across them");
    } else if (wants_grad(logits)) {
        no_leaf_of_the_default_stream(logits);
        return Adjust::apply(logits, history, lengths, repetition, presence, frequency, bias, mask);
    }
    return adjust_forward(logits, out, history, lengths, repetition, presence, frequency, bias, mask);
}

// ---- draw, log-probabilities

struct Rows {
    MgLogits l{};
    Tensor x, temperature;
};

Rows rows(const Tensor &logits, const Number &temperature, int tokens_type) {
    lead_of(logits);
    TORCH_CHECK_VALUE(logits.size(-1) <= (1 << 24), "rows of ", logits.size(-1), " tokens are not supported (at most 2^24)");
    Rows r;
    r.x = rows_of(logits);
    auto [t, number] = per_row("temperature", temperature, logits);
    r.temperature = t;
    r.l.n = r.x.size(0);
    r.l.k = static_cast<int32_t>(r.x.size(1));
    r.l.dtype = floating("logits", logits);
    r.l.stride = row_stride(r.x);
    r.l.temperature_dev = static_cast<const float *>(address(t));
    r.l.temperature = number;
    r.l.tokens_type = tokens_type;
    return r;
}

std::pair<Tensor, Tensor> draw(const Tensor &logits, const Maybe &uniforms, const Number &temperature, at::ScalarType dtype) {
    Rows r = rows(logits, temperature, whole("dtype", dtype));
    const auto lead = lead_of(logits);
    no_gradient("temperature", temperature);
    TORCH_CHECK_VALUE(dtype != at::kByte || logits.size(-1) <= 255, "tokens as uint8 take rows of at most 255, got ", logits.size(-1));
    Tensor u;
    if (uniforms) {
        beside("uniforms", *uniforms, logits);
        TORCH_CHECK_VALUE((uniforms->scalar_type() == at::kFloat || uniforms->scalar_type() == at::kDouble) && uniforms->sizes() == lead, "uniforms must be float32 or float64 of shape ",
                          lead, ", got ", uniforms->scalar_type(), " ", uniforms->sizes());
        u = uniforms->contiguous();
    }
    const Tensor tokens = at::empty(lead, logits.options().dtype(dtype)), logprobs = at::empty(lead, logits.options().dtype(at::kFloat));
    On on(logits);
    const Tensor ws = workspace(entry.draw_workspace(&r.l), logits);
    check(entry.draw(&r.l, address(r.x), address(u), u.defined() && u.scalar_type() == at::kDouble ? MG_F64 : MG_F32, address(tokens),
                     static_cast<float *>(address(logprobs)), address(ws), bytes_of(ws), on.stream));
    return {tokens, logprobs};
}

std::vector<Tensor> logprobs_forward(const Tensor &logits, const Tensor &given, const Number &temperature, bool stats) {
    Rows r = rows(logits, temperature, whole("tokens", beside("tokens", given, logits).scalar_type()));
    const auto lead = lead_of(logits);
    TORCH_CHECK_VALUE(given.sizes() == lead, "tokens must be of shape ", lead, ", got ", given.sizes());
    const Tensor tokens = given.contiguous();
    const auto floats = logits.options().dtype(at::kFloat);
    const Tensor logprobs = at::empty(lead, floats), entropies = at::empty(lead, floats), kept = stats && r.l.k > MG_LOGPROB_NO_STATS ? at::empty({r.l.n, 4}, floats) : Tensor();
    On on(logits);
    const Tensor ws = workspace(entry.logprobs_workspace(&r.l), logits);
    check(entry.logprobs(&r.l, address(r.x), address(tokens), static_cast<float *>(address(logprobs)), static_cast<float *>(address(entropies)),
                         static_cast<float *>(address(kept)), address(ws), bytes_of(ws), on.stream));
    return {logprobs, entropies, kept};
}

struct Logprobs : torch::autograd::Function<Logprobs> {
    static variable_list forward(AutogradContext *ctx, const Tensor &logits, const Tensor &tokens, const Number &temperature) {
        auto out = logprobs_forward(logits, tokens, temperature, true);
        const Tensor *of_rows = std::get_if<Tensor>(&temperature);
        ctx->save_for_backward({logits, tokens, of_rows ? *of_rows : Tensor(), out[2]});
        ctx->saved_data["temperature"] = of_rows ? 0.0 : std::get<double>(temperature);
        ctx->set_materialize_grads(false);
        out.pop_back();
        return out;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        once(grads);
        const auto saved = ctx->get_saved_variables();
        const Tensor &logits = saved[0];
        Rows r = rows(logits, saved[2].defined() ? Number(saved[2]) : Number(ctx->saved_data["temperature"].toDouble()), whole("tokens", saved[1].scalar_type()));
        const Tensor tokens = saved[1].contiguous(), out = at::empty(logits.sizes(), logits.options());
        Tensor g[2];
        int64_t stride[2] = {0, 0};
        for (int i = 0; i < 2; ++i)
            if (grads[i].defined()) {
                g[i] = grads[i].scalar_type() == at::kFloat ? grads[i] : grads[i].to(at::kFloat);
                if (g[i].dim() != 1) g[i] = g[i].reshape({-1});
                stride[i] = row_stride(g[i]);
            }
        On on(logits);
        check(entry.logprobs_grad(&r.l, address(r.x), address(tokens), static_cast<const float *>(address(saved[3])), static_cast<const float *>(address(g[0])), stride[0],
                                  static_cast<const float *>(address(g[1])), stride[1], address(out), on.stream));
        return {out, Tensor(), Tensor()};
    }
};

std::pair<Tensor, Tensor> token_logprobs(const Tensor &logits, const Tensor &tokens, const Number &temperature) {
    on_gpu("logits", logits);
    no_tangent("logits", logits);
    no_gradient("temperature", temperature);
    if (wants_grad(logits)) no_leaf_of_the_default_stream(logits);
    const auto out = wants_grad(logits) ? Logprobs::apply(logits, tokens, temperature) : logprobs_forward(logits, tokens, temperature, false);
    return {out[0], out[1]};
}

void bind(const std::vector<uintptr_t> &at, py::object error) {
    TORCH_CHECK_VALUE(at.size() * sizeof(void *) == sizeof entry, "wrong number of entry points");
    std::memcpy(static_cast<void *>(&entry), at.data(), sizeof entry);
    error_type = std::move(error);
}

}  // namespace

PYBIND11_MODULE(_policy_torch, m) {
    m.def("bind", &bind);
    m.def("embed", &embed);
    m.def("embed_grad", &embed_grad);
    m.def("adjust_logits", &adjust_logits);
    m.def("draw", &draw);
    m.def("token_logprobs", &token_logprobs);
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const Failure &e) {
            PyErr_SetString(error_type.ptr(), e.what());
        }
    });
    m.add_object("_cleanup", py::capsule([] { error_type.release(); }));
}
