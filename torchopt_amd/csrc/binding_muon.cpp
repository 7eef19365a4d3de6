// torchopt_amd._C.muon_op -- the operators for matrix-shaped parameters (include/toa_muon.h) over
// PyTorch tensors: checks, outputs, device, stream and workspace, then one call into the C ABI.
// The reference has no counterpart; manners are those of torchopt_amd._C.adam_op.
#include "binding_common.hpp"

#include <algorithm>
#include <array>
#include <cmath>
#include <tuple>

#include "toa_muon.h"

namespace py = pybind11;
using namespace toa_binding;

namespace {

void check(int rc, const char *name) {
    TORCH_CHECK(rc == 0, name, ": ", toa_muon_error_string(rc), " (code ", rc, ")");
}

using Coefficients = std::array<double, 3>;

toa_muon_series seriesOf(int steps, const Coefficients &c, double eps) {
    return {steps, c[0], c[1], c[2], eps};
}

// Nothing here carries the tangents of forward-mode differentiation on: a result without one would
// count as a constant.
void requireNoTangent(const char *name, const TensorList &l) {
    for (const Tensor &t : l)
        TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(/*level=*/0).defined(), name,
                                    ": forward-mode derivatives are not served, got a dual tensor");
}

// Same device and dtype throughout, no tangents, and an element type the library serves.
int gate(const char *name, const TensorList &l) {
    for (const Tensor &t : l) {
        if (!t.is_cuda()) throw std::runtime_error("Not implemented");
        TORCH_CHECK(!t.is_neg(), name, ": expected tensors that are what their memory holds; use "
                                       "resolve_neg() on views with the negative bit");
        TORCH_CHECK(t.device() == l[0].device(), name, ": expected all tensors on ", l[0].device(),
                    ", got one on ", t.device());
        TORCH_CHECK(t.scalar_type() == l[0].scalar_type(), name, ": expected scalar type ",
                    l[0].scalar_type(), " but found ", t.scalar_type());
    }
    requireNoTangent(name, l);
    const int code = dtypeCode(l[0], name);
    TORCH_CHECK(code != TOA_F64, "\"", name, "\" not implemented for 'Double'");
    return code;
}

// The matrices of a list: a tensor's last two dimensions, once for every index of the others.
struct Matrices {
    std::vector<int64_t> rows, cols;

    explicit Matrices(const char *name, const TensorList &l) {
        for (const Tensor &t : l) {
            TORCH_CHECK(t.dim() >= 2, name, ": expected matrices (at least 2 dimensions), got sizes ",
                        t.sizes());
            if (t.numel() == 0) continue;
            const int64_t m = t.size(-2), n = t.size(-1), count = t.numel() / (m * n);
            rows.insert(rows.end(), (size_t)count, m);
            cols.insert(cols.end(), (size_t)count, n);
        }
    }
};

std::vector<toa_muon_view> viewsOf(const TensorList &l, size_t count) {
    std::vector<toa_muon_view> out;
    out.reserve(count);
    for (const Tensor &t : l) {
        if (t.numel() == 0) continue;
        const int64_t d = t.dim(), rs = t.stride(d - 2), cs = t.stride(d - 1);
        char *data = (char *)t.data_ptr();
        std::vector<int64_t> at((size_t)d, 0);
        for (;;) {
            int64_t offset = 0;
            for (int64_t k = 0; k < d - 2; ++k) offset += at[(size_t)k] * t.stride(k);
            out.push_back({data + offset * (int64_t)t.element_size(), rs, cs});
            int64_t k = d - 3;
            while (k >= 0 && ++at[(size_t)k] == t.size(k)) at[(size_t)k--] = 0;
            if (k < 0) break;
        }
    }
    return out;
}

Tensor workspaceFor(const char *name, const Tensor &like, size_t bytes, int status) {
    check(status, name);
    return at::empty({(int64_t)bytes}, like.options().dtype(at::kByte).requires_grad(false));
}

// ---- orthogonalize and its gradient --------------------------------------------------------

// Results, and what the gradient can use of the way to them (or nothing, where that is nothing or more
// than `keep` bytes).
std::pair<TensorList, c10::optional<Tensor>> orthogonalizeKeepMulti(const py::object &inputs_o,
                                                                    int64_t keep, int steps,
                                                                    const Coefficients &c,
                                                                    double eps) {
    const char *name = "muonOrthogonalizeMulti";
    const TensorList in = toTensorList(inputs_o, "inputs");
    TensorList out;
    c10::optional<Tensor> kept;
    if (in.empty()) return {out, kept};
    const int code = gate(name, in);
    const Matrices m(name, in);
    for (const Tensor &t : in) out.push_back(at::empty_like(t));
    const toa_muon_series series = seriesOf(steps, c, eps);
    const OnDeviceOf dev(in[0]);
    int status = 0;
    size_t kept_bytes = 0;
    if (keep > 0) {
        kept_bytes = toa_muon_kept_bytes(code, m.rows.size(), m.rows.data(), m.cols.data(), &series, &status);
        if (kept_bytes > (size_t)keep) kept_bytes = 0;
        if (kept_bytes) kept = workspaceFor(name, in[0], kept_bytes, status);
    }
    const size_t bytes = toa_muon_orthogonalize_workspace(
        code, m.rows.size(), m.rows.data(), m.cols.data(), &series, kept_bytes != 0, &status);
    const Tensor ws = workspaceFor(name, in[0], bytes, status);
    check(toa_muon_orthogonalize_multi(code, m.rows.size(), m.rows.data(), m.cols.data(),
                                       viewsOf(in, m.rows.size()).data(),
                                       viewsOf(out, m.rows.size()).data(), &series,
                                       kept ? kept->data_ptr() : nullptr, kept_bytes, ws.data_ptr(),
                                       bytes, dev.stream()),
          name);
    return {out, kept};
}

TensorList orthogonalizeMulti(const py::object &inputs_o, int steps, const Coefficients &c,
                              double eps) {
    return orthogonalizeKeepMulti(inputs_o, 0, steps, c, eps).first;
}

TensorList orthogonalizeBackwardMulti(const py::object &grads_o, const py::object &inputs_o,
                                      int steps, const Coefficients &c, double eps,
                                      const c10::optional<Tensor> &kept) {
    const char *name = "muonOrthogonalizeBackwardMulti";
    const TensorList in = toTensorList(inputs_o, "inputs");
    TensorList dy = toTensorList(grads_o, "grads"), out;
    TORCH_CHECK(dy.size() == in.size(), name, ": tensor lists differ in length");
    if (in.empty()) return out;
    TensorList all = in;
    all.insert(all.end(), dy.begin(), dy.end());
    const int code = gate(name, all);
    const Matrices m(name, in);
    for (size_t k = 0; k < in.size(); ++k) {
        TORCH_CHECK(dy[k].sizes() == in[k].sizes(), name, ": sizes differ, ", in[k].sizes(), " vs ",
                    dy[k].sizes());
        out.push_back(at::empty_like(in[k]));
        dy[k] = asLayoutOf(dy[k], out[k]);  // (an expanded cotangent becomes a dense one)
    }
    const toa_muon_series series = seriesOf(steps, c, eps);
    const OnDeviceOf dev(in[0]);
    int status;
    size_t kept_bytes = 0;
    if (kept) {
        kept_bytes = toa_muon_kept_bytes(code, m.rows.size(), m.rows.data(), m.cols.data(), &series, &status);
        check(status, name);
        TORCH_CHECK(kept->device() == in[0].device() && kept->scalar_type() == at::kByte &&
                        kept->is_contiguous() && kept_bytes && (size_t)kept->numel() == kept_bytes,
                    name, ": kept is not what the forward pass kept of these inputs");
    }
    const size_t bytes = toa_muon_backward_workspace(code, m.rows.size(), m.rows.data(),
                                                     m.cols.data(), &series, kept_bytes != 0, &status);
    const Tensor ws = workspaceFor(name, in[0], bytes, status);
    check(toa_muon_orthogonalize_backward_multi(
              code, m.rows.size(), m.rows.data(), m.cols.data(), viewsOf(in, m.rows.size()).data(),
              viewsOf(dy, m.rows.size()).data(), viewsOf(out, m.rows.size()).data(), &series,
              kept ? kept->data_ptr() : nullptr, kept_bytes, ws.data_ptr(), bytes, dev.stream()),
          name);
    return out;
}

// ---- the optimizer step ----------------------------------------------------------------------

// A parameter as a matrix: its first dimension times all the others, in memory order.  Columns may
// come in any order (orthogonalisation commutes with permuting them), so any dense layout whose
// first dimension is the outermost will do; a matrix may also lie column by column.
toa_muon_view matrixOf(const char *name, const Tensor &t, int64_t &rows, int64_t &cols) {
    TORCH_CHECK(t.dim() >= 2, name, ": expected matrices (at least 2 dimensions), got sizes ",
                t.sizes());
    requireDense(name, "params", t);
    rows = t.size(0);
    cols = rows ? t.numel() / rows : 0;
    if (t.numel() == 0) return {nullptr, 1, 1};
    if (t.dim() == 2) return {t.data_ptr(), rows > 1 ? t.stride(0) : cols, cols > 1 ? t.stride(1) : 1};
    TORCH_CHECK(rows == 1 || t.stride(0) == cols, name,
                ": a tensor of more than 2 dimensions must have its first one outermost, got sizes ",
                t.sizes(), " strides ", t.strides());
    return {t.data_ptr(), cols, 1};
}

bool sameOrder(const Tensor &a, const Tensor &b) {
    if (a.sizes() != b.sizes()) return false;
    for (int64_t k = 0; k < a.dim(); ++k)
        if (a.size(k) > 1 && a.stride(k) != b.stride(k)) return false;
    return true;
}

struct Span {
    char *from, *to;
    bool written;
    Span(const Tensor &t, bool written)
        : from((char *)t.data_ptr()), to(from + (size_t)t.numel() * t.element_size()),
          written(written) {}
};

// No element that the call writes may be written twice or be read as something else.
void requireApart(const char *name, std::vector<Span> &spans) {
    std::sort(spans.begin(), spans.end(), [](const Span &a, const Span &b) { return a.from < b.from; });
    char *any = nullptr, *written = nullptr;  // how far what came before reaches
    for (const Span &s : spans) {
        TORCH_CHECK(s.from >= (s.written ? any : written), name,
                    ": a tensor that is written overlaps another one (is it given twice?)");
        any = std::max(any, s.to);
        if (s.written) written = std::max(written, s.to);
    }
}

void touch(const Tensor &t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

int adjustOf(const char *name, const py::object &o) {
    if (o.is_none()) return TOA_MUON_ASPECT;
    const std::string s = o.cast<std::string>();
    if (s == "original") return TOA_MUON_ASPECT;
    if (s == "match_rms_adamw") return TOA_MUON_RMS;
    TORCH_CHECK_VALUE(s == "none", name, ": adjust_lr_fn must be None, 'original', "
                      "'match_rms_adamw' or 'none', got '", s, "'");
    return TOA_MUON_UNIT;
}

void stepMulti(const char *name, const TensorList &out, TensorList grads, const TensorList &mu,
               const py::object &scales_o, toa_muon_hyper hyper, toa_muon_series series) {
    TORCH_CHECK(grads.size() == out.size() && mu.size() == out.size(), name,
                ": tensor lists differ in length");
    if (out.empty()) return;
    for (const Tensor &t : mu)
        if (!t.is_cuda()) throw std::runtime_error("Not implemented");
    requireNoTangent(name, mu);
    TensorList all = out;
    all.insert(all.end(), grads.begin(), grads.end());
    const int code = gate(name, all);
    const at::ScalarType kept = mu[0].scalar_type();
    TORCH_CHECK(kept == out[0].scalar_type() || kept == at::kFloat || kept == at::kChar, name,
                ": the momentum must have the parameters' scalar type ", out[0].scalar_type(),
                ", Float or Char (8-bit blocks), got ", kept);
    const int kept_code = kept == at::kChar ? TOA_I8 : dtypeCode(mu[0], name);
    const bool blocks = kept_code == TOA_I8;
    TORCH_CHECK(blocks != scales_o.is_none(), name,
                blocks ? ": an 8-bit momentum needs its scales" : ": scales belong to an 8-bit momentum");
    const TensorList scales = blocks ? toTensorList(scales_o, "scales") : TensorList();
    requireNoTangent(name, scales);
    TORCH_CHECK(!blocks || scales.size() == out.size(), name, ": tensor lists differ in length");

    std::vector<int64_t> rows(out.size()), cols(out.size());
    std::vector<toa_muon_view> vo(out.size()), vg(out.size()), vm(out.size());
    std::vector<float *> vs(out.size(), nullptr);
    std::vector<Span> spans;
    for (size_t k = 0; k < out.size(); ++k) {
        TORCH_CHECK(mu[k].device() == out[0].device() && mu[k].scalar_type() == kept, name,
                    ": the momentum must live on ", out[0].device(), " with one scalar type, ", kept);
        TORCH_CHECK(grads[k].sizes() == out[k].sizes(), name, ": sizes differ, ", out[k].sizes(),
                    " vs ", grads[k].sizes());
        vo[k] = matrixOf(name, out[k], rows[k], cols[k]);
        TORCH_CHECK(out[k].numel() == 0 || sameOrder(out[k], mu[k]), name,
                    ": params and momentum must share sizes and memory layout, got ", out[k].sizes(),
                    " ", out[k].strides(), " vs ", mu[k].sizes(), " ", mu[k].strides());
        if (!sameOrder(grads[k], out[k])) grads[k] = at::empty_like(out[k]).copy_(grads[k]);
        vg[k] = vm[k] = vo[k];
        vg[k].data = grads[k].data_ptr();
        vm[k].data = mu[k].data_ptr();
        if (blocks) {
            const Tensor &s = scales[k];
            TORCH_CHECK(s.device() == out[0].device() && s.scalar_type() == at::kFloat &&
                            s.is_contiguous() && s.numel() == (out[k].numel() + 127) / 128,
                        name, ": scales must be contiguous Float tensors on ", out[0].device(),
                        " with one element for each 128 of their momentum");
            vs[k] = s.data_ptr<float>();
            if (s.numel()) spans.emplace_back(s, true);
        }
        if (out[k].numel()) {
            spans.emplace_back(out[k], true);
            spans.emplace_back(mu[k], true);
            if (hyper.apply) spans.emplace_back(grads[k], false);
        }
    }
    requireApart(name, spans);
    const OnDeviceOf dev(out[0]);
    int status;
    const size_t bytes = toa_muon_orthogonalize_workspace(code, rows.size(), rows.data(),
                                                          cols.data(), &series, 0, &status);
    const Tensor ws = workspaceFor(name, out[0], bytes, status);
    check(toa_muon_step_multi(code, kept_code, rows.size(), rows.data(), cols.data(), vo.data(),
                              vg.data(), vm.data(), blocks ? vs.data() : nullptr, &hyper, &series,
                              ws.data_ptr(), bytes, dev.stream()),
          name);
    for (size_t k = 0; k < out.size(); ++k) {
        touch(out[k]);
        touch(mu[k]);
        if (blocks) touch(scales[k]);
    }
}

py::tuple fusedStepMulti(const py::object &params_o, const py::object &updates_o,
                         const py::object &mu_o, const py::object &scales_o, double momentum,
                         double lr, bool nesterov, double weight_decay, bool maximize, int steps,
                         const Coefficients &c, double eps, const py::object &adjust_lr_fn) {
    const char *name = "muonFusedStepMulti";
    const toa_muon_hyper hyper{momentum, lr, weight_decay, nesterov, maximize,
                               adjustOf(name, adjust_lr_fn), 1};
    stepMulti(name, toTensorList(params_o, "params"), toTensorList(updates_o, "updates"),
              toTensorList(mu_o, "mu"), scales_o, hyper, seriesOf(steps, c, eps));
    return py::make_tuple(params_o, updates_o, mu_o, scales_o);
}

py::tuple forwardMulti(const py::object &updates_o, const py::object &mu_o,
                       const py::object &scales_o, double momentum, bool nesterov, int steps,
                       const Coefficients &c, double eps, const py::object &adjust_lr_fn) {
    const char *name = "muonForwardMulti";
    const toa_muon_hyper hyper{momentum, 0.0, 0.0, nesterov, 0, adjustOf(name, adjust_lr_fn), 0};
    const TensorList updates = toTensorList(updates_o, "updates");
    stepMulti(name, updates, updates, toTensorList(mu_o, "mu"), scales_o, hyper,
              seriesOf(steps, c, eps));
    return py::make_tuple(updates_o, mu_o, scales_o);
}

// ---- 8-bit blocks ------------------------------------------------------------------------------

std::tuple<TensorList, TensorList> quantizeMulti(const py::object &inputs_o) {
    const char *name = "muonQuantizeMulti";
    const TensorList in = toTensorList(inputs_o, "inputs");
    TensorList codes, scales;
    if (in.empty()) return {codes, scales};
    const int code = gate(name, in);
    std::vector<const void *> src;
    std::vector<size_t> n;
    std::vector<int8_t *> dst;
    std::vector<float *> dst_scales;
    for (const Tensor &t : in) {
        requireDense(name, "inputs", t);
        codes.push_back(at::empty_like(t, t.options().dtype(at::kChar).requires_grad(false)));
        scales.push_back(at::empty({(t.numel() + 127) / 128},
                                   t.options().dtype(at::kFloat).requires_grad(false)));
        src.push_back(t.data_ptr());
        n.push_back((size_t)t.numel());
        dst.push_back((int8_t *)codes.back().data_ptr());
        dst_scales.push_back((float *)scales.back().data_ptr());
    }
    const OnDeviceOf dev(in[0]);
    check(toa_muon_quantize_multi(code, in.size(), src.data(), n.data(), dst.data(),
                                  dst_scales.data(), dev.stream()),
          name);
    return {codes, scales};
}

py::object dequantizeMulti(const py::object &out_o, const py::object &codes_o,
                           const py::object &scales_o) {
    const char *name = "muonDequantizeMulti";
    const TensorList out = toTensorList(out_o, "out"), codes = toTensorList(codes_o, "codes"),
                     scales = toTensorList(scales_o, "scales");
    TORCH_CHECK(codes.size() == out.size() && scales.size() == out.size(), name,
                ": tensor lists differ in length");
    if (out.empty()) return out_o;
    const int code = gate(name, out);
    requireNoTangent(name, scales);
    std::vector<const int8_t *> src;
    std::vector<const float *> src_scales;
    std::vector<size_t> n;
    std::vector<void *> dst;
    std::vector<Span> spans;
    for (size_t k = 0; k < out.size(); ++k) {
        requireDense(name, "out", out[k]);
        TORCH_CHECK(codes[k].device() == out[0].device() && codes[k].scalar_type() == at::kChar &&
                        sameOrder(out[k], codes[k]),
                    name, ": codes must be Char tensors on ", out[0].device(),
                    " with the sizes and memory layout of out");
        TORCH_CHECK(scales[k].device() == out[0].device() &&
                        scales[k].scalar_type() == at::kFloat && scales[k].is_contiguous() &&
                        scales[k].numel() == (out[k].numel() + 127) / 128,
                    name, ": scales must be contiguous Float tensors on ", out[0].device(),
                    " with one element for each 128 codes");
        src.push_back((const int8_t *)codes[k].data_ptr());
        src_scales.push_back((const float *)scales[k].data_ptr());
        n.push_back((size_t)out[k].numel());
        dst.push_back(out[k].data_ptr());
        if (!n.back()) continue;
        spans.emplace_back(out[k], true);
        spans.emplace_back(codes[k], false);
        spans.emplace_back(scales[k], false);
    }
    requireApart(name, spans);
    const OnDeviceOf dev(out[0]);
    check(toa_muon_dequantize_multi(code, out.size(), src.data(), src_scales.data(), n.data(),
                                    dst.data(), dev.stream()),
          name);
    for (const Tensor &t : out) touch(t);
    return out_o;
}

}  // namespace

void defineMuonOp(py::module &mod) {
    using namespace py::literals;
    py::module m = mod.def_submodule("muon_op", "Operators for matrix-shaped parameters");
    const Coefficients c{3.4445, -4.7750, 2.0315};
    m.def("orthogonalize_multi", &orthogonalizeMulti,
          "Newton-Schulz orthogonalisation of every matrix of a list (last two dimensions)",
          "inputs"_a, "steps"_a = 5, "coefficients"_a = c, "eps"_a = 1e-7);
    m.def("orthogonalize_keep_multi", &orthogonalizeKeepMulti,
          "orthogonalize_multi, and a buffer with the iterates for the gradient, or None where it "
          "would hold more than `keep` bytes (or nothing)",
          "inputs"_a, "keep"_a, "steps"_a = 5, "coefficients"_a = c, "eps"_a = 1e-7);
    m.def("orthogonalize_backward_multi", &orthogonalizeBackwardMulti,
          "gradient of orthogonalize_multi with respect to its inputs, from what "
          "orthogonalize_keep_multi kept of the same inputs if that is given",
          "grads"_a, "inputs"_a, "steps"_a = 5, "coefficients"_a = c, "eps"_a = 1e-7,
          "kept"_a = py::none());
    m.def("forward_multi_", &forwardMulti,
          "momentum and orthogonalisation in place; mutates and returns (updates, mu, scales)",
          "updates"_a, "mu"_a, "scales"_a, "momentum"_a, py::kw_only(), "nesterov"_a = true,
          "steps"_a = 5, "coefficients"_a = c, "eps"_a = 1e-7, "adjust_lr_fn"_a = py::none());
    m.def("fused_step_multi_", &fusedStepMulti,
          "the whole optimizer step; mutates params, mu and scales, returns "
          "(params, updates, mu, scales)",
          "params"_a, "updates"_a, "mu"_a, "scales"_a, "momentum"_a, "lr"_a, py::kw_only(),
          "nesterov"_a = true, "weight_decay"_a = 0.0, "maximize"_a = false, "steps"_a = 5,
          "coefficients"_a = c, "eps"_a = 1e-7, "adjust_lr_fn"_a = py::none());
    m.def("quantize_multi", &quantizeMulti,
          "8-bit blocks of every tensor of a list -> (codes, scales)", "inputs"_a);
    m.def("dequantize_multi_", &dequantizeMulti,
          "writes what 8-bit blocks stand for into `out` and returns it", "out"_a, "codes"_a,
          "scales"_a);
}
