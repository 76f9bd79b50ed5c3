// A feed-forward block's operators: root-mean-square norm with the residual's
// addition, layers with their activation and residual, and values in 8 bits (no
// counterpart in the reference).  Each forward and each backward is one call of
// ts_hip.h; gradients go to the recorded inputs by position, as for every op.
#include "ts_hip.h"
#include "ts_host.h"

namespace ts {

namespace {

void *S() { return Runtime::get().stream(); }

const float *data_of(const Tensor *t) { return t ? t->dev() : nullptr; }

// rows of the last axis
size_t rows_of(const Tensor &t) {
    size_t n = 1;
    for (size_t k = 0; k + 1 < t.dims().size(); ++k) n *= t.dims()[k];
    return n;
}

size_t norm_cols(const Tensor &x, const Tensor &weight, const Tensor *residual, float eps) {
    if (x.dims().empty()) throw Error("rms_norm requires at least 1 dimension, got 0");
    const size_t cols = x.dims().back();
    if (weight.dims().size() != 1 || weight.dims()[0] != cols)
        throw Error("rms_norm: weight " + dims_str(weight.dims()) + " for rows of " + std::to_string(cols));
    if (residual && residual->dims() != x.dims())
        throw Error("rms_norm: residual " + dims_str(residual->dims()) + " added to " + dims_str(x.dims()));
    if (!(eps >= 0.0f)) throw Error("rms_norm: eps must not be negative");
    return cols;
}

void need_matrix(const Tensor &t, const char *what) {
    if (t.dims().size() != 2)
        throw Error(std::string(what) + " requires a matrix, got " + dims_str(t.dims()));
}

// y = norm(h), h = x (+ residual): y in full or in 8 bits
void run_norm(const Tensor &x, const Tensor *residual, const Tensor &weight, float eps, Tensor *h, Tensor *y, Packed8 *p) {
    const size_t cols = x.dims().back(), rows = rows_of(x);
    if (!x.size()) return;
    const float *xp = x.dev(), *rp = data_of(residual), *wp = weight.dev();
    float *hp = h ? h->dev_mut() : nullptr, *yp = y ? y->dev_mut() : nullptr;
    uint8_t *codes = p ? p->codes() : nullptr, *scales = p ? p->scales() : nullptr;
    const double bytes = 4.0 * x.size() * (residual ? 3 : 1) + (p ? 33.0 / 32 : 4.0) * x.size() + 4.0 * cols;
    launch(KernelClass::Reduction, bytes, "ts_hip_rms_norm", [&] {
        return p ? ts_hip_rms_norm_packed(xp, rp, wp, rows, cols, eps, hp, codes, scales, S())
                 : ts_hip_rms_norm(xp, rp, wp, rows, cols, eps, hp, yp, S());
    });
}

void check_layer(const std::vector<size_t> &weight, size_t fan_in, size_t weight_in, size_t fan_out, const Tensor *bias,
                 const Tensor *residual, const std::vector<size_t> &out) {
    if (weight.size() != 2) throw Error("linear requires a weight matrix, got " + dims_str(weight));
    if (weight_in != fan_in)
        throw Error("Inner dimensions must match: " + std::to_string(fan_in) + " vs " + std::to_string(weight_in));
    if (bias && (bias->dims().size() != 1 || bias->dims()[0] != fan_out))
        throw Error("linear: bias " + dims_str(bias->dims()) + " for " + std::to_string(fan_out) + " outputs");
    if (residual && residual->dims() != out)
        throw Error("linear: residual " + dims_str(residual->dims()) + " added to " + dims_str(out));
}

std::unique_ptr<Allocation> workspace(size_t floats) {
    return floats ? std::make_unique<Allocation>(floats) : nullptr;
}

}  // namespace

// ---- norm ----------------------------------------------------------------------

Tensor Tensor::rms_norm(const Tensor &weight, float eps) const {
    norm_cols(*this, weight, nullptr, eps);
    Tensor y = new_uninit(dims_);
    run_norm(*this, nullptr, weight, eps, nullptr, &y, nullptr);
    if ((requires_grad_ || weight.requires_grad_) && is_grad_enabled()) {
        GradFn fn{GradFn::Kind::RmsNorm};
        fn.scalar = eps;
        fn.saved = {saved(), weight.saved()};
        fn.req_left = requires_grad_;
        fn.req_right = weight.requires_grad_;
        record(y, {id_, weight.id_}, std::move(fn));
    }
    return y;
}

std::pair<Tensor, Tensor> Tensor::add_rms_norm(const Tensor &residual, const Tensor &weight, float eps) const {
    norm_cols(*this, weight, &residual, eps);
    Tensor y = new_uninit(dims_), h = new_uninit(dims_);
    run_norm(*this, &residual, weight, eps, &h, &y, nullptr);
    if (is_grad_enabled()) {
        if (requires_grad_ || residual.requires_grad_) {  // the sum, as add_tensor records it
            std::vector<size_t> ids;
            if (requires_grad_) ids.push_back(id_);
            if (residual.requires_grad_) ids.push_back(residual.id_);
            record(h, std::move(ids), GradFn{GradFn::Kind::Add});
        }
        if (h.requires_grad_ || weight.requires_grad_) {
            GradFn fn{GradFn::Kind::RmsNorm};
            fn.scalar = eps;
            fn.saved = {h.saved(), weight.saved()};
            fn.req_left = h.requires_grad_;
            fn.req_right = weight.requires_grad_;
            record(y, {h.id_, weight.id_}, std::move(fn));
        }
    }
    return {std::move(y), std::move(h)};
}

Packed8 Tensor::rms_norm_packed(const Tensor &weight, float eps) const {
    need_matrix(*this, "rms_norm_packed");
    norm_cols(*this, weight, nullptr, eps);
    Packed8 p = Packed8::new_uninit(dims_[0], dims_[1]);
    run_norm(*this, nullptr, weight, eps, nullptr, nullptr, &p);
    return p;
}

std::pair<Packed8, Tensor> Tensor::add_rms_norm_packed(const Tensor &residual, const Tensor &weight, float eps) const {
    need_matrix(*this, "add_rms_norm_packed");
    norm_cols(*this, weight, &residual, eps);
    Packed8 p = Packed8::new_uninit(dims_[0], dims_[1]);
    Tensor h = new_uninit(dims_);
    run_norm(*this, &residual, weight, eps, &h, nullptr, &p);
    if ((requires_grad_ || residual.requires_grad_) && is_grad_enabled()) {
        std::vector<size_t> ids;
        if (requires_grad_) ids.push_back(id_);
        if (residual.requires_grad_) ids.push_back(residual.id_);
        record(h, std::move(ids), GradFn{GradFn::Kind::Add});
    }
    return {std::move(p), std::move(h)};
}

std::vector<std::optional<Tensor>> rms_norm_backward(const GradFn &fn, const Tensor &go) {
    const SavedTensor &h = fn.saved[0], &w = fn.saved[1];
    const size_t cols = h.dims.back(), rows = cols ? go.size() / cols : 0;
    Tensor dh, dw;
    if (fn.req_left) dh = Tensor::new_uninit(h.dims);
    if (fn.req_right) dw = rows ? Tensor::new_uninit(w.dims) : Tensor::zeros(w.dims);
    if (go.size()) {
        const size_t ws = fn.req_right ? ts_hip_rms_norm_backward_workspace_floats(rows, cols) : 0;
        const auto work = workspace(ws);
        const float *hp = h.ptr(), *wp = w.ptr(), *gp = go.dev();
        float *dhp = fn.req_left ? dh.dev_mut() : nullptr, *dwp = fn.req_right ? dw.dev_mut() : nullptr;
        launch(KernelClass::Reduction, (fn.req_left ? 12.0 : 8.0) * go.size() + 8.0 * cols, "ts_hip_rms_norm_backward", [&] {
            return ts_hip_rms_norm_backward(hp, wp, gp, rows, cols, fn.scalar, dhp, dwp, work ? work->get() : nullptr, ws,
                                            Runtime::get().ticket(), S());
        });
    }
    std::vector<std::optional<Tensor>> r(2);
    if (fn.req_left) r[0] = std::move(dh);
    if (fn.req_right) r[1] = std::move(dw);
    return r;
}

// ---- layers --------------------------------------------------------------------

Tensor Tensor::linear(const Tensor &weight, const Tensor *bias, Activation act, const Tensor *residual,
                      Checkpoint checkpoint) const {
    if (dims_.empty()) throw Error("linear requires at least 1 dimension, got 0");
    const bool matrix = weight.dims_.size() == 2;
    std::vector<size_t> od = dims_;
    od.back() = matrix ? weight.dims_[1] : 0;
    check_layer(weight.dims_, dims_.back(), matrix ? weight.dims_[0] : 0, od.back(), bias, residual, od);
    Tensor y = new_uninit(od);
    const ts_hip_linear_shape shape = {rows_of(*this), dims_.back(), od.back()};
    const bool req_b = bias && bias->requires_grad_, req_r = residual && residual->requires_grad_;
    const bool recorded = (requires_grad_ || weight.requires_grad_ || req_b || req_r) && is_grad_enabled();
    // what the backward pass reads: X for the weight's gradient, the slopes (or X,
    // to compute them again) for every gradient but the residual's
    const bool slope_needed = recorded && act != Activation::None && (requires_grad_ || weight.requires_grad_ || req_b);
    const bool x_needed = recorded && (weight.requires_grad_ || slope_needed);
    Tensor slope;
    std::shared_ptr<Packed8> kept;
    if (x_needed && checkpoint == Checkpoint::EightBit && size_)
        kept = std::make_shared<Packed8>(Packed8::new_uninit(shape.batch, shape.fan_in));
    if (slope_needed && !kept) slope = new_uninit(od);
    if (y.size_ || kept) {
        const size_t ws = ts_hip_linear_workspace_floats(&shape);
        const auto work = workspace(ws);
        const float *xp = dev(), *wp = weight.dev(), *bp = data_of(bias), *rp = data_of(residual);
        float *yp = y.dev_mut(), *sp = slope.size_ ? slope.dev_mut() : nullptr;
        uint8_t *codes = kept ? kept->codes() : nullptr, *scales = kept ? kept->scales() : nullptr;
        launch(KernelClass::Gemm, 2.0 * shape.batch * shape.fan_in * shape.fan_out, "ts_hip_linear", [&] {
            return ts_hip_linear(&shape, xp, wp, bp, static_cast<int>(act), rp, yp, sp, codes, scales,
                                 work ? work->get() : nullptr, ws, S());
        });
    }
    if (recorded) {
        GradFn fn{GradFn::Kind::Linear};
        fn.activation = act;
        fn.input_shape = dims_;
        fn.saved = {x_needed && !kept ? saved() : SavedTensor{nullptr, dims_}, weight.saved(),
                    bias ? bias->saved() : SavedTensor{}, slope.saved()};
        fn.checkpoint = std::move(kept);
        fn.req_left = requires_grad_;
        fn.req_right = weight.requires_grad_;
        fn.has_bias = bias != nullptr;
        fn.has_residual = residual != nullptr;
        fn.req_bias = req_b;
        fn.req_residual = req_r;
        std::vector<size_t> ids = {id_, weight.id_};
        if (bias) ids.push_back(bias->id_);
        if (residual) ids.push_back(residual->id_);
        record(y, std::move(ids), std::move(fn));
    }
    return y;
}

std::vector<std::optional<Tensor>> linear_backward(const GradFn &fn, const Tensor &go) {
    const SavedTensor &x = fn.saved[0], &w = fn.saved[1], &b = fn.saved[2], &slope = fn.saved[3];
    const ts_hip_linear_shape shape = {w.dims[0] ? [&] {
                                           size_t n = 1;
                                           for (size_t d : fn.input_shape) n *= d;
                                           return n / w.dims[0];
                                       }()
                                                 : (w.dims[1] ? go.size() / w.dims[1] : 0),
                                       w.dims[0], w.dims[1]};
    Tensor dx, dw, db;
    if (fn.req_left) dx = Tensor::new_uninit(fn.input_shape);
    if (fn.req_right) dw = Tensor::new_uninit(w.dims);
    if (fn.req_bias) db = Tensor::new_uninit(b.dims);
    if (dx.size() || dw.size() || db.size()) {
        const size_t ws = ts_hip_linear_backward_workspace_floats(&shape);
        const auto work = workspace(ws);
        const float *xp = x.ptr(), *wp = w.ptr(), *bp = b.ptr(), *sp = slope.ptr(), *gp = go.dev();
        const uint8_t *codes = fn.checkpoint ? fn.checkpoint->codes() : nullptr;
        const uint8_t *scales = fn.checkpoint ? fn.checkpoint->scales() : nullptr;
        float *dxp = dx.size() ? dx.dev_mut() : nullptr, *dwp = dw.size() ? dw.dev_mut() : nullptr,
              *dbp = db.size() ? db.dev_mut() : nullptr;
        const int again = fn.checkpoint && fn.activation != Activation::None ? 1 : 0;
        const double flops = 2.0 * shape.batch * shape.fan_in * shape.fan_out * ((dxp ? 1 : 0) + (dwp ? 1 : 0) + again);
        launch(KernelClass::Gemm, flops, "ts_hip_linear_backward", [&] {
            return ts_hip_linear_backward(&shape, xp, codes, scales, wp, bp, static_cast<int>(fn.activation), sp, gp, dxp,
                                          dwp, dbp, work ? work->get() : nullptr, ws, S());
        });
    }
    std::vector<std::optional<Tensor>> r(2);
    if (fn.req_left) r[0] = std::move(dx);
    if (fn.req_right) r[1] = std::move(dw);
    if (fn.has_bias) r.push_back(fn.req_bias ? std::optional<Tensor>(std::move(db)) : std::nullopt);
    if (fn.has_residual) r.push_back(fn.req_residual ? std::optional<Tensor>(go.alias()) : std::nullopt);
    return r;
}

// ---- values in 8 bits ------------------------------------------------------------

size_t Packed8::pitch() const { return ts_hip_packed_pitch(cols_); }

Packed8 Packed8::new_uninit(size_t rows, size_t cols) {
    Packed8 p;
    p.rows_ = rows;
    p.cols_ = cols;
    if (rows && cols) {
        p.codes_ = std::make_shared<Allocation>(rows * (p.pitch() / 4));
        p.scales_ = std::make_shared<Allocation>(rows * (p.pitch() / 128));
    }
    return p;
}

Packed8 Packed8::from_device(uint8_t *codes, uint8_t *scales, size_t rows, size_t cols, std::function<void()> release) {
    Packed8 p;
    p.rows_ = rows;
    p.cols_ = cols;
    if (!rows || !cols) {
        if (release) release();
        return p;
    }
    const size_t pitch = p.pitch();
    if (pitch < cols || rows > SIZE_MAX / pitch)
        throw Error("Packed8: [" + std::to_string(rows) + ", " + std::to_string(cols) + "] is larger than any memory");
    Runtime::get();
    const size_t nc = rows * pitch, ns = nc / 32;
    if (reinterpret_cast<uintptr_t>(codes) % 16 || reinterpret_cast<uintptr_t>(scales) % 4)
        throw Error("Packed8: codes must be 16-byte aligned and scales 4-byte aligned");
    if (!codes || !scales || ts_hip_check_device_range(codes, nc) != TS_HIP_OK ||
        ts_hip_check_device_range(scales, ns) != TS_HIP_OK)
        throw Error("Packed8: the codes and scales of [" + std::to_string(rows) + ", " + std::to_string(cols) +
                    "] are not each in one allocation of device memory");
    // one release call for the two buffers
    std::shared_ptr<void> both(nullptr, [release](void *) {
        if (release) release();
    });
    p.codes_ = std::make_shared<Allocation>(reinterpret_cast<float *>(codes), nc / 4, [both]() mutable { both.reset(); });
    p.scales_ = std::make_shared<Allocation>(reinterpret_cast<float *>(scales), ns / 4, [both]() mutable { both.reset(); });
    return p;
}

Packed8 Tensor::pack8() const {
    need_matrix(*this, "pack8");
    Packed8 p = Packed8::new_uninit(dims_[0], dims_[1]);
    if (size_) {
        const float *x = dev();
        launch(KernelClass::Elementwise, 4.0 * size_ + 33.0 / 32 * size_, "ts_hip_pack8",
               [&] { return ts_hip_pack8(x, dims_[0], dims_[1], p.codes(), p.scales(), S()); });
    }
    return p;
}

Tensor Packed8::unpack() const {
    Tensor t = Tensor::new_uninit({rows_, cols_});
    if (t.size())
        launch(KernelClass::Elementwise, 4.0 * t.size() + 33.0 / 32 * t.size(), "ts_hip_unpack8",
               [&] { return ts_hip_unpack8(codes(), scales(), rows_, cols_, t.dev_mut(), S()); });
    return t;
}

Tensor Packed8::linear(const Packed8 &weight, const Tensor *bias, Activation act, const Tensor *residual) const {
    const std::vector<size_t> od = {rows_, weight.rows_};
    check_layer({weight.rows_, weight.cols_}, cols_, weight.cols_, weight.rows_, bias, residual, od);
    Tensor y = Tensor::new_uninit(od);
    if (y.size()) {
        const size_t ws = ts_hip_linear_packed_workspace_floats(rows_, cols_, weight.rows_);
        const auto work = workspace(ws);
        const float *bp = data_of(bias), *rp = data_of(residual);
        launch(KernelClass::Gemm, 2.0 * rows_ * cols_ * weight.rows_, "ts_hip_linear_packed", [&] {
            return ts_hip_linear_packed(codes(), scales(), weight.codes(), weight.scales(), rows_, cols_, weight.rows_, bp,
                                        static_cast<int>(act), rp, y.dev_mut(), work ? work->get() : nullptr, ws, S());
        });
    }
    return y;
}

}  // namespace ts
