// Dispatcher ops (torch.ops.ocb_native.*) of the kernels whose whole call is short: routing and the block-scaled linear layer.
// Their Python form (argument checks, allocation, an autograd function each way) costs several times the kernels' time for a few
// hundred tokens, so allocation, launches and the autograd node live here. The kernels themselves stay behind the C interface of
// ocb_api.h; bind_kernels() resolves them in the library that ops/_lib.py loads.

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <dlfcn.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/library.h>

#include <atomic>

#include "ocb_api.h"

namespace {

using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Kernels {
    decltype(&ocb_moe_route) route = nullptr;
    decltype(&ocb_moe_route_grad) route_grad = nullptr;
    decltype(&ocb_quantize_block_fp8) quantize = nullptr;
    decltype(&ocb_linear_block_fp8) linear = nullptr;
    decltype(&ocb_linear_block_fp8_fused) linear_fused = nullptr;
    decltype(&ocb_gemm_block_fp8) gemm_block = nullptr;
    decltype(&ocb_gemm_bf16) gemm_bf16 = nullptr;
    decltype(&ocb_grouped_gemm_bf16) grouped_gemm_bf16 = nullptr;
} kernels;

template <class F>
void resolve(void* handle, const char* name, F& fn) {
    fn = reinterpret_cast<F>(dlsym(handle, name));
    TORCH_CHECK(fn != nullptr, "the kernel library has no entry point ", name);
}

PyObject* kernel_error = nullptr;  // the class in ops/_lib.py, which lives as long as the process

struct KernelFailure : torch::PyTorchError {
    using PyTorchError::PyTorchError;
    PyObject* python_type() override { return kernel_error; }
};

void bind_kernels(c10::string_view path, int64_t error_class) {
    void* handle = dlopen(std::string(path).c_str(), RTLD_NOW | RTLD_LOCAL);
    TORCH_CHECK(handle != nullptr, "cannot load the kernel library: ", dlerror());
    kernel_error = reinterpret_cast<PyObject*>(error_class);
    resolve(handle, "ocb_moe_route", kernels.route);
    resolve(handle, "ocb_moe_route_grad", kernels.route_grad);
    resolve(handle, "ocb_quantize_block_fp8", kernels.quantize);
    resolve(handle, "ocb_linear_block_fp8", kernels.linear);
    resolve(handle, "ocb_linear_block_fp8_fused", kernels.linear_fused);
    resolve(handle, "ocb_gemm_block_fp8", kernels.gemm_block);
    resolve(handle, "ocb_gemm_bf16", kernels.gemm_bf16);
    resolve(handle, "ocb_grouped_gemm_bf16", kernels.grouped_gemm_bf16);
}

std::atomic<int64_t> launches{0};
using RangePush = void (*)(const char*);
using RangePop = void (*)();
std::atomic<RangePush> range_push{nullptr};  // both or neither
std::atomic<RangePop> range_pop{nullptr};

int64_t launch_count() { return launches.load(std::memory_order_relaxed); }

void set_ranges(int64_t push, int64_t pop) {
    range_push.store(nullptr);
    range_pop.store(reinterpret_cast<RangePop>(pop));
    range_push.store(reinterpret_cast<RangePush>(push));
}

struct Range {
    RangePop pop = nullptr;
    explicit Range(const char* name) {
        const RangePush push = range_push.load();
        if (push == nullptr) return;
        pop = range_pop.load();
        push(name);
    }
    ~Range() {
        if (pop != nullptr) pop();
    }
};

template <class Launcher, class... Args>
void launch(const char* name, Launcher launcher, Args... args) {
    launches.fetch_add(1, std::memory_order_relaxed);
    const Range range(name);
    const int rc = launcher(args...);
    if (rc != 0) throw KernelFailure(std::string(name) + " failed with code " + std::to_string(rc));
}

int dtype_code(const Tensor& t) { return t.scalar_type() == at::kBFloat16 ? OCB_BF16 : OCB_F32; }

cudaStream_t stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

const float* floats(const optional<Tensor>& t) { return t.has_value() && t->defined() ? t->const_data_ptr<float>() : nullptr; }

// ---- routing -----------------------------------------------------------------------------------------------------------

struct RouteOptions {
    int top_k, sigmoid, n_groups, top_groups, normalize;
};

std::tuple<Tensor, Tensor, Tensor, Tensor> run_route(const Tensor& logits, const optional<Tensor>& bias, const RouteOptions& o) {
    const c10::cuda::OptionalCUDAGuard guard(logits.device());
    const int64_t n = logits.size(0), e = logits.size(1);
    TORCH_CHECK_VALUE(n <= INT32_MAX, "routing takes fewer than 2^31 tokens");
    const auto opt = logits.options();
    Tensor weights = at::empty({n, o.top_k}, opt.dtype(at::kFloat)), experts = at::empty({n, o.top_k}, opt.dtype(at::kLong));
    Tensor scores = at::empty({n, e}, opt.dtype(at::kFloat)), counts = at::empty({e}, opt.dtype(at::kInt));
    launch("ocb_moe_route", kernels.route, logits.const_data_ptr(), scores.mutable_data_ptr<float>(), weights.mutable_data_ptr<float>(),
                        reinterpret_cast<long long*>(experts.mutable_data_ptr<int64_t>()), counts.mutable_data_ptr<int>(), floats(bias),
                        static_cast<int>(n), static_cast<int>(e), o.top_k, o.sigmoid, o.normalize, o.n_groups, o.top_groups,
                        logits.stride(0), dtype_code(logits), stream_of(logits));
    return {weights, experts, scores, counts};
}

struct Route : torch::autograd::Function<Route> {
    static variable_list forward(AutogradContext* ctx, const Tensor& logits, const optional<Tensor>& bias, const RouteOptions& o) {
        auto [weights, experts, scores, counts] = run_route(logits, bias, o);
        ctx->save_for_backward({o.sigmoid ? logits : scores, experts});
        ctx->saved_data["sigmoid"] = static_cast<int64_t>(o.sigmoid);
        ctx->saved_data["normalize"] = static_cast<int64_t>(o.normalize);
        ctx->saved_data["bf16"] = logits.scalar_type() == at::kBFloat16;
        ctx->mark_non_differentiable({experts, counts});
        ctx->set_materialize_grads(false);
        return {weights, experts, scores, counts};
    }

    // The gradient in tensor operations, for a graph that is going to be differentiated itself. kept: the logits (sigmoid) or the
    // scores, with their own history. Same formulas as the kernel's.
    static Tensor differentiable(const Tensor& kept, const Tensor& experts, const Tensor& d_weights, const Tensor& d_scores, bool sigmoid,
                                 int64_t normalize) {
        const Tensor x = kept.to(at::kFloat), p = sigmoid ? x.sigmoid() : x, s = sigmoid ? p + 1e-7 : x;
        Tensor d = d_scores.defined() ? d_scores.to(at::kFloat) : at::zeros_like(s);
        if (d_weights.defined()) {
            Tensor g = d_weights.to(at::kFloat);
            if (normalize != 0) {
                const Tensor chosen = s.gather(1, experts), top = chosen.detach().amax(1, true), none = top < 0x1p-120;
                const Tensor scale = at::ldexp(at::ones_like(top), 1 - std::get<1>(at::frexp(top))).masked_fill(none, 0.0);
                const Tensor c = (chosen * scale).masked_fill(none, 1.0), total = (normalize == 1 ? c : c * c).sum(1, true);
                const Tensor norm = normalize == 1 ? total : total.sqrt(), w = c / norm, along = (g * w).sum(1, true);
                g = (g - (normalize == 1 ? along : along * w)) / norm * scale;
            }
            d = d.scatter_add(1, experts, g);
        }
        return sigmoid ? d * p * (-x).sigmoid() : s * (d - (d * s).sum(1, true));
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const Tensor &d_weights = grads[0], &d_scores = grads[2];
        if (!d_weights.defined() && !d_scores.defined()) return {Tensor(), Tensor(), Tensor()};
        const auto saved = ctx->get_saved_variables();
        const Tensor &kept = saved[0], &experts = saved[1];
        const c10::cuda::OptionalCUDAGuard guard(kept.device());
        const int sigmoid = static_cast<int>(ctx->saved_data["sigmoid"].toInt());
        if (at::GradMode::is_enabled())
            return {differentiable(kept, experts, d_weights, d_scores, sigmoid != 0, ctx->saved_data["normalize"].toInt())
                        .to(ctx->saved_data["bf16"].toBool() ? at::kBFloat16 : at::kFloat), Tensor(), Tensor()};
        const Tensor dw = d_weights.defined() ? d_weights.to(at::kFloat).contiguous() : d_weights;
        const Tensor ds = d_scores.defined() ? d_scores.to(at::kFloat).contiguous() : d_scores;
        Tensor d_logits = at::empty({kept.size(0), kept.size(1)}, kept.options().dtype(ctx->saved_data["bf16"].toBool() ? at::kBFloat16 : at::kFloat));
        launch("ocb_moe_route_grad", kernels.route_grad, sigmoid ? nullptr : kept.const_data_ptr<float>(), sigmoid ? kept.const_data_ptr() : nullptr,
                                 reinterpret_cast<const long long*>(experts.const_data_ptr<int64_t>()),
                                 dw.defined() ? dw.const_data_ptr<float>() : nullptr, ds.defined() ? ds.const_data_ptr<float>() : nullptr,
                                 d_logits.mutable_data_ptr(), static_cast<int>(kept.size(0)), static_cast<int>(kept.size(1)),
                                 static_cast<int>(experts.size(1)), sigmoid, static_cast<int>(ctx->saved_data["normalize"].toInt()),
                                 kept.stride(0), dtype_code(d_logits), stream_of(kept));
        return {d_logits, Tensor(), Tensor()};
    }
};

std::tuple<Tensor, Tensor, Tensor, Tensor> route(const Tensor& logits, int64_t top_k, bool sigmoid, const optional<Tensor>& bias,
                                                 int64_t n_groups, int64_t top_groups, int64_t normalize) {
    const RouteOptions o{static_cast<int>(top_k), sigmoid, static_cast<int>(n_groups), static_cast<int>(top_groups),
                         static_cast<int>(normalize)};
    TORCH_CHECK(!logits._fw_grad(0).defined(), "the routing kernel computes no tangents: routing differentiates forwards in tensor operations");
    if (!logits.requires_grad() || !at::GradMode::is_enabled()) return run_route(logits, bias, o);
    const variable_list out = Route::apply(logits, bias, o);
    return {out[0], out[1], out[2], out[3]};
}

// ---- block-scaled linear layer -------------------------------------------------------------------------------------------

int64_t blocks(int64_t n) { return (n + 127) / 128; }
int64_t pitch_of(int64_t cols) { return (cols + 15) & -16; }

Tensor bytes(int64_t n, const Tensor& like) { return at::empty({n}, like.options().dtype(at::kByte)); }

// A [rows, cols] matrix in bf16 with contiguous rows.
Tensor matrix(const Tensor& t, int64_t cols) {
    Tensor m = t.dim() == 2 ? t : t.reshape({cols == 0 ? t.numel() : t.numel() / cols, cols});
    if (m.scalar_type() != at::kBFloat16) m = m.to(at::kBFloat16);
    return m.stride(1) == 1 || m.size(1) == 1 ? m : m.contiguous();
}

// The same where its rows start on 16-byte boundaries, else a copy (rows broadcast from one have stride 0).
Tensor aligned(const Tensor& m) {
    const bool fits = m.stride(0) >= m.size(1) && m.stride(0) % 8 == 0 && reinterpret_cast<uintptr_t>(m.const_data_ptr()) % 16 == 0;
    return fits ? m : m.clone(at::MemoryFormat::Contiguous);
}

// The kernels round 32-bit sizes up to tiles.
void check_sizes(int64_t m, int64_t n, int64_t k) {
    constexpr int64_t most = INT32_MAX - 512;
    TORCH_CHECK_VALUE(m <= most && n <= most && k <= most, "the block-scaled product takes no dimension above ", most);
}

// `groups` stacked matrices [rows, cols]: their codes [rows, cols rounded up to 16] and behind them the scales of their tiles.
Tensor tile_buffer(const Tensor& weight, int64_t groups) {
    const c10::cuda::OptionalCUDAGuard guard(weight.device());
    const Tensor w = matrix(weight, weight.size(1));
    const int64_t rows = w.size(0) / groups, cols = w.size(1), pitch = pitch_of(cols), codes = groups * rows * pitch;
    check_sizes(rows, cols, groups);
    Tensor buffer = bytes(codes + 4 * groups * blocks(rows) * blocks(cols), w);
    if (rows == 0 || cols == 0) return buffer;
    uint8_t* at = buffer.mutable_data_ptr<uint8_t>();
    launch("ocb_quantize_block_fp8", kernels.quantize, w.const_data_ptr(), nullptr, nullptr, nullptr, nullptr, at, reinterpret_cast<float*>(at + codes),
                           static_cast<int>(groups), static_cast<int>(rows), static_cast<int>(cols), w.stride(0), pitch,
                           rows * w.stride(0), rows * pitch, stream_of(w));
    return buffer;
}

// Where the tile-quantised matrices [rows, cols] of a product are.
struct Weight {
    const void* codes;
    const float* scales;
    int64_t rows, cols, pitch, group_bytes;
    int64_t s_group, s_row, s_col;  // strides of the scales between groups, rows and columns of tiles
    int64_t groups;
};

Weight in_buffer(const Tensor& tiles, int64_t groups, int64_t rows, int64_t cols) {
    const uint8_t* at = tiles.const_data_ptr<uint8_t>();
    const int64_t pitch = pitch_of(cols);
    return {at, reinterpret_cast<const float*>(at + groups * rows * pitch), rows, cols, pitch, rows * pitch,
            blocks(rows) * blocks(cols), blocks(cols), 1, groups};
}

// x by rows times W (transposed or not); `columns`: also x by columns.
Tensor product(const Tensor& x, const Weight& w, bool trans, const int* offsets, Tensor* columns, int64_t status) {
    const int64_t m = x.size(0), k = x.size(1), n = trans ? w.rows : w.cols;
    check_sizes(m, n, k);
    Tensor out = at::empty({m, n}, x.options());
    const int64_t pitch = pitch_of(k), codes = m * pitch;
    if (columns != nullptr) *columns = bytes(codes + 4 * blocks(m) * k, x);
    if (m == 0 || n == 0) return out;
    if (k == 0) return out.zero_();
    Tensor rows;  // few rows are quantised inside the product
    if (kernels.linear_fused(static_cast<int>(m), static_cast<int>(w.groups), offsets != nullptr) == 0) rows = bytes(codes + 4 * blocks(k) * m, x);
    uint8_t* at = rows.defined() ? rows.mutable_data_ptr<uint8_t>() : nullptr;
    uint8_t* at_c = columns != nullptr ? columns->mutable_data_ptr<uint8_t>() : nullptr;
    launch("ocb_linear_block_fp8", kernels.linear, x.const_data_ptr(), x.stride(0), at, at != nullptr ? reinterpret_cast<float*>(at + codes) : nullptr, at_c,
                         at_c != nullptr ? reinterpret_cast<float*>(at_c + codes) : nullptr, pitch, w.codes, w.scales, offsets,
                         static_cast<int>(w.groups), out.mutable_data_ptr(), static_cast<int>(m), static_cast<int>(n),
                         static_cast<int>(k), w.pitch, w.group_bytes, trans ? w.s_col : w.s_row, trans ? w.s_row : w.s_col, w.s_group,
                         trans ? 0 : 1, n, 0, reinterpret_cast<int*>(status), stream_of(x));
    return out;
}

// x [M, K] by rows times checked codes [(G,) N, K] (trans) or [(G,) K, N] with their tile scales.
Tensor block_product(const Tensor& x, const Tensor& codes, const Tensor& scales, const optional<Tensor>& offsets, bool trans, int64_t status) {
    const c10::cuda::OptionalCUDAGuard guard(x.device());
    const bool grouped = codes.dim() == 3;
    const int64_t groups = grouped ? codes.size(0) : 1, rows = codes.size(-2), cols = codes.size(-1);
    const int64_t pitch = rows > 1 ? codes.stride(-2) : pitch_of(cols);
    const Weight w{codes.const_data_ptr(), scales.const_data_ptr<float>(), rows, cols, pitch, groups > 1 ? codes.stride(0) : rows * pitch,
                   grouped ? scales.stride(0) : 0, scales.stride(-2), scales.stride(-1), groups};
    return product(matrix(x, trans ? cols : rows), w, trans, offsets.has_value() ? offsets->const_data_ptr<int>() : nullptr, nullptr, status);
}

// The gradients of a layer whose own derivative is not built: where a graph of them is kept, differentiating it is an error.
variable_list first_order(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    for (Tensor& g : grads)
        if (g.defined()) g = g.detach().requires_grad_(true);
    const auto error = std::make_shared<torch::autograd::DelayedError>("the block-scaled layers have no second derivative",
                                                                       static_cast<int>(grads.size()));
    return (*error)(std::move(grads));
}

// What the kernels write to and read from by address alone: `main_grad` of a weight w (rows of a dense one may be apart), and its
// codes and scales as tile_buffer() makes them.
void check_main_grad(const Tensor& grad, int64_t rows, int64_t cols, at::Device device, bool stacked) {
    TORCH_CHECK_VALUE(grad.scalar_type() == at::kFloat && grad.device() == device, "main_grad must be float32 on ", device, ", got ",
                      grad.scalar_type(), " on ", grad.device());
    const bool fits = stacked ? grad.numel() == rows * cols && grad.is_contiguous()
                              : grad.dim() == 2 && grad.size(0) == rows && grad.size(1) == cols && (cols <= 1 || grad.stride(1) == 1) &&
                                    (rows <= 1 || grad.stride(0) >= cols);
    TORCH_CHECK_VALUE(fits, "main_grad of shape ", grad.sizes(), " and strides ", grad.strides(), " does not fit a weight of shape [", rows,
                      ", ", cols, "]: ", stacked ? "it" : "rows", " must be contiguous");
}

// The `main_grad` that the weight's Python object has by now (undefined: none), and the note there that it has been added to. Only
// asked for a weight that had one in the forward pass: taking the interpreter's lock costs a few microseconds.
Tensor main_grad_of(const Tensor& weight) {
    const pybind11::gil_scoped_acquire gil;
    const auto object = pybind11::reinterpret_steal<pybind11::object>(THPVariable_Wrap(weight));
    const auto grad = pybind11::getattr(object, "main_grad", pybind11::none());
    return THPVariable_Check(grad.ptr()) ? THPVariable_Unpack(grad.ptr()) : Tensor();
}
void note_main_grad(const Tensor& weight) {
    const pybind11::gil_scoped_acquire gil;
    const auto object = pybind11::reinterpret_steal<pybind11::object>(THPVariable_Wrap(weight));
    if (pybind11::hasattr(object, "grad_added_to_main_grad")) pybind11::setattr(object, "grad_added_to_main_grad", pybind11::bool_(true));
}

void check_cached(const optional<Tensor>& tiles, const Tensor& w, int64_t groups) {
    if (!tiles.has_value()) return;
    const int64_t rows = w.size(0) / groups, cols = w.size(1);
    TORCH_CHECK_VALUE(tiles->scalar_type() == at::kByte && tiles->device() == w.device() && tiles->is_contiguous() &&
                          tiles->numel() == groups * (rows * pitch_of(cols) + 4 * blocks(rows) * blocks(cols)),
                      "the kept 8-bit form (", tiles->numel(), " x ", tiles->scalar_type(), " on ", tiles->device(),
                      ") is not that of a weight of shape ", w.sizes(), " on ", w.device());
}

struct BlockLinear : torch::autograd::Function<BlockLinear> {
    // weight: what the gradient belongs to; w: its bf16 values [N, K]
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Tensor& w, const optional<Tensor>& cached,
                          bool has_main_grad, bool needs_dw, bool high_precision, int64_t status) {
        const c10::cuda::OptionalCUDAGuard guard(x.device());
        const int64_t n = w.size(0), k = w.size(1);
        const Tensor x2 = matrix(x, k), tiles = cached.has_value() ? *cached : tile_buffer(w, 1);
        const bool in_fp8 = needs_dw && !high_precision;
        Tensor columns;  // what the backward pass keeps of x: its column-scaled form, one byte per element
        Tensor y = product(x2, in_buffer(tiles, 1, n, k), true, nullptr, in_fp8 ? &columns : nullptr, status);
        ctx->save_for_backward({tiles, in_fp8 ? columns : needs_dw ? x2 : Tensor()});
        if (has_main_grad) ctx->saved_data["weight"] = weight;
        ctx->saved_data["m"] = x2.size(0);
        ctx->saved_data["n"] = n;
        ctx->saved_data["k"] = k;
        ctx->saved_data["x_shape"] = x.sizes().vec();
        ctx->saved_data["x_dtype"] = x.scalar_type();
        ctx->saved_data["w_dtype"] = weight.scalar_type();
        ctx->saved_data["needs_dx"] = x.requires_grad();
        ctx->saved_data["needs_dw"] = needs_dw;
        ctx->saved_data["in_fp8"] = in_fp8;
        ctx->saved_data["status"] = status;
        auto shape = x.sizes().vec();
        shape.back() = n;
        return y.view(shape);
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &tiles = saved[0], &kept = saved[1];
        const int64_t m = ctx->saved_data["m"].toInt(), n = ctx->saved_data["n"].toInt(), k = ctx->saved_data["k"].toInt();
        const int64_t status = ctx->saved_data["status"].toInt();
        const bool needs_dw = ctx->saved_data["needs_dw"].toBool(), in_fp8 = ctx->saved_data["in_fp8"].toBool();
        const c10::cuda::OptionalCUDAGuard guard(tiles.device());
        const Tensor dy = matrix(grads[0], n);
        Tensor dx, dw, columns;
        if (ctx->saved_data["needs_dx"].toBool()) {
            dx = product(dy, in_buffer(tiles, 1, n, k), false, nullptr, in_fp8 ? &columns : nullptr, status);
            dx = dx.view(ctx->saved_data["x_shape"].toIntVector()).to(ctx->saved_data["x_dtype"].toScalarType());
        }
        if (needs_dw) {
            const auto w_dtype = ctx->saved_data["w_dtype"].toScalarType();
            const auto weight = ctx->saved_data.find("weight");
            const Tensor main_grad = weight != ctx->saved_data.end() ? main_grad_of(weight->second.toTensor()) : Tensor();
            const bool accumulate = main_grad.defined();
            if (accumulate) check_main_grad(main_grad, n, k, dy.device(), false);
            // the kernels write bf16 or fp32, whichever the parameter has
            Tensor out = accumulate ? main_grad : at::empty({n, k}, dy.options().dtype(w_dtype == at::kBFloat16 ? at::kBFloat16 : at::kFloat));
            const int epilogue = out.scalar_type() == at::kBFloat16 ? 0 : accumulate ? 1 : 2;
            if (m == 0 || n == 0 || k == 0) {
                if (!accumulate) out.zero_();
            } else if (!in_fp8) {
                const Tensor a = aligned(dy), b = aligned(kept);
                launch("ocb_gemm_bf16", kernels.gemm_bf16, a.const_data_ptr(), b.const_data_ptr(), out.mutable_data_ptr(), static_cast<int>(n),
                                        static_cast<int>(k), static_cast<int>(m), a.stride(0), b.stride(0), out.stride(0), 1, 1, epilogue, reinterpret_cast<int*>(status), stream_of(dy));
            } else {
                const int64_t pitch_y = pitch_of(n), pitch_x = pitch_of(k);
                if (!columns.defined()) {
                    columns = bytes(m * pitch_y + 4 * blocks(m) * n, dy);
                    uint8_t* at = columns.mutable_data_ptr<uint8_t>();
                    launch("ocb_quantize_block_fp8", kernels.quantize, dy.const_data_ptr(), nullptr, nullptr, at, reinterpret_cast<float*>(at + m * pitch_y), nullptr,
                                           nullptr, 1, static_cast<int>(m), static_cast<int>(n), dy.stride(0), pitch_y, 0, 0, stream_of(dy));
                }
                const uint8_t *a = columns.const_data_ptr<uint8_t>(), *b = kept.const_data_ptr<uint8_t>();
                launch("ocb_gemm_block_fp8", kernels.gemm_block, a, b, out.mutable_data_ptr(), reinterpret_cast<const float*>(a + m * pitch_y),
                                         reinterpret_cast<const float*>(b + m * pitch_x), nullptr, 1, static_cast<int>(n),
                                         static_cast<int>(k), static_cast<int>(m), pitch_y, pitch_x, out.stride(0), 0, n, 1, 0, k, 1, 0, 0,
                                         1, 1, epilogue, reinterpret_cast<int*>(status), stream_of(dy));
            }
            if (accumulate) note_main_grad(weight->second.toTensor());
            else dw = out.scalar_type() == w_dtype ? out : out.to(w_dtype);
        }
        return first_order({dx, dw, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()});
    }
};

// The experts' layer: rows sorted by group, weights stacked [G * N, K] (trans) or [G * K, N]; weight gradient in bf16.
struct BlockGroupedLinear : torch::autograd::Function<BlockGroupedLinear> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Tensor& w, const Tensor& offsets,
                          const optional<Tensor>& cached, bool has_main_grad, bool trans, bool needs_dw, int64_t status) {
        const c10::cuda::OptionalCUDAGuard guard(x.device());
        const int64_t groups = offsets.size(0) - 1, rows = w.size(0) / groups, cols = w.size(1);
        const Tensor x2 = matrix(x, x.size(1)), tiles = cached.has_value() ? *cached : tile_buffer(w, groups);
        Tensor y = product(x2, in_buffer(tiles, groups, rows, cols), trans, offsets.const_data_ptr<int>(), nullptr, status);
        ctx->save_for_backward({tiles, offsets, needs_dw ? x2 : Tensor()});
        if (has_main_grad) ctx->saved_data["weight"] = weight;
        ctx->saved_data["rows"] = rows;
        ctx->saved_data["cols"] = cols;
        ctx->saved_data["trans"] = trans;
        ctx->saved_data["x_dtype"] = x.scalar_type();
        ctx->saved_data["w_dtype"] = weight.scalar_type();
        ctx->saved_data["needs_dx"] = x.requires_grad();
        ctx->saved_data["needs_dw"] = needs_dw;
        ctx->saved_data["status"] = status;
        return y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &tiles = saved[0], &offsets = saved[1], &x = saved[2];
        const int64_t groups = offsets.size(0) - 1, rows = ctx->saved_data["rows"].toInt(), cols = ctx->saved_data["cols"].toInt();
        const int64_t status = ctx->saved_data["status"].toInt();
        const bool trans = ctx->saved_data["trans"].toBool();
        const c10::cuda::OptionalCUDAGuard guard(tiles.device());
        const Tensor dy = matrix(grads[0], trans ? rows : cols);
        Tensor dx, dw;
        if (ctx->saved_data["needs_dx"].toBool())
            dx = product(dy, in_buffer(tiles, groups, rows, cols), !trans, offsets.const_data_ptr<int>(), nullptr, status)
                     .to(ctx->saved_data["x_dtype"].toScalarType());
        if (ctx->saved_data["needs_dw"].toBool()) {
            const auto w_dtype = ctx->saved_data["w_dtype"].toScalarType();
            const auto weight = ctx->saved_data.find("weight");
            const Tensor main_grad = weight != ctx->saved_data.end() ? main_grad_of(weight->second.toTensor()) : Tensor();
            const bool accumulate = main_grad.defined();
            if (accumulate) check_main_grad(main_grad, groups * rows, cols, dy.device(), true);
            Tensor out = accumulate ? main_grad
                                    : at::empty({groups * rows, cols}, dy.options().dtype(w_dtype == at::kBFloat16 ? at::kBFloat16 : at::kFloat));
            if (dy.size(0) == 0) {
                if (!accumulate) out.zero_();
            } else {
                const Tensor a = aligned(trans ? dy : x), b = aligned(trans ? x : dy);
                launch("ocb_grouped_gemm_bf16", kernels.grouped_gemm_bf16, a.const_data_ptr(), b.const_data_ptr(), out.mutable_data_ptr(), offsets.const_data_ptr<int>(),
                                                static_cast<int>(groups), 2, static_cast<int>(dy.size(0)), static_cast<int>(rows),
                                                static_cast<int>(cols), 0, a.stride(0), b.stride(0), cols, 1,
                                                out.scalar_type() == at::kBFloat16 ? 0 : accumulate ? 1 : 2,
                                                reinterpret_cast<int*>(status), stream_of(dy));
            }
            if (accumulate) note_main_grad(weight->second.toTensor());
            else dw = out.scalar_type() == w_dtype ? out : out.to(w_dtype);
        }
        return first_order({dx, dw, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()});
    }
};

Tensor block_grouped_linear(const Tensor& x, const Tensor& weight, const Tensor& w, const Tensor& offsets, const optional<Tensor>& cached,
                            const optional<Tensor>& main_grad, bool trans, int64_t status) {
    const bool needs_dw = at::GradMode::is_enabled() && (weight.requires_grad() || main_grad.has_value());
    if (needs_dw && main_grad.has_value()) check_main_grad(*main_grad, w.size(0), w.size(1), w.device(), true);
    check_cached(cached, w, offsets.size(0) - 1);
    return BlockGroupedLinear::apply(x, weight, w, offsets, cached, main_grad.has_value(), trans, needs_dw, status);
}

Tensor block_linear(const Tensor& x, const Tensor& weight, const Tensor& w, const optional<Tensor>& cached,
                    const optional<Tensor>& main_grad, bool high_precision, int64_t status) {
    const bool needs_dw = at::GradMode::is_enabled() && (weight.requires_grad() || main_grad.has_value());
    if (needs_dw && main_grad.has_value()) check_main_grad(*main_grad, w.size(0), w.size(1), w.device(), false);
    check_cached(cached, w, 1);
    return BlockLinear::apply(x, weight, w, cached, main_grad.has_value(), needs_dw, high_precision, status);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(ocb_native, m) {
    m.def("bind_kernels(str path, int error_class) -> ()", &bind_kernels);
    m.def("launch_count() -> int", &launch_count);
    m.def("set_ranges(int push, int pop) -> ()", &set_ranges);
    m.def("route(Tensor logits, int top_k, bool sigmoid, Tensor? bias, int n_groups, int top_groups, int normalize) -> (Tensor, Tensor, Tensor, Tensor)",
          &route);
    m.def("block_tile_buffer(Tensor w, int groups) -> Tensor", &tile_buffer);
    m.def("block_grouped_linear(Tensor x, Tensor weight, Tensor w, Tensor offsets, Tensor? cached, Tensor? main_grad, bool trans, int status) -> Tensor",
          &block_grouped_linear);
    m.def("block_product(Tensor x, Tensor codes, Tensor scales, Tensor? offsets, bool trans, int status) -> Tensor", &block_product);
    m.def("block_linear(Tensor x, Tensor weight, Tensor w, Tensor? cached, Tensor? main_grad, bool high_precision, int status) -> Tensor",
          &block_linear);
}
