// Torch side of the differentiable operators: checks of arguments, output tensors, autograd
// nodes. The computation is in liblattice_b200.so, behind its C ABI; this file only names
// device pointers and streams. It is C++ because a training step on a small tensor is bound by
// the host: a forward and backward pass over 8 x 256 values took 166 us with the nodes and the
// calls in Python, most of it in the interpreter and in the autograd engine's own thread.
#include <torch/extension.h>

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <string>
#include <tuple>
#include <vector>

#include "lattice_b200.h"

// A contract violation is a ValueError in Python.
#define REQUIRE(condition, ...)                            \
    do {                                                   \
        if (!(condition)) {                                \
            throw py::value_error(c10::str(__VA_ARGS__));  \
        }                                                  \
    } while (0)

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptionalTensor = std::optional<Tensor>;

void check(int code) {
    if (code == LAT_OK) {
        return;
    }
    const std::string message = lat_last_error();
    REQUIRE(code != LAT_INVALID_ARGUMENT, message);
    TORCH_CHECK(false, message);
}

void require_cuda(const Tensor& t, const char* name) {
    TORCH_CHECK(t.is_cuda(), name, " must live on a CUDA device: this build has no CPU route.");
}

int dtype_code(const Tensor& t) {
    if (t.scalar_type() == at::kFloat) {
        return LAT_F32;
    }
    REQUIRE(t.scalar_type() == at::kHalf, "this operator supports float32 and float16 tensors.");
    return LAT_F16;
}

// A feature matrix whose rows are dense; its rows may lie apart.
struct Matrix {
    Tensor t;
    int64_t rows, channels, stride;
};

Matrix matrix(const Tensor& t, const char* name) {
    require_cuda(t, name);
    REQUIRE(t.dim() == 2, name, " must have shape (N, C).");
    Tensor dense = t.stride(1) == 1 ? t : t.contiguous();
    REQUIRE(t.size(1) <= 0x7fffffff, name, " has too many channels.");
    const int64_t stride = dense.size(0) > 1 ? dense.stride(0) : dense.size(1);
    return {dense, dense.size(0), dense.size(1), stride};
}

Matrix matching(const Tensor& t, const Matrix& like, const char* name) {
    require_cuda(t, name);
    REQUIRE(t.sizes() == like.t.sizes() && t.scalar_type() == like.t.scalar_type() &&
                          t.device() == like.t.device(),
                      name, " must match the features in shape, dtype and device.");
    return matrix(t, name);
}

const void* data(const Tensor& t) { return t.defined() && t.numel() > 0 ? t.const_data_ptr() : nullptr; }
void* mutable_data(const Tensor& t) { return t.defined() && t.numel() > 0 ? t.data_ptr() : nullptr; }
const float* floats(const Tensor& t) { return static_cast<const float*>(data(t)); }
float* mutable_floats(const Tensor& t) { return static_cast<float*>(mutable_data(t)); }

// Optional vector of `length` values beside the features; undefined without one.
Tensor vector_argument(const Tensor& t, const char* name, int64_t length, const Matrix& like, at::ScalarType type) {
    if (!t.defined()) {
        return t;
    }
    REQUIRE(t.is_cuda(), name, " must be a CUDA tensor.");
    REQUIRE(t.device() == like.t.device(), name, " must be on the same device as the features.");
    REQUIRE(t.scalar_type() == type, name, " dtype must match the features.");
    REQUIRE(t.dim() == 1 && t.size(0) == length, name, " must have shape (", length, ",).");
    return t.contiguous();
}

Tensor new_like(const Matrix& like, at::IntArrayRef sizes) { return at::empty(sizes, like.t.options()); }
Tensor new_floats(const Matrix& like, at::IntArrayRef sizes) { return at::empty(sizes, like.t.options().dtype(at::kFloat)); }

Tensor new_workspace(const Matrix& like, size_t bytes) {
    return at::empty({static_cast<int64_t>(bytes)}, like.t.options().dtype(at::kByte));
}

void* stream_of(const Matrix& like) { return at::cuda::getCurrentCUDAStream(like.t.device().index()).stream(); }

bool wants_gradient(std::initializer_list<Tensor> tensors) {
    if (!at::GradMode::is_enabled()) {
        return false;
    }
    for (const Tensor& t : tensors) {
        if (t.defined() && t.requires_grad()) {
            return true;
        }
    }
    return false;
}

OptionalTensor none_if_undefined(const Tensor& t) { return t.defined() ? OptionalTensor(t) : std::nullopt; }
Tensor plain(const OptionalTensor& t) { return t.value_or(Tensor()); }

// The same values behind a node that raises `message` when someone differentiates through them. The
// node attaches itself only to what requires a gradient, so every tensor enters it as one that does.
variable_list raising(variable_list values, const char* message) {
    for (Tensor& t : values) {
        if (t.defined()) {
            t = t.detach().requires_grad_(true);
        }
    }
    const auto node = std::make_shared<torch::autograd::DelayedError>(message, static_cast<int64_t>(values.size()));
    return (*node)(std::move(values));
}

// The backward passes are not differentiable themselves: with a graph of them asked for, their
// results say so when someone tries.
variable_list once(variable_list grads) {
    return at::GradMode::is_enabled() ? raising(std::move(grads), "this operator has no second derivative") : grads;
}

// ---- row normalisation ------------------------------------------------------------------------

std::tuple<Tensor, Tensor, Tensor> row_norm_forward(
    const Tensor& feats_in, const Tensor& weight_in, const Tensor& bias_in, double eps, bool rms
) {
    const Matrix feats = matrix(feats_in, "feats");
    const int dtype = dtype_code(feats.t);
    const Tensor weight = vector_argument(weight_in, "weight", feats.channels, feats, feats.t.scalar_type());
    const Tensor bias = vector_argument(bias_in, "bias", feats.channels, feats, feats.t.scalar_type());
    const Tensor out = new_like(feats, {feats.rows, feats.channels});
    const Tensor mean = rms ? Tensor() : new_floats(feats, {feats.rows});
    const Tensor rstd = new_floats(feats, {feats.rows});
    const c10::cuda::CUDAGuard guard(feats.t.device());
    check(lat_row_norm_forward(
        dtype, rms, data(feats.t), feats.rows, static_cast<int32_t>(feats.channels), feats.stride, data(weight),
        data(bias), static_cast<float>(eps), mutable_data(out), mutable_floats(mean), mutable_floats(rstd),
        stream_of(feats)));
    return {out, mean, rstd};
}

std::tuple<Tensor, Tensor, Tensor> row_norm_backward(
    const Tensor& grad_in, const Tensor& feats_in, const Tensor& weight_in, const Tensor& mean_in,
    const Tensor& rstd_in, bool rms, bool want_weight, bool want_bias
) {
    const Matrix feats = matrix(feats_in, "feats");
    const Matrix grad = matching(grad_in, feats, "grad");
    const int dtype = dtype_code(feats.t);
    const int32_t channels = static_cast<int32_t>(feats.channels);
    const Tensor weight = vector_argument(weight_in, "weight", feats.channels, feats, feats.t.scalar_type());
    const Tensor mean = rms ? Tensor() : vector_argument(mean_in, "mean", feats.rows, feats, at::kFloat);
    const Tensor rstd = vector_argument(rstd_in, "rstd", feats.rows, feats, at::kFloat);
    const Tensor grad_feats = new_like(feats, {feats.rows, feats.channels});
    const Tensor grad_weight = want_weight ? new_like(feats, {feats.channels}) : Tensor();
    const Tensor grad_bias = want_bias ? new_like(feats, {feats.channels}) : Tensor();
    const size_t bytes = want_weight || want_bias ? lat_row_norm_backward_workspace_bytes(feats.rows, channels) : 0;
    const Tensor workspace = bytes > 0 ? new_workspace(feats, bytes) : Tensor();
    const c10::cuda::CUDAGuard guard(feats.t.device());
    check(lat_row_norm_backward(
        dtype, rms, data(grad.t), grad.stride, data(feats.t), feats.rows, channels, feats.stride, data(weight),
        floats(mean), floats(rstd), mutable_data(grad_feats), mutable_data(grad_weight), mutable_data(grad_bias),
        mutable_data(workspace), bytes, stream_of(feats)));
    return {grad_feats, grad_weight, grad_bias};
}

struct RowNorm : torch::autograd::Function<RowNorm> {
    static Tensor forward(
        AutogradContext* ctx, const Tensor& feats, const OptionalTensor& weight, const OptionalTensor& bias, double eps,
        bool rms
    ) {
        auto [out, mean, rstd] = row_norm_forward(feats, plain(weight), plain(bias), eps, rms);
        ctx->saved_data["rms"] = rms;
        ctx->saved_data["bias"] = bias.has_value();
        ctx->save_for_backward({feats, plain(weight), mean, rstd});
        return out;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        // inputs: the features, then the weight and the bias as far as there are any
        const size_t bias_place = saved[1].defined() ? 2 : 1;
        auto [feats, weight, bias] = row_norm_backward(
            grads[0], saved[0], saved[1], saved[2], saved[3], ctx->saved_data["rms"].toBool(),
            saved[1].defined() && ctx->needs_input_grad(1),
            ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(bias_place));
        return once({feats, weight, bias, Tensor(), Tensor()});
    }
};

// ---- dropout ----------------------------------------------------------------------------------

Tensor dropout_values(
    const Tensor& feats_in, const Tensor& residual_in, double p, int64_t seed, const Tensor& seed_word, int64_t offset
) {
    require_cuda(feats_in, "feats");
    REQUIRE(feats_in.dim() == 2, "feats must have shape (N, C).");
    const Tensor feats = feats_in.contiguous();
    const int dtype = dtype_code(feats);
    REQUIRE(p >= 0.0 && p < 1.0, "p must satisfy 0 <= p < 1.");
    Tensor residual;
    if (residual_in.defined()) {
        require_cuda(residual_in, "residual");
        REQUIRE(residual_in.sizes() == feats.sizes() && residual_in.scalar_type() == feats.scalar_type() &&
                              residual_in.device() == feats.device(),
                          "residual must match the features in shape, dtype and device.");
        residual = residual_in.contiguous();
    }
    if (seed_word.defined()) {
        REQUIRE(
            seed_word.is_cuda() && seed_word.device() == feats.device() && seed_word.scalar_type() == at::kLong &&
                seed_word.numel() == 1,
            "seed must be an int or an int64 CUDA tensor of one element on the feature device.");
    }
    const Tensor out = at::empty(feats.sizes(), feats.options());
    const c10::cuda::CUDAGuard guard(feats.device());
    check(lat_dropout(
        dtype, data(feats), data(residual), feats.numel(), p, static_cast<uint64_t>(seed),
        static_cast<const uint64_t*>(data(seed_word)), static_cast<uint64_t>(offset), mutable_data(out),
        at::cuda::getCurrentCUDAStream(feats.device().index()).stream()));
    return out;
}

struct Dropout : torch::autograd::Function<Dropout> {
    static Tensor forward(
        AutogradContext* ctx, const Tensor& feats, const OptionalTensor& residual, double p, int64_t seed,
        const OptionalTensor& seed_word, int64_t offset
    ) {
        ctx->saved_data["p"] = p;
        ctx->saved_data["seed"] = seed;
        ctx->saved_data["offset"] = offset;
        // saved as a variable, so that changing it before the backward pass, which draws the mask
        // again, is noticed
        ctx->saved_data["residual"] = residual.has_value();
        ctx->save_for_backward({plain(seed_word)});
        return dropout_values(feats, plain(residual), p, seed, plain(seed_word), offset);
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        Tensor feats;
        if (ctx->needs_input_grad(0)) {
            feats = dropout_values(grads[0], Tensor(), ctx->saved_data["p"].toDouble(), ctx->saved_data["seed"].toInt(),
                                   saved[0], ctx->saved_data["offset"].toInt());
        }
        const bool to_residual = ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(1);
        return once({feats, to_residual ? grads[0] : Tensor(), Tensor(), Tensor(), Tensor(), Tensor()});
    }
};

// an int of any size counts modulo 2^64
int64_t word_of(const py::handle& value) {
    const auto number = py::reinterpret_steal<py::object>(PyNumber_Index(value.ptr()));
    if (!number) {
        throw py::error_already_set();
    }
    return static_cast<int64_t>(PyLong_AsUnsignedLongLongMask(number.ptr()));
}

Tensor dropout(
    const Tensor& feats, double p, const py::object& seed, const py::object& offset, const OptionalTensor& residual_in
) {
    const bool on_device = THPVariable_Check(seed.ptr());
    const Tensor word = on_device ? THPVariable_Unpack(seed.ptr()) : Tensor();
    const int64_t number = on_device ? 0 : word_of(seed), place = word_of(offset);
    const Tensor residual = residual_in.value_or(Tensor());
    if (wants_gradient({feats, residual})) {
        return Dropout::apply(feats, none_if_undefined(residual), p, number, none_if_undefined(word), place);
    }
    return dropout_values(feats, residual, p, number, word, place);
}

// ---- gated recurrence -------------------------------------------------------------------------

Tensor state_argument(const Tensor& t, const char* name, int64_t rows, const Matrix& like) {
    if (!t.defined()) {
        return t;
    }
    require_cuda(t, name);
    REQUIRE(t.dim() == 2 && t.size(0) == rows && t.size(1) == like.channels &&
                          t.scalar_type() == at::kFloat && t.device() == like.t.device(),
                      name, " must have shape (", rows, ", ", like.channels,
                      ") and float32 dtype on the feature device.");
    return t.contiguous();
}

Tensor offsets_argument(const Tensor& t, const Matrix& like) {
    require_cuda(t, "offsets");
    REQUIRE(t.scalar_type() == at::kInt, "offsets must be int32.");
    REQUIRE(t.dim() == 1 && t.numel() >= 1 && t.device() == like.t.device(),
                      "offsets must hold one int32 entry per sequence and one more, on the feature device.");
    REQUIRE(t.numel() <= 0x7fffffff, "offsets has too many entries.");
    return t.contiguous();
}

void check_rows(const Matrix& feats) {
    REQUIRE(feats.rows <= 0x7fffffff, "feats has too many rows.");
}

std::tuple<Tensor, Tensor, Tensor> recurrence_forward(
    const Tensor& feats_in, const Tensor& gate_in, const Tensor& offsets_in, const Tensor& initial_in, bool reverse,
    bool want_state, bool want_carries, const Tensor& status
) {
    const Matrix feats = matrix(feats_in, "feats");
    const int dtype = dtype_code(feats.t);
    const Matrix gate = matching(gate_in, feats, "gate");
    check_rows(feats);
    const Tensor offsets = offsets_argument(offsets_in, feats);
    const int64_t sequences = offsets.numel() - 1;
    const Tensor initial = state_argument(initial_in, "initial_state", sequences, feats);
    const int32_t rows = static_cast<int32_t>(feats.rows), channels = static_cast<int32_t>(feats.channels);
    const Tensor out = new_like(feats, {feats.rows, feats.channels});
    const Tensor final = want_state ? new_floats(feats, {sequences, feats.channels}) : Tensor();
    const Tensor carries = want_carries ? new_floats(feats, {lat_recurrence_carry_rows(rows), feats.channels}) : Tensor();
    const size_t bytes = lat_recurrence_workspace_bytes(dtype, rows, channels);
    const Tensor workspace = new_workspace(feats, bytes);
    const c10::cuda::CUDAGuard guard(feats.t.device());
    check(lat_recurrence_forward(
        dtype, data(feats.t), feats.stride, data(gate.t), gate.stride, rows, channels,
        static_cast<const int32_t*>(data(offsets)), static_cast<int32_t>(sequences), floats(initial), reverse,
        mutable_data(out), mutable_floats(final), mutable_floats(carries), mutable_data(workspace), bytes,
        static_cast<int32_t*>(mutable_data(status)), stream_of(feats)));
    return {out, final, carries};
}

std::tuple<Tensor, Tensor, Tensor> recurrence_backward(
    const Tensor& grad_in, const Tensor& grad_final_in, const Tensor& feats_in, const Tensor& gate_in,
    const Tensor& offsets_in, const Tensor& initial_in, bool reverse, const Tensor& carries_in, bool want_initial,
    const Tensor& status
) {
    const Matrix feats = matrix(feats_in, "feats");
    const int dtype = dtype_code(feats.t);
    const Matrix gate = matching(gate_in, feats, "gate"), grad = matching(grad_in, feats, "grad");
    check_rows(feats);
    const Tensor offsets = offsets_argument(offsets_in, feats);
    const int64_t sequences = offsets.numel() - 1;
    const Tensor initial = state_argument(initial_in, "initial_state", sequences, feats);
    const Tensor grad_final = state_argument(grad_final_in, "grad_final", sequences, feats);
    const int32_t rows = static_cast<int32_t>(feats.rows), channels = static_cast<int32_t>(feats.channels);
    const Tensor carries = state_argument(carries_in, "carries", lat_recurrence_carry_rows(rows), feats);
    const Tensor grad_feats = new_like(feats, {feats.rows, feats.channels});
    const Tensor grad_gate = new_like(feats, {feats.rows, feats.channels});
    const Tensor grad_initial = want_initial ? new_floats(feats, {sequences, feats.channels}) : Tensor();
    const size_t bytes = lat_recurrence_workspace_bytes(dtype, rows, channels);
    const Tensor workspace = new_workspace(feats, bytes);
    const c10::cuda::CUDAGuard guard(feats.t.device());
    check(lat_recurrence_backward(
        dtype, data(grad.t), grad.stride, floats(grad_final), data(feats.t), feats.stride, data(gate.t), gate.stride,
        rows, channels, static_cast<const int32_t*>(data(offsets)), static_cast<int32_t>(sequences), floats(initial),
        reverse, floats(carries), mutable_data(grad_feats), mutable_data(grad_gate), mutable_floats(grad_initial),
        mutable_data(workspace), bytes, static_cast<int32_t*>(mutable_data(status)), stream_of(feats)));
    return {grad_feats, grad_gate, grad_initial};
}

struct Recurrence : torch::autograd::Function<Recurrence> {
    static variable_list forward(
        AutogradContext* ctx, const Tensor& feats, const Tensor& gate, const OptionalTensor& initial,
        const Tensor& offsets, bool reverse, bool want_state, const Tensor& status
    ) {
        auto [out, final, carries] =
            recurrence_forward(feats, gate, offsets, plain(initial), reverse, want_state, true, status);
        ctx->set_materialize_grads(false);
        ctx->saved_data["reverse"] = reverse;
        ctx->saved_data["status"] = status;   // written by kernels meanwhile: not a saved variable
        ctx->save_for_backward({feats, gate, plain(initial), offsets, carries});
        return want_state ? variable_list{out, final} : variable_list{out};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor grad = grads[0].defined() ? grads[0] : at::zeros(saved[0].sizes(), saved[0].options());
        auto [feats, gate, initial] = recurrence_backward(
            grad, grads.size() > 1 ? grads[1] : Tensor(), saved[0], saved[1], saved[3], saved[2],
            ctx->saved_data["reverse"].toBool(), saved[4],
            saved[2].defined() && ctx->needs_input_grad(2), ctx->saved_data["status"].toTensor());
        return once({feats, gate, initial, Tensor(), Tensor(), Tensor(), Tensor()});
    }
};

// Whether the ranges of memory that two tensors span have a byte in common.
bool overlap(const Tensor& a, const Tensor& b) {
    if (a.numel() == 0 || b.numel() == 0) {
        return false;
    }
    const auto begin = [](const Tensor& t) { return reinterpret_cast<uintptr_t>(t.const_data_ptr()); };
    const auto end = [&](const Tensor& t) {
        int64_t last = 0;
        for (int64_t d = 0; d < t.dim(); ++d) {
            last += (t.size(d) - 1) * t.stride(d);
        }
        return begin(t) + (last + 1) * t.element_size();
    };
    return begin(a) < end(b) && begin(b) < end(a);
}

std::tuple<Tensor, Tensor> recurrence_step(
    const Tensor& feats_in, const Tensor& gate_in, const OptionalTensor& state_in, const OptionalTensor& out_state_in
) {
    const Matrix feats = matrix(feats_in, "feats");
    const int dtype = dtype_code(feats.t);
    const Matrix gate = matching(gate_in, feats, "gate");
    REQUIRE(state_in.has_value(), "state must have shape (N, C) and float32 dtype on the feature device.");
    const Tensor state = state_argument(*state_in, "state", feats.rows, feats);
    Tensor next = out_state_in.value_or(Tensor());
    if (next.defined()) {
        // a state that this function returned may go on; another one would keep a graph that its new
        // values do not come from
        REQUIRE(!wants_gradient({next}) || dynamic_cast<torch::autograd::Error*>(next.grad_fn().get()) != nullptr,
                "out_state must not require a gradient.");
        REQUIRE(state_argument(next, "out_state", feats.rows, feats).is_same(next), "out_state must be contiguous.");
        // a thread reads and writes one place of the state; every other overlap is a race
        REQUIRE(next.const_data_ptr() == state.const_data_ptr() || !overlap(next, state),
                "out_state must be state or lie apart from it.");
        REQUIRE(!overlap(next, feats.t) && !overlap(next, gate.t), "out_state must lie apart from the features and the gate.");
        next.unsafeGetTensorImpl()->bump_version();   // written in place
    } else {
        next = new_floats(feats, {feats.rows, feats.channels});
    }
    const Tensor out = new_like(feats, {feats.rows, feats.channels});
    const c10::cuda::CUDAGuard guard(feats.t.device());
    check(lat_recurrence_step(
        dtype, data(feats.t), feats.stride, data(gate.t), gate.stride, floats(state), feats.rows,
        static_cast<int32_t>(feats.channels), mutable_data(out), mutable_floats(next), stream_of(feats)));
    if (wants_gradient({feats_in, gate_in, *state_in})) {
        const variable_list results =
            raising({out, next}, "gated_recurrence_step has no gradient: use gated_recurrence, or torch.no_grad()");
        return {results[0], results[1]};
    }
    return {out, next};
}

using Three = std::tuple<OptionalTensor, OptionalTensor, OptionalTensor>;
Three optional(const std::tuple<Tensor, Tensor, Tensor>& t) {
    return {none_if_undefined(std::get<0>(t)), none_if_undefined(std::get<1>(t)), none_if_undefined(std::get<2>(t))};
}

} // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("row_norm_forward", [](const Tensor& feats, const OptionalTensor& weight, const OptionalTensor& bias, double eps,
                                 bool rms) { return optional(row_norm_forward(feats, plain(weight), plain(bias), eps, rms)); });
    m.def("row_norm_backward",
          [](const Tensor& grad, const Tensor& feats, const OptionalTensor& weight, const OptionalTensor& mean,
             const Tensor& rstd, bool rms, bool want_weight, bool want_bias) {
              return optional(row_norm_backward(grad, feats, plain(weight), plain(mean), rstd, rms, want_weight, want_bias));
          });
    // None where no gradient is asked for
    m.def("row_norm_recorded", [](const Tensor& feats, const OptionalTensor& weight_in, const OptionalTensor& bias_in,
                                  double eps, bool rms) -> OptionalTensor {
        if (!wants_gradient({feats, plain(weight_in), plain(bias_in)})) {
            return std::nullopt;
        }
        return RowNorm::apply(feats, weight_in, bias_in, eps, rms);
    });
    m.def("dropout", &dropout);
    m.def("recurrence_forward",
          [](const Tensor& feats, const Tensor& gate, const Tensor& offsets, const OptionalTensor& initial, bool reverse,
             bool want_state, bool want_carries, const Tensor& status) {
              return optional(recurrence_forward(feats, gate, offsets, plain(initial), reverse, want_state, want_carries, status));
          });
    m.def("recurrence_backward",
          [](const Tensor& grad, const OptionalTensor& grad_final, const Tensor& feats, const Tensor& gate,
             const Tensor& offsets, const OptionalTensor& initial, bool reverse, const Tensor& carries, bool want_initial,
             const Tensor& status) {
              return optional(recurrence_backward(grad, plain(grad_final), feats, gate, offsets, plain(initial), reverse,
                                                  carries, want_initial, status));
          });
    // the values and, if wanted, the final state; recorded where a gradient is asked for
    m.def("recurrence", [](const Tensor& feats, const Tensor& gate, const Tensor& offsets, const OptionalTensor& initial_in,
                           bool reverse, bool want_state, const Tensor& status) -> std::tuple<Tensor, OptionalTensor> {
        const Tensor initial = plain(initial_in);
        if (wants_gradient({feats, gate, initial})) {
            const auto out = Recurrence::apply(feats, gate, initial_in, offsets, reverse, want_state, status);
            return {out[0], want_state ? OptionalTensor(out[1]) : std::nullopt};
        }
        auto [out, final, carries] = recurrence_forward(feats, gate, offsets, initial, reverse, want_state, false, status);
        return {out, none_if_undefined(final)};
    });
    m.def("recurrence_step", &recurrence_step);
}
