// torch.ops.mops.* in C++: the five operations as PyTorch operators with
// autograd, for callers that cannot afford (or do not have) an interpreter
// around every call: eager-mode training loops, scripted modules loaded from
// C++.
//
// Operator names and schemas are those of the reference's TorchScript
// extension (mops-torch/src/register.cpp:5-38 of lab-cosmo/mops). What is
// behind them is this library only: every operator checks its tensors, makes
// them contiguous, points the library at PyTorch's current stream and calls
// the `mops::cuda::` templates of <mops.hpp>; ROCm tensors are the only ones
// accepted (host tensors: "device path only", as everywhere in this library).
//
// Autograd: one torch::autograd::Function per operation whose backward is the
// library's vjp, computing only the gradients that are asked for. For the
// three operations that have a second derivative (HPE, SAP, OPSA, as in the
// reference) the vjp is itself a Function whose backward is the library's
// vjp_vjp. There is no gradient with respect to C or to index tensors.
//
// The operators of the layers (mops/layers.h) follow the same pattern, for 16-bit
// types as well. The embedding and the products by group are linear in each
// argument, so derivatives of their gradients, of any order, are calls of the same
// operators; of the residual update's gradients there is none, and asking for one
// is an error.
//
// mops_amd/torch.py loads this library when it has been built and registers
// the same operators from Python otherwise.
#include <algorithm>
#include <array>
#include <limits>
#include <stdexcept>
#include <string>
#include <vector>

#include <torch/script.h>

#include "mops.hpp"

#include "torch_tensors.hpp"

namespace {

using namespace mops::amd::torch_tensors;

using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

// ------------------------------------------------------------ arguments --
void require_device(const at::Tensor& tensor, const char* name, const char* operation) {
    if (!tensor.is_cuda()) { // ROCm tensors carry the CUDA device type
        throw std::runtime_error(
            std::string("mops::") + operation + ": " + name +
            " must be on a ROCm device; this library implements the device path only"
        );
    }
}

at::Tensor values(const at::Tensor& tensor, const at::Tensor& like, const char* name, const char* operation) {
    require_device(tensor, name, operation);
    if (tensor.scalar_type() != at::kFloat && tensor.scalar_type() != at::kDouble) {
        throw std::runtime_error(std::string("mops::") + operation + ": " + name + " must be float32 or float64");
    }
    if (tensor.scalar_type() != like.scalar_type() || tensor.device() != like.device()) {
        throw std::runtime_error(
            std::string("mops::") + operation + ": " + name + " must have the dtype and the device of A"
        );
    }
    return tensor.contiguous();
}

at::Tensor indices(const at::Tensor& tensor, const at::Tensor& like, const char* name, const char* operation) {
    require_device(tensor, name, operation);
    if (tensor.device() != like.device()) {
        throw std::runtime_error(std::string("mops::") + operation + ": " + name + " must be on the device of A");
    }
    if (!at::isIntegralType(tensor.scalar_type(), /*includeBool=*/false)) {
        throw std::runtime_error(std::string("mops::") + operation + ": " + name + " must hold integers");
    }
    return tensor.to(at::kInt).contiguous();
}

/// Whether a call on these tensors has to leave something for autograd. Without it (inference, and
/// a backward pass that is not itself differentiated) an operator calls the library directly: a
/// Function and its context cost 1 us, of a call of 6.
bool recorded(std::initializer_list<const at::Tensor*> tensors) {
    for (const at::Tensor* tensor : tensors) {
        if (!tensor->defined() || tensor->unsafeGetTensorImpl()->autograd_meta() == nullptr) {
            continue;
        }
        if ((at::GradMode::is_enabled() && tensor->requires_grad()) || tensor->_fw_grad(0).defined()) {
            return true; // (forward-mode gradients: Function says that there are none)
        }
    }
    return false;
}

at::Tensor nothing(const at::Tensor& like) { return at::empty({0}, like.options()); }
at::Tensor or_undefined(const at::Tensor& tensor, bool wanted) { return wanted ? tensor : at::Tensor(); }

// ------------------------------------------------------------------ HPE --
at::Tensor hpe_forward(const at::Tensor& A_, const at::Tensor& C_, const at::Tensor& P_) {
    const char* op = "homogeneous_polynomial_evaluation";
    const at::Tensor A = values(A_, A_, "A", op), C = values(C_, A_, "C", op), P = indices(P_, A_, "indices_A", op);
    OnTorchStream stream(A);
    at::Tensor output = new_tensor({A.dim() == 2 ? A.size(0) : 0}, A);
    by_dtype(A, [&](auto zero) {
        using T = decltype(zero);
        mops::cuda::homogeneous_polynomial_evaluation<T>(
            view<T, 1>(output, "output"), view<T, 2>(A, "A"), view<T, 1>(C, "C"), view<int32_t, 2>(P, "indices_A")
        );
    });
    return output;
}

at::Tensor hpe_vjp(const at::Tensor& gO_, const at::Tensor& A_, const at::Tensor& C_, const at::Tensor& P_) {
    const char* op = "homogeneous_polynomial_evaluation_vjp";
    const at::Tensor A = values(A_, A_, "A", op), C = values(C_, A_, "C", op), P = indices(P_, A_, "indices_A", op);
    const at::Tensor gO = values(gO_, A_, "grad_output", op);
    OnTorchStream stream(A);
    at::Tensor grad_A = new_like(A);
    by_dtype(A, [&](auto zero) {
        using T = decltype(zero);
        mops::cuda::homogeneous_polynomial_evaluation_vjp<T>(
            view<T, 2>(grad_A, "grad_A"), view<T, 1>(gO, "grad_output"), view<T, 2>(A, "A"), view<T, 1>(C, "C"),
            view<int32_t, 2>(P, "indices_A")
        );
    });
    return grad_A;
}

std::array<at::Tensor, 2> hpe_vjp_vjp(
    const at::Tensor& ggA_, const at::Tensor& gO_, const at::Tensor& A_, const at::Tensor& C_, const at::Tensor& P_,
    bool want_ggO, bool want_A2
) {
    const char* op = "homogeneous_polynomial_evaluation_vjp_vjp";
    const at::Tensor A = values(A_, A_, "A", op), C = values(C_, A_, "C", op), P = indices(P_, A_, "indices_A", op);
    const at::Tensor gO = values(gO_, A_, "grad_output", op);
    const at::Tensor ggA = ggA_.defined() ? values(ggA_, A_, "grad_grad_A", op) : at::Tensor();
    OnTorchStream stream(A);
    at::Tensor ggO = want_ggO ? new_like(gO) : at::Tensor();
    at::Tensor A2 = want_A2 ? new_like(A) : at::Tensor();
    by_dtype(A, [&](auto zero) {
        using T = decltype(zero);
        mops::cuda::homogeneous_polynomial_evaluation_vjp_vjp<T>(
            view<T, 1>(ggO, "grad_grad_output"), view<T, 2>(A2, "grad_A_2"), view<T, 2>(ggA, "grad_grad_A"),
            view<T, 1>(gO, "grad_output"), view<T, 2>(A, "A"), view<T, 1>(C, "C"), view<int32_t, 2>(P, "indices_A")
        );
    });
    return {ggO, A2};
}

struct HpeVjp : public Function<HpeVjp> {
    static at::Tensor forward(AutogradContext* ctx, at::Tensor gO, at::Tensor A, at::Tensor C, at::Tensor P) {
        ctx->save_for_backward({gO, A, C, P});
        return hpe_vjp(gO, A, C, P);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        if (ctx->needs_input_grad(2)) {
            throw std::runtime_error("gradients with respect to C are not supported");
        }
        const bool want_ggO = ctx->needs_input_grad(0), want_A2 = ctx->needs_input_grad(1);
        const auto second = hpe_vjp_vjp(grads[0], saved[0], saved[1], saved[2], saved[3], want_ggO, want_A2);
        return {second[0], second[1], at::Tensor(), at::Tensor()};
    }
};

struct Hpe : public Function<Hpe> {
    static at::Tensor forward(AutogradContext* ctx, at::Tensor A, at::Tensor C, at::Tensor P) {
        ctx->save_for_backward({A, C, P});
        return hpe_forward(A, C, P);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        if (ctx->needs_input_grad(1)) {
            throw std::runtime_error("gradients with respect to C are not supported");
        }
        at::Tensor grad_A;
        if (ctx->needs_input_grad(0)) {
            grad_A = recorded({&grads[0], &saved[0], &saved[1]}) ? HpeVjp::apply(grads[0], saved[0], saved[1], saved[2])
                                                                 : hpe_vjp(grads[0], saved[0], saved[1], saved[2]);
        }
        return {grad_A, at::Tensor(), at::Tensor()};
    }
};

// ------------------------------------------------------------ OPSA, SAP --
// Both have two differentiable inputs (A, B) and a second derivative; they differ in
// their other arguments, which `Extra` carries: OPSA {indices_output}, SAP {C, indices_A,
// indices_B, indices_output}.
struct Opsa {
    static constexpr const char* name = "outer_product_scatter_add";
    static constexpr size_t n_extra = 1;
    static std::vector<at::Tensor> prepare(const std::vector<at::Tensor>& extra, const at::Tensor& A, const char* op) {
        return {indices(extra[0], A, "indices_output", op)};
    }
    static at::Tensor output_like(const at::Tensor& A, const at::Tensor& B, int64_t output_size) {
        return new_tensor({output_size, A.dim() == 2 ? A.size(1) : 0, B.dim() == 2 ? B.size(1) : 0}, A);
    }
    template <typename T>
    static void forward(at::Tensor& O, const at::Tensor& A, const at::Tensor& B, const std::vector<at::Tensor>& e) {
        mops::cuda::outer_product_scatter_add<T>(
            view<T, 3>(O, "output"), view<T, 2>(A, "A"), view<T, 2>(B, "B"), view<int32_t, 1>(e[0], "indices_output")
        );
    }
    template <typename T>
    static void vjp(
        at::Tensor& gA, at::Tensor& gB, const at::Tensor& gO, const at::Tensor& A, const at::Tensor& B,
        const std::vector<at::Tensor>& e
    ) {
        mops::cuda::outer_product_scatter_add_vjp<T>(
            view<T, 2>(gA, "grad_A"), view<T, 2>(gB, "grad_B"), view<T, 3>(gO, "grad_output"), view<T, 2>(A, "A"),
            view<T, 2>(B, "B"), view<int32_t, 1>(e[0], "indices_output")
        );
    }
    template <typename T>
    static void vjp_vjp(
        at::Tensor& ggO, at::Tensor& A2, at::Tensor& B2, const at::Tensor& ggA, const at::Tensor& ggB,
        const at::Tensor& gO, const at::Tensor& A, const at::Tensor& B, const std::vector<at::Tensor>& e
    ) {
        mops::cuda::outer_product_scatter_add_vjp_vjp<T>(
            view<T, 3>(ggO, "grad_grad_output"), view<T, 2>(A2, "grad_A_2"), view<T, 2>(B2, "grad_B_2"),
            view<T, 2>(ggA, "grad_grad_A"), view<T, 2>(ggB, "grad_grad_B"), view<T, 3>(gO, "grad_output"),
            view<T, 2>(A, "A"), view<T, 2>(B, "B"), view<int32_t, 1>(e[0], "indices_output")
        );
    }
    template <typename T> static mops::Tensor<T, 3> grad_output_view(const at::Tensor& gO) {
        return view<T, 3>(gO, "grad_output");
    }
};

struct Sap {
    static constexpr const char* name = "sparse_accumulation_of_products";
    static constexpr size_t n_extra = 4;
    static std::vector<at::Tensor> prepare(const std::vector<at::Tensor>& extra, const at::Tensor& A, const char* op) {
        return {
            values(extra[0], A, "C", op), indices(extra[1], A, "indices_A", op), indices(extra[2], A, "indices_B", op),
            indices(extra[3], A, "indices_output", op)};
    }
    static at::Tensor output_like(const at::Tensor& A, const at::Tensor&, int64_t output_size) {
        return new_tensor({A.dim() == 2 ? A.size(0) : 0, output_size}, A);
    }
    template <typename T>
    static void forward(at::Tensor& O, const at::Tensor& A, const at::Tensor& B, const std::vector<at::Tensor>& e) {
        mops::cuda::sparse_accumulation_of_products<T>(
            view<T, 2>(O, "output"), view<T, 2>(A, "A"), view<T, 2>(B, "B"), view<T, 1>(e[0], "C"),
            view<int32_t, 1>(e[1], "indices_A"), view<int32_t, 1>(e[2], "indices_B"),
            view<int32_t, 1>(e[3], "indices_output")
        );
    }
    template <typename T>
    static void vjp(
        at::Tensor& gA, at::Tensor& gB, const at::Tensor& gO, const at::Tensor& A, const at::Tensor& B,
        const std::vector<at::Tensor>& e
    ) {
        mops::cuda::sparse_accumulation_of_products_vjp<T>(
            view<T, 2>(gA, "grad_A"), view<T, 2>(gB, "grad_B"), view<T, 2>(gO, "grad_output"), view<T, 2>(A, "A"),
            view<T, 2>(B, "B"), view<T, 1>(e[0], "C"), view<int32_t, 1>(e[1], "indices_A"),
            view<int32_t, 1>(e[2], "indices_B"), view<int32_t, 1>(e[3], "indices_output")
        );
    }
    template <typename T>
    static void vjp_vjp(
        at::Tensor& ggO, at::Tensor& A2, at::Tensor& B2, const at::Tensor& ggA, const at::Tensor& ggB,
        const at::Tensor& gO, const at::Tensor& A, const at::Tensor& B, const std::vector<at::Tensor>& e
    ) {
        mops::cuda::sparse_accumulation_of_products_vjp_vjp<T>(
            view<T, 2>(ggO, "grad_grad_output"), view<T, 2>(A2, "grad_A_2"), view<T, 2>(B2, "grad_B_2"),
            view<T, 2>(ggA, "grad_grad_A"), view<T, 2>(ggB, "grad_grad_B"), view<T, 2>(gO, "grad_output"),
            view<T, 2>(A, "A"), view<T, 2>(B, "B"), view<T, 1>(e[0], "C"), view<int32_t, 1>(e[1], "indices_A"),
            view<int32_t, 1>(e[2], "indices_B"), view<int32_t, 1>(e[3], "indices_output")
        );
    }
};

/// grad_A, grad_B of a bilinear operation; a gradient that is not wanted comes back undefined.
template <typename Op>
std::array<at::Tensor, 2> bilinear_vjp(
    const at::Tensor& gO_, const at::Tensor& A_, const at::Tensor& B_, const std::vector<at::Tensor>& extra_,
    bool want_A, bool want_B
) {
    const std::string op = std::string(Op::name) + "_vjp";
    const at::Tensor A = values(A_, A_, "A", op.c_str()), B = values(B_, A_, "B", op.c_str());
    const at::Tensor gO = values(gO_, A_, "grad_output", op.c_str());
    const std::vector<at::Tensor> extra = Op::prepare(extra_, A, op.c_str());
    OnTorchStream stream(A);
    at::Tensor gA = want_A ? new_like(A) : at::Tensor();
    at::Tensor gB = want_B ? new_like(B) : at::Tensor();
    by_dtype(A, [&](auto zero) { Op::template vjp<decltype(zero)>(gA, gB, gO, A, B, extra); });
    return {gA, gB};
}

template <typename Op> struct BilinearVjp : public Function<BilinearVjp<Op>> {
    // inputs: grad_output, A, B, extra tensors..., then which gradients are wanted
    static variable_list forward(
        AutogradContext* ctx, at::Tensor gO, at::Tensor A, at::Tensor B, at::TensorList extra_list, bool want_A,
        bool want_B
    ) {
        // (a TensorList, not a vector: only that makes the tensors in it inputs of the Function)
        const variable_list extra = extra_list.vec();
        variable_list saved = {gO, A, B};
        saved.insert(saved.end(), extra.begin(), extra.end());
        ctx->save_for_backward(saved);
        ctx->saved_data["want_A"] = want_A;
        ctx->saved_data["want_B"] = want_B;
        const auto gradients = bilinear_vjp<Op>(gO, A, B, extra, want_A, want_B);
        // a Function's outputs must be defined: an empty tensor stands for "not computed"
        return {want_A ? gradients[0] : nothing(A), want_B ? gradients[1] : nothing(B)};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const at::Tensor &gO_ = saved[0], &A_ = saved[1], &B_ = saved[2];
        const std::vector<at::Tensor> extra_(saved.begin() + 3, saved.end());
        const std::string op = std::string(Op::name) + "_vjp_vjp";
        // the inputs of forward(): grad_output 0, A 1, B 2, the list of extra tensors from 3 on
        for (size_t at = 0; at < Op::n_extra; at++) {
            if (at::isFloatingType(extra_[at].scalar_type()) && ctx->needs_input_grad(3 + at)) {
                throw std::runtime_error("gradients with respect to C are not supported");
            }
        }
        const bool have_A = ctx->saved_data["want_A"].toBool() && grads[0].defined();
        const bool have_B = ctx->saved_data["want_B"].toBool() && grads[1].defined();
        const bool want_ggO = ctx->needs_input_grad(0), want_A2 = ctx->needs_input_grad(1),
                   want_B2 = ctx->needs_input_grad(2);
        const at::Tensor A = values(A_, A_, "A", op.c_str()), B = values(B_, A_, "B", op.c_str());
        const at::Tensor gO = values(gO_, A_, "grad_output", op.c_str());
        const at::Tensor ggA = have_A ? values(grads[0], A_, "grad_grad_A", op.c_str()) : at::Tensor();
        const at::Tensor ggB = have_B ? values(grads[1], A_, "grad_grad_B", op.c_str()) : at::Tensor();
        const std::vector<at::Tensor> extra = Op::prepare(extra_, A, op.c_str());
        OnTorchStream stream(A);
        at::Tensor ggO = want_ggO ? new_like(gO) : at::Tensor();
        at::Tensor A2 = want_A2 ? new_like(A) : at::Tensor();
        at::Tensor B2 = want_B2 ? new_like(B) : at::Tensor();
        by_dtype(A, [&](auto zero) {
            Op::template vjp_vjp<decltype(zero)>(ggO, A2, B2, ggA, ggB, gO, A, B, extra);
        });
        variable_list result = {ggO, A2, B2};
        result.resize(3 + Op::n_extra + 2); // nothing for the extra tensors and the two flags
        return result;
    }
};

template <typename Op>
at::Tensor bilinear_forward(
    const at::Tensor& A_, const at::Tensor& B_, const std::vector<at::Tensor>& extra_, int64_t output_size
) {
    const at::Tensor A = values(A_, A_, "A", Op::name), B = values(B_, A_, "B", Op::name);
    const std::vector<at::Tensor> extra = Op::prepare(extra_, A, Op::name);
    OnTorchStream stream(A);
    at::Tensor output = Op::output_like(A, B, output_size);
    by_dtype(A, [&](auto zero) { Op::template forward<decltype(zero)>(output, A, B, extra); });
    return output;
}

template <typename Op> struct Bilinear : public Function<Bilinear<Op>> {
    static at::Tensor forward(
        AutogradContext* ctx, at::Tensor A_, at::Tensor B_, at::TensorList extra_list, int64_t output_size
    ) {
        const variable_list extra_ = extra_list.vec();
        variable_list saved = {A_, B_};
        saved.insert(saved.end(), extra_.begin(), extra_.end());
        ctx->save_for_backward(saved);
        return bilinear_forward<Op>(A_, B_, extra_, output_size);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const std::vector<at::Tensor> extra(saved.begin() + 2, saved.end());
        for (size_t at = 0; at < Op::n_extra; at++) {
            if (at::isFloatingType(extra[at].scalar_type()) && ctx->needs_input_grad(2 + at)) {
                throw std::runtime_error("gradients with respect to C are not supported");
            }
        }
        const bool want_A = ctx->needs_input_grad(0), want_B = ctx->needs_input_grad(1);
        variable_list result(2 + Op::n_extra + 1);
        if (want_A || want_B) {
            if (recorded({&grads[0], &saved[0], &saved[1]})) {
                const auto gradients =
                    BilinearVjp<Op>::apply(grads[0], saved[0], saved[1], at::TensorList(extra), want_A, want_B);
                result[0] = or_undefined(gradients[0], want_A);
                result[1] = or_undefined(gradients[1], want_B);
            } else {
                const auto gradients = bilinear_vjp<Op>(grads[0], saved[0], saved[1], extra, want_A, want_B);
                result[0] = gradients[0];
                result[1] = gradients[1];
            }
        }
        return result;
    }
};

// ------------------------------------------------------- OPSAW, SASAW --
// Three differentiable inputs (A, B, W), no second derivative (the reference has none:
// mops/src/opsaw/cpu.tpp:133-150, mops/src/sasaw/cpu.tpp:173-194).
at::Tensor opsaw_forward(
    const at::Tensor& A_, const at::Tensor& B_, const at::Tensor& W_, const at::Tensor& PW_, const at::Tensor& PO_
) {
    const char* op = "outer_product_scatter_add_with_weights";
    const at::Tensor A = values(A_, A_, "A", op), B = values(B_, A_, "B", op), W = values(W_, A_, "W", op);
    const at::Tensor PW = indices(PW_, A_, "indices_W", op), PO = indices(PO_, A_, "indices_output", op);
    OnTorchStream stream(A);
    at::Tensor output =
        new_tensor({W.dim() == 2 ? W.size(0) : 0, A.dim() == 2 ? A.size(1) : 0, B.dim() == 2 ? B.size(1) : 0}, A);
    by_dtype(A, [&](auto zero) {
        using T = decltype(zero);
        mops::cuda::outer_product_scatter_add_with_weights<T>(
            view<T, 3>(output, "output"), view<T, 2>(A, "A"), view<T, 2>(B, "B"), view<T, 2>(W, "W"),
            view<int32_t, 1>(PW, "indices_W"), view<int32_t, 1>(PO, "indices_output")
        );
    });
    return output;
}

struct OpsawFunction : public Function<OpsawFunction> {
    static at::Tensor forward(
        AutogradContext* ctx, at::Tensor A_, at::Tensor B_, at::Tensor W_, at::Tensor PW_, at::Tensor PO_
    ) {
        ctx->save_for_backward({A_, B_, W_, PW_, PO_});
        return opsaw_forward(A_, B_, W_, PW_, PO_);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const char* op = "outer_product_scatter_add_with_weights_vjp";
        const auto saved = ctx->get_saved_variables();
        const bool want_A = ctx->needs_input_grad(0), want_B = ctx->needs_input_grad(1),
                   want_W = ctx->needs_input_grad(2);
        const at::Tensor A = values(saved[0], saved[0], "A", op), B = values(saved[1], saved[0], "B", op),
                         W = values(saved[2], saved[0], "W", op);
        const at::Tensor PW = indices(saved[3], saved[0], "indices_W", op),
                         PO = indices(saved[4], saved[0], "indices_output", op);
        const at::Tensor gO = values(grads[0], saved[0], "grad_output", op);
        OnTorchStream stream(A);
        at::Tensor gA = want_A ? new_like(A) : at::Tensor();
        at::Tensor gB = want_B ? new_like(B) : at::Tensor();
        at::Tensor gW = want_W ? new_like(W) : at::Tensor();
        by_dtype(A, [&](auto zero) {
            using T = decltype(zero);
            mops::cuda::outer_product_scatter_add_with_weights_vjp<T>(
                view<T, 2>(gA, "grad_A"), view<T, 2>(gB, "grad_B"), view<T, 2>(gW, "grad_W"),
                view<T, 3>(gO, "grad_output"), view<T, 2>(A, "A"), view<T, 2>(B, "B"), view<T, 2>(W, "W"),
                view<int32_t, 1>(PW, "indices_W"), view<int32_t, 1>(PO, "indices_output")
            );
        });
        return {gA, gB, gW, at::Tensor(), at::Tensor()};
    }
};

at::Tensor sasaw_forward(
    const at::Tensor& A_, const at::Tensor& B_, const at::Tensor& C_, const at::Tensor& W_, const at::Tensor& PA_,
    const at::Tensor& PW1_, const at::Tensor& PW2_, const at::Tensor& PO1_, const at::Tensor& PO2_, int64_t output_size
) {
    const char* op = "sparse_accumulation_scatter_add_with_weights";
    const at::Tensor A = values(A_, A_, "A", op), B = values(B_, A_, "B", op), C = values(C_, A_, "C", op),
                     W = values(W_, A_, "W", op);
    const at::Tensor PA = indices(PA_, A_, "indices_A", op), PW1 = indices(PW1_, A_, "indices_W_1", op),
                     PW2 = indices(PW2_, A_, "indices_W_2", op), PO1 = indices(PO1_, A_, "indices_output_1", op),
                     PO2 = indices(PO2_, A_, "indices_output_2", op);
    OnTorchStream stream(A);
    at::Tensor output =
        new_tensor({W.dim() == 3 ? W.size(0) : 0, output_size, B.dim() == 2 ? B.size(1) : 0}, A);
    by_dtype(A, [&](auto zero) {
        using T = decltype(zero);
        mops::cuda::sparse_accumulation_scatter_add_with_weights<T>(
            view<T, 3>(output, "output"), view<T, 2>(A, "A"), view<T, 2>(B, "B"), view<T, 1>(C, "C"),
            view<T, 3>(W, "W"), view<int32_t, 1>(PA, "indices_A"), view<int32_t, 1>(PW1, "indices_W_1"),
            view<int32_t, 1>(PW2, "indices_W_2"), view<int32_t, 1>(PO1, "indices_output_1"),
            view<int32_t, 1>(PO2, "indices_output_2")
        );
    });
    return output;
}

struct SasawFunction : public Function<SasawFunction> {
    static at::Tensor forward(
        AutogradContext* ctx, at::Tensor A_, at::Tensor B_, at::Tensor C_, at::Tensor W_, at::Tensor PA_,
        at::Tensor PW1_, at::Tensor PW2_, at::Tensor PO1_, at::Tensor PO2_, int64_t output_size
    ) {
        ctx->save_for_backward({A_, B_, C_, W_, PA_, PW1_, PW2_, PO1_, PO2_});
        return sasaw_forward(A_, B_, C_, W_, PA_, PW1_, PW2_, PO1_, PO2_, output_size);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const char* op = "sparse_accumulation_scatter_add_with_weights_vjp";
        const auto saved = ctx->get_saved_variables();
        if (ctx->needs_input_grad(2)) {
            throw std::runtime_error("gradients with respect to C are not supported");
        }
        const bool want_A = ctx->needs_input_grad(0), want_B = ctx->needs_input_grad(1),
                   want_W = ctx->needs_input_grad(3);
        const at::Tensor& like = saved[0];
        const at::Tensor A = values(saved[0], like, "A", op), B = values(saved[1], like, "B", op),
                         C = values(saved[2], like, "C", op), W = values(saved[3], like, "W", op);
        const at::Tensor PA = indices(saved[4], like, "indices_A", op), PW1 = indices(saved[5], like, "indices_W_1", op),
                         PW2 = indices(saved[6], like, "indices_W_2", op),
                         PO1 = indices(saved[7], like, "indices_output_1", op),
                         PO2 = indices(saved[8], like, "indices_output_2", op);
        const at::Tensor gO = values(grads[0], like, "grad_output", op);
        OnTorchStream stream(A);
        at::Tensor gA = want_A ? new_like(A) : at::Tensor();
        at::Tensor gB = want_B ? new_like(B) : at::Tensor();
        at::Tensor gW = want_W ? new_like(W) : at::Tensor();
        by_dtype(A, [&](auto zero) {
            using T = decltype(zero);
            mops::cuda::sparse_accumulation_scatter_add_with_weights_vjp<T>(
                view<T, 2>(gA, "grad_A"), view<T, 2>(gB, "grad_B"), view<T, 3>(gW, "grad_W"),
                view<T, 3>(gO, "grad_output"), view<T, 2>(A, "A"), view<T, 2>(B, "B"), view<T, 1>(C, "C"),
                view<T, 3>(W, "W"), view<int32_t, 1>(PA, "indices_A"), view<int32_t, 1>(PW1, "indices_W_1"),
                view<int32_t, 1>(PW2, "indices_W_2"), view<int32_t, 1>(PO1, "indices_output_1"),
                view<int32_t, 1>(PO2, "indices_output_2")
            );
        });
        variable_list result(10);
        result[0] = gA;
        result[1] = gB;
        result[3] = gW;
        return result;
    }
};

// -------------------------------------------------- layers' operators --
/// `like`: the tensor whose type and device all others have, by its name.
at::Tensor layer_values(
    const at::Tensor& tensor, const at::Tensor& like, const char* name, const char* like_name, const char* operation
) {
    require_device(tensor, name, operation);
    if (!is_layer_dtype(tensor.scalar_type())) {
        throw std::runtime_error(
            std::string("mops::") + operation + ": " + name + " must be float32, float64, bfloat16 or float16"
        );
    }
    if (tensor.scalar_type() != like.scalar_type() || tensor.device() != like.device()) {
        throw std::runtime_error(
            std::string("mops::") + operation + ": " + name + " must have the dtype and the device of " + like_name
        );
    }
    return tensor.contiguous();
}
/// (undefined stays undefined: not given.) A number that does not fit 32 bits is outside of every range, and has to stay
/// outside: it becomes -1 or the largest one, not what its lower half happens to be.
at::Tensor layer_indices(const at::Tensor& tensor, const at::Tensor& like, const char* name, const char* operation) {
    if (!tensor.defined()) {
        return tensor;
    }
    require_device(tensor, name, operation);
    if (tensor.device() != like.device() || !at::isIntegralType(tensor.scalar_type(), /*includeBool=*/false)) {
        throw std::runtime_error(
            std::string("mops::") + operation + ": " + name + " must hold integers, on the device of the other tensors"
        );
    }
    if (tensor.element_size() > 4) {
        return tensor.to(at::kLong).clamp(-1, std::numeric_limits<int32_t>::max()).to(at::kInt).contiguous();
    }
    return tensor.to(at::kInt).contiguous();
}

std::tuple<at::Tensor, at::Tensor> order_by_group(const at::Tensor& indices_, int64_t n_groups) {
    const char* op = "order_by_group";
    require_device(indices_, "indices", op);
    const at::Tensor indices = layer_indices(indices_, indices_, "indices", op);
    if (n_groups < 0) {
        throw std::runtime_error("mops::order_by_group: n_groups must not be negative");
    }
    OnTorchStream stream(indices);
    at::Tensor order = new_like(indices), offsets = new_tensor({n_groups + 1}, indices);
    mops::cuda::order_by_group(
        view<int32_t, 1>(order, "order"), view<int32_t, 1>(offsets, "offsets"), view<int32_t, 1>(indices, "indices")
    );
    return {order, offsets};
}

at::Tensor embedding_forward(const at::Tensor& table_, const at::Tensor& indices_, double scale) {
    const char* op = "scaled_embedding";
    const at::Tensor table = layer_values(table_, table_, "table", "table", op);
    const at::Tensor indices = layer_indices(indices_, table_, "indices", op);
    OnTorchStream stream(table);
    at::Tensor output = new_tensor({indices.dim() == 1 ? indices.size(0) : 0, table.dim() == 2 ? table.size(1) : 0}, table);
    by_layer_dtype(table, [&](auto zero) {
        using T = decltype(zero);
        mops::cuda::scaled_embedding<T>(
            view<T, 2>(output, "output"), view<T, 2>(table, "table"), view<int32_t, 1>(indices, "indices"), scale
        );
    });
    return output;
}

at::Tensor embedding_vjp(const at::Tensor& grad_output_, const at::Tensor& indices_, int64_t table_rows, double scale) {
    const char* op = "scaled_embedding_vjp";
    const at::Tensor grad_output = layer_values(grad_output_, grad_output_, "grad_output", "grad_output", op);
    const at::Tensor indices = layer_indices(indices_, grad_output_, "indices", op);
    OnTorchStream stream(grad_output);
    at::Tensor grad_table = new_tensor({table_rows, grad_output.dim() == 2 ? grad_output.size(1) : 0}, grad_output);
    by_layer_dtype(grad_output, [&](auto zero) {
        using T = decltype(zero);
        mops::cuda::scaled_embedding_vjp<T>(
            view<T, 2>(grad_table, "grad_table"), view<T, 2>(grad_output, "grad_output"),
            view<int32_t, 1>(indices, "indices"), mops::Tensor<int32_t, 1>{nullptr, {0}},
            mops::Tensor<int32_t, 1>{nullptr, {0}}, scale
        );
    });
    return grad_table;
}

at::Tensor scaled_embedding(const at::Tensor& table, const at::Tensor& indices, double scale);

struct EmbeddingVjp : public Function<EmbeddingVjp> {
    static at::Tensor forward(
        AutogradContext* ctx, at::Tensor grad_output, at::Tensor indices, int64_t table_rows, double scale
    ) {
        ctx->save_for_backward({indices});
        ctx->saved_data["scale"] = scale;
        return embedding_vjp(grad_output, indices, table_rows, scale);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const at::Tensor indices = ctx->get_saved_variables()[0];
        return {
            scaled_embedding(grads[0], indices, ctx->saved_data["scale"].toDouble()), at::Tensor(), at::Tensor(),
            at::Tensor(),
        };
    }
};

struct EmbeddingFunction : public Function<EmbeddingFunction> {
    static at::Tensor forward(AutogradContext* ctx, at::Tensor table, at::Tensor indices, double scale) {
        ctx->save_for_backward({indices});
        ctx->saved_data["table_rows"] = table.dim() == 2 ? table.size(0) : 0;
        ctx->saved_data["scale"] = scale;
        return embedding_forward(table, indices, scale);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const at::Tensor indices = ctx->get_saved_variables()[0];
        const int64_t table_rows = ctx->saved_data["table_rows"].toInt();
        const double scale = ctx->saved_data["scale"].toDouble();
        const at::Tensor grad_table = recorded({&grads[0]})
                                          ? EmbeddingVjp::apply(grads[0], indices, table_rows, scale)
                                          : embedding_vjp(grads[0], indices, table_rows, scale);
        return {grad_table, at::Tensor(), at::Tensor()};
    }
};

at::Tensor grouped_forward(
    const at::Tensor& A_, const at::Tensor& W_, const at::Tensor& offsets_, const at::Tensor& order_
) {
    const char* op = "grouped_matrix_product";
    const at::Tensor A = layer_values(A_, A_, "A", "A", op), W = layer_values(W_, A_, "W", "A", op);
    const at::Tensor offsets = layer_indices(offsets_, A_, "offsets", op), order = layer_indices(order_, A_, "order", op);
    OnTorchStream stream(A);
    at::Tensor output = new_tensor({A.dim() == 2 ? A.size(0) : 0, W.dim() == 3 ? W.size(2) : 0}, A);
    by_layer_dtype(A, [&](auto zero) {
        using T = decltype(zero);
        mops::cuda::grouped_matrix_product<T>(
            view<T, 2>(output, "output"), view<T, 2>(A, "A"), view<T, 3>(W, "W"), view<int32_t, 1>(offsets, "offsets"),
            view<int32_t, 1>(order, "order")
        );
    });
    return output;
}

/// An argument of a Function that may be missing: undefined tensors are none it takes.
c10::optional<at::Tensor> optional(const at::Tensor& tensor) {
    return tensor.defined() ? c10::optional<at::Tensor>(tensor) : c10::nullopt;
}
at::Tensor or_undefined(const c10::optional<at::Tensor>& tensor) { return tensor.has_value() ? *tensor : at::Tensor(); }

/// grad_A, grad_W; a gradient that is not wanted comes back undefined.
std::array<at::Tensor, 2> grouped_vjp(
    const at::Tensor& grad_output_, const at::Tensor& A_, const at::Tensor& W_, const at::Tensor& offsets_,
    const at::Tensor& order_, bool want_A, bool want_W
) {
    const char* op = "grouped_matrix_product_vjp";
    const at::Tensor A = layer_values(A_, A_, "A", "A", op), W = layer_values(W_, A_, "W", "A", op);
    const at::Tensor offsets = layer_indices(offsets_, A_, "offsets", op), order = layer_indices(order_, A_, "order", op);
    const at::Tensor grad_output = layer_values(grad_output_, A_, "grad_output", "A", op);
    OnTorchStream stream(A);
    at::Tensor grad_A = want_A ? new_like(A) : at::Tensor(), grad_W = want_W ? new_like(W) : at::Tensor();
    by_layer_dtype(A, [&](auto zero) {
        using T = decltype(zero);
        mops::cuda::grouped_matrix_product_vjp<T>(
            view<T, 2>(grad_A, "grad_A"), view<T, 3>(grad_W, "grad_W"), view<T, 2>(grad_output, "grad_output"),
            view<T, 2>(A, "A"), view<T, 3>(W, "W"), view<int32_t, 1>(offsets, "offsets"),
            view<int32_t, 1>(order, "order")
        );
    });
    return {grad_A, grad_W};
}

at::Tensor grouped_product(const at::Tensor& A, const at::Tensor& W, const at::Tensor& offsets, const at::Tensor& order);
std::array<at::Tensor, 2> grouped_gradients(
    const at::Tensor& grad_output, const at::Tensor& A, const at::Tensor& W, const at::Tensor& offsets,
    const at::Tensor& order, bool want_A, bool want_W
);

struct GroupedVjp : public Function<GroupedVjp> {
    static variable_list forward(
        AutogradContext* ctx, at::Tensor grad_output, at::Tensor A, at::Tensor W, at::Tensor offsets,
        c10::optional<at::Tensor> order_, bool want_A, bool want_W
    ) {
        const at::Tensor order = or_undefined(order_);
        ctx->save_for_backward({grad_output, A, W, offsets, order});
        ctx->saved_data["want_A"] = want_A;
        ctx->saved_data["want_W"] = want_W;
        ctx->set_materialize_grads(false);
        const auto gradients = grouped_vjp(grad_output, A, W, offsets, order, want_A, want_W);
        return {want_A ? gradients[0] : nothing(A), want_W ? gradients[1] : nothing(W)};
    }
    /// With u, v for grad_A = c W^T and grad_W = A^T c (c: grad_output), all of them by group: the gradient for c is
    /// u W + A v (each rounded by itself, as autograd adds up gradients), that for A is c v^T, that for W is u^T c.
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const at::Tensor &grad_output = saved[0], &A = saved[1], &W = saved[2], &offsets = saved[3], &order = saved[4];
        const at::Tensor u = or_undefined(grads[0], ctx->saved_data["want_A"].toBool());
        const at::Tensor v = or_undefined(grads[1], ctx->saved_data["want_W"].toBool());
        variable_list result(7);
        if (ctx->needs_input_grad(0)) {
            const at::Tensor from_u = u.defined() ? grouped_product(u, W, offsets, order) : at::Tensor();
            const at::Tensor from_v = v.defined() ? grouped_product(A, v, offsets, order) : at::Tensor();
            result[0] = from_u.defined() && from_v.defined() ? from_u + from_v : from_u.defined() ? from_u : from_v;
        }
        if (ctx->needs_input_grad(1) && v.defined()) {
            result[1] = grouped_gradients(grad_output, A, v, offsets, order, true, false)[0];
        }
        if (ctx->needs_input_grad(2) && u.defined()) {
            result[2] = grouped_gradients(grad_output, u, W, offsets, order, false, true)[1];
        }
        return result;
    }
};

std::array<at::Tensor, 2> grouped_gradients(
    const at::Tensor& grad_output, const at::Tensor& A, const at::Tensor& W, const at::Tensor& offsets,
    const at::Tensor& order, bool want_A, bool want_W
) {
    if (!recorded({&grad_output, &A, &W})) {
        return grouped_vjp(grad_output, A, W, offsets, order, want_A, want_W);
    }
    const variable_list gradients = GroupedVjp::apply(grad_output, A, W, offsets, optional(order), want_A, want_W);
    return {or_undefined(gradients[0], want_A), or_undefined(gradients[1], want_W)};
}

struct GroupedFunction : public Function<GroupedFunction> {
    static at::Tensor forward(
        AutogradContext* ctx, at::Tensor A, at::Tensor W, at::Tensor offsets, c10::optional<at::Tensor> order
    ) {
        ctx->save_for_backward({A, W, offsets, or_undefined(order)});
        return grouped_forward(A, W, offsets, or_undefined(order));
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const auto gradients = grouped_gradients(
            grads[0], saved[0], saved[1], saved[2], saved[3], ctx->needs_input_grad(0), ctx->needs_input_grad(1)
        );
        return {gradients[0], gradients[1], at::Tensor(), at::Tensor()};
    }
};

/// residual, block, gate, weight_block, weight_next
std::array<at::Tensor, 5> update_inputs(const std::array<at::Tensor, 5>& tensors, const char* op) {
    const char* names[5] = {"residual", "block", "gate", "weight_block", "weight_next"};
    std::array<at::Tensor, 5> inputs;
    for (size_t i = 0; i < 5; i++) {
        inputs[i] = layer_values(tensors[i], tensors[0], names[i], names[0], op);
    }
    return inputs;
}

std::tuple<at::Tensor, at::Tensor> update_forward(
    const std::array<at::Tensor, 5>& tensors, double residual_scale, double epsilon
) {
    const auto in = update_inputs(tensors, "gated_residual_norm");
    OnTorchStream stream(in[0]);
    at::Tensor state = new_like(in[0]), next = new_like(in[0]);
    by_layer_dtype(in[0], [&](auto zero) {
        using T = decltype(zero);
        mops::cuda::gated_residual_norm<T>(
            view<T, 2>(state, "state"), view<T, 2>(next, "next"), view<T, 2>(in[0], "residual"),
            view<T, 2>(in[1], "block"), view<T, 2>(in[2], "gate"), view<T, 1>(in[3], "weight_block"),
            view<T, 1>(in[4], "weight_next"), residual_scale, epsilon
        );
    });
    return {state, next};
}

typedef std::array<bool, 5> Wanted;

/// The gradients; undefined where not wanted. grad_state, grad_next: undefined for zero.
std::array<at::Tensor, 5> update_vjp(
    const at::Tensor& grad_state, const at::Tensor& grad_next, const std::array<at::Tensor, 5>& tensors,
    double residual_scale, double epsilon, const Wanted& wanted
) {
    const char* op = "gated_residual_norm_vjp";
    const auto in = update_inputs(tensors, op);
    const std::array<at::Tensor, 2> grads = {grad_state, grad_next};
    std::array<at::Tensor, 2> cotangent;
    for (size_t i = 0; i < 2; i++) {
        cotangent[i] = grads[i].defined()
                           ? layer_values(grads[i], in[0], i == 0 ? "grad_state" : "grad_next", "residual", op)
                           : at::Tensor();
    }
    OnTorchStream stream(in[0]);
    std::array<at::Tensor, 5> out;
    for (size_t i = 0; i < 5; i++) {
        out[i] = wanted[i] ? new_like(in[i]) : at::Tensor();
    }
    by_layer_dtype(in[0], [&](auto zero) {
        using T = decltype(zero);
        mops::cuda::gated_residual_norm_vjp<T>(
            view<T, 2>(out[0], "grad_residual"), view<T, 2>(out[1], "grad_block"), view<T, 2>(out[2], "grad_gate"),
            view<T, 1>(out[3], "grad_weight_block"), view<T, 1>(out[4], "grad_weight_next"),
            view<T, 2>(cotangent[0], "grad_state"), view<T, 2>(cotangent[1], "grad_next"),
            view<T, 2>(in[0], "residual"), view<T, 2>(in[1], "block"), view<T, 2>(in[2], "gate"),
            view<T, 1>(in[3], "weight_block"), view<T, 1>(in[4], "weight_next"), residual_scale, epsilon
        );
    });
    return out;
}

/// The gradients where they are recorded themselves: there is no derivative of them, which whoever asks for one is told.
struct UpdateVjp : public Function<UpdateVjp> {
    static variable_list forward(
        AutogradContext*, c10::optional<at::Tensor> grad_state_, c10::optional<at::Tensor> grad_next_, at::Tensor residual,
        at::Tensor block, at::Tensor gate, at::Tensor weight_block, at::Tensor weight_next, double residual_scale,
        double epsilon, Wanted wanted
    ) {
        const at::Tensor grad_state = or_undefined(grad_state_), grad_next = or_undefined(grad_next_);
        const std::array<at::Tensor, 5> in = {residual, block, gate, weight_block, weight_next};
        const auto gradients = update_vjp(grad_state, grad_next, in, residual_scale, epsilon, wanted);
        variable_list results;
        for (size_t i = 0; i < 5; i++) {
            results.push_back(wanted[i] ? gradients[i] : nothing(residual));
        }
        return results;
    }
    static variable_list backward(AutogradContext*, variable_list) {
        throw std::runtime_error("mops::gated_residual_norm: second derivatives are not supported");
    }
};

struct UpdateFunction : public Function<UpdateFunction> {
    static variable_list forward(
        AutogradContext* ctx, at::Tensor residual, at::Tensor block, at::Tensor gate, at::Tensor weight_block,
        at::Tensor weight_next, double residual_scale, double epsilon
    ) {
        ctx->save_for_backward({residual, block, gate, weight_block, weight_next});
        ctx->saved_data["residual_scale"] = residual_scale;
        ctx->saved_data["epsilon"] = epsilon;
        ctx->set_materialize_grads(false); // (a gradient that is not there is not read)
        const auto [state, next] =
            update_forward({residual, block, gate, weight_block, weight_next}, residual_scale, epsilon);
        return {state, next};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto in = ctx->get_saved_variables();
        const double scale = ctx->saved_data["residual_scale"].toDouble(), epsilon = ctx->saved_data["epsilon"].toDouble();
        Wanted wanted;
        for (size_t i = 0; i < 5; i++) {
            wanted[i] = ctx->needs_input_grad(i);
        }
        variable_list result(7);
        if (recorded({&grads[0], &grads[1], &in[0], &in[1], &in[2], &in[3], &in[4]})) {
            const variable_list gradients =
                UpdateVjp::apply(
                    optional(grads[0]), optional(grads[1]), in[0], in[1], in[2], in[3], in[4], scale, epsilon, wanted
                );
            for (size_t i = 0; i < 5; i++) {
                result[i] = or_undefined(gradients[i], wanted[i]);
            }
        } else {
            const auto gradients = update_vjp(grads[0], grads[1], {in[0], in[1], in[2], in[3], in[4]}, scale, epsilon, wanted);
            std::copy(gradients.begin(), gradients.end(), result.begin());
        }
        return result;
    }
};

// ------------------------------------------------------------ operators --
at::Tensor scaled_embedding(const at::Tensor& table, const at::Tensor& indices, double scale) {
    return recorded({&table}) ? EmbeddingFunction::apply(table, indices, scale)
                              : embedding_forward(table, indices, scale);
}

at::Tensor grouped_product(const at::Tensor& A, const at::Tensor& W, const at::Tensor& offsets, const at::Tensor& order) {
    return recorded({&A, &W}) ? GroupedFunction::apply(A, W, offsets, optional(order))
                              : grouped_forward(A, W, offsets, order);
}

at::Tensor grouped_matrix_product(
    const at::Tensor& A, const at::Tensor& W, const at::Tensor& offsets, const c10::optional<at::Tensor>& order
) {
    return grouped_product(A, W, offsets, or_undefined(order));
}

std::tuple<at::Tensor, at::Tensor> gated_residual_norm(
    const at::Tensor& residual, const at::Tensor& block, const at::Tensor& gate, const at::Tensor& weight_block,
    const at::Tensor& weight_next, double residual_scale, double epsilon
) {
    if (!recorded({&residual, &block, &gate, &weight_block, &weight_next})) {
        return update_forward({residual, block, gate, weight_block, weight_next}, residual_scale, epsilon);
    }
    const variable_list results =
        UpdateFunction::apply(residual, block, gate, weight_block, weight_next, residual_scale, epsilon);
    return {results[0], results[1]};
}

at::Tensor homogeneous_polynomial_evaluation(const at::Tensor& A, const at::Tensor& C, const at::Tensor& indices_A) {
    return recorded({&A, &C}) ? Hpe::apply(A, C, indices_A) : hpe_forward(A, C, indices_A);
}

at::Tensor outer_product_scatter_add(
    const at::Tensor& A, const at::Tensor& B, const at::Tensor& indices_output, int64_t output_size
) {
    const variable_list extra = {indices_output};
    return recorded({&A, &B}) ? Bilinear<Opsa>::apply(A, B, at::TensorList(extra), output_size)
                              : bilinear_forward<Opsa>(A, B, extra, output_size);
}

at::Tensor sparse_accumulation_of_products(
    const at::Tensor& A, const at::Tensor& B, const at::Tensor& C, const at::Tensor& indices_A,
    const at::Tensor& indices_B, const at::Tensor& indices_output, int64_t output_size
) {
    const variable_list extra = {C, indices_A, indices_B, indices_output};
    return recorded({&A, &B, &C}) ? Bilinear<Sap>::apply(A, B, at::TensorList(extra), output_size)
                                  : bilinear_forward<Sap>(A, B, extra, output_size);
}

at::Tensor outer_product_scatter_add_with_weights(
    const at::Tensor& A, const at::Tensor& B, const at::Tensor& W, const at::Tensor& indices_W,
    const at::Tensor& indices_output
) {
    return recorded({&A, &B, &W}) ? OpsawFunction::apply(A, B, W, indices_W, indices_output)
                                  : opsaw_forward(A, B, W, indices_W, indices_output);
}

at::Tensor sparse_accumulation_scatter_add_with_weights(
    const at::Tensor& A, const at::Tensor& B, const at::Tensor& C, const at::Tensor& W, const at::Tensor& indices_A,
    const at::Tensor& indices_W_1, const at::Tensor& indices_W_2, const at::Tensor& indices_output_1,
    const at::Tensor& indices_output_2, int64_t output_size
) {
    return recorded({&A, &B, &C, &W})
               ? SasawFunction::apply(
                     A, B, C, W, indices_A, indices_W_1, indices_W_2, indices_output_1, indices_output_2, output_size
                 )
               : sasaw_forward(
                     A, B, C, W, indices_A, indices_W_1, indices_W_2, indices_output_1, indices_output_2, output_size
                 );
}

} // namespace

TORCH_LIBRARY(mops, m) {
    m.def("order_by_group(Tensor indices, int n_groups) -> (Tensor, Tensor)", order_by_group);
    m.def("scaled_embedding(Tensor table, Tensor indices, float scale=1.) -> Tensor", scaled_embedding);
    m.def(
        "grouped_matrix_product(Tensor A, Tensor W, Tensor offsets, Tensor? order=None) -> Tensor",
        grouped_matrix_product
    );
    m.def(
        "gated_residual_norm(Tensor residual, Tensor block, Tensor gate, Tensor weight_block, Tensor weight_next, "
        "float residual_scale=1., float epsilon=1e-06) -> (Tensor, Tensor)",
        gated_residual_norm
    );
    m.def(
        "homogeneous_polynomial_evaluation(Tensor A, Tensor C, Tensor indices_A) -> Tensor",
        homogeneous_polynomial_evaluation
    );
    m.def(
        "outer_product_scatter_add(Tensor A, Tensor B, Tensor indices_output, int output_size) -> Tensor",
        outer_product_scatter_add
    );
    m.def(
        "sparse_accumulation_of_products(Tensor A, Tensor B, Tensor C, Tensor indices_A, Tensor indices_B, "
        "Tensor indices_output, int output_size) -> Tensor",
        sparse_accumulation_of_products
    );
    m.def(
        "outer_product_scatter_add_with_weights(Tensor A, Tensor B, Tensor W, Tensor indices_W, "
        "Tensor indices_output) -> Tensor",
        outer_product_scatter_add_with_weights
    );
    m.def(
        "sparse_accumulation_scatter_add_with_weights(Tensor A, Tensor B, Tensor C, Tensor W, Tensor indices_A, "
        "Tensor indices_W_1, Tensor indices_W_2, Tensor indices_output_1, Tensor indices_output_2, "
        "int output_size) -> Tensor",
        sparse_accumulation_scatter_add_with_weights
    );
}
