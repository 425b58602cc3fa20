// What the callers of this library on PyTorch tensors (torch_ops.cpp,
// array_ops.cpp) share: views, the stream, and outputs.
#ifndef MOPS_AMD_TORCH_TENSORS_HPP
#define MOPS_AMD_TORCH_TENSORS_HPP

#include <stdexcept>
#include <string>
#include <type_traits>
#include <vector>

#include <ATen/hip/EmptyTensor.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/InferenceMode.h>
#include <torch/types.h>

#include "mops/amd.h"
#include "mops/layers.hpp"
#include "mops/tensor.hpp"

namespace mops::amd::torch_tensors {

template <typename T, size_t N> mops::Tensor<T, N> view(const at::Tensor& tensor, const char* name) {
    mops::Tensor<T, N> result{nullptr, {}};
    for (size_t d = 0; d < N; d++) {
        result.shape[d] = 0;
    }
    if (!tensor.defined()) {
        return result; // "not wanted" / "not given": a null view
    }
    if (static_cast<size_t>(tensor.dim()) != N) {
        throw std::runtime_error(
            std::string(name) + " must have " + std::to_string(N) + " dimensions, got " + std::to_string(tensor.dim())
        );
    }
    if constexpr (sizeof(T) == 2) { // (the bits; by_layer_dtype has looked at the type)
        result.data = static_cast<T*>(tensor.data_ptr());
    } else {
        result.data = tensor.data_ptr<T>();
    }
    for (size_t d = 0; d < N; d++) {
        result.shape[d] = static_cast<size_t>(tensor.size(static_cast<int64_t>(d)));
    }
    return result;
}

/// The library's launches go to PyTorch's current stream of the tensors' device, without blocking.
/// (In a ROCm build of PyTorch the HIP device type goes under the name of CUDA: these are the
/// guard and the stream of that build.)
struct OnTorchStream {
    c10::hip::HIPGuardMasqueradingAsCUDA guard;
    explicit OnTorchStream(const at::Tensor& tensor) : guard(tensor.device()) {
        mops_amd_set_stream(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream());
        mops_amd_set_synchronous(0);
    }
};

template <typename Body> void by_dtype(const at::Tensor& like, Body&& body) {
    if (like.scalar_type() == at::kFloat) {
        body(float{});
    } else {
        body(double{});
    }
}

/// The element types of the layers' operators (mops/layers.h).
inline bool is_layer_dtype(at::ScalarType type) {
    return type == at::kFloat || type == at::kDouble || type == at::kBFloat16 || type == at::kHalf;
}
template <typename Body> void by_layer_dtype(const at::Tensor& like, Body&& body) {
    if (like.scalar_type() == at::kBFloat16) {
        body(mops::bfloat16{});
    } else if (like.scalar_type() == at::kHalf) {
        body(mops::float16{});
    } else {
        by_dtype(like, body);
    }
}

/// An uninitialised tensor beside `like` (the library overwrites its outputs completely), from the
/// caching allocator without a turn through the dispatcher: 0.5 us instead of 0.7.
inline at::Tensor new_tensor(at::IntArrayRef sizes, const at::Tensor& like) {
    return at::detail::empty_cuda(
        sizes, like.scalar_type(), c10::nullopt, like.device(), c10::nullopt, c10::nullopt
    );
}
inline at::Tensor new_like(const at::Tensor& like) { return new_tensor(like.sizes(), like); }

/// What the sums of an element type are held in.
template <typename T> using sum_t = std::conditional_t<std::is_same_v<T, double>, double, float>;
inline at::ScalarType sum_dtype(const at::Tensor& like) {
    return like.scalar_type() == at::kDouble ? at::kDouble : at::kFloat;
}
/// A sum for each row of `like`.
inline at::Tensor new_sums(const at::Tensor& like) {
    return at::detail::empty_cuda(
        {like.dim() > 0 ? like.size(0) : 0}, sum_dtype(like), c10::nullopt, like.device(), c10::nullopt, c10::nullopt
    );
}

// ------------------------------------------------------ lists of gradients --
/// A tensor whose numbers fill a piece of device memory, in whatever order of dimensions.
inline bool is_gradient(const at::Tensor& t) {
    return t.is_cuda() && t.layout() == at::kStrided && t.has_storage() && !t.is_neg() &&
           is_layer_dtype(t.scalar_type()) && t.is_non_overlapping_and_dense();
}
/// Whether it may be written to here: a tensor that was made in inference mode has no version to count up outside of it, and
/// counting throws (too late, behind the launches that write).
inline bool is_writable(const at::Tensor& t) { return !t.is_inference() || c10::InferenceMode::is_enabled(); }
/// Autograd is told (of tensors that are writable).
inline void mark_written(const std::vector<at::Tensor>& gradients) {
    for (const at::Tensor& gradient : gradients) {
        gradient.unsafeGetTensorImpl()->bump_version();
    }
}
/// Their likes, in the same order of dimensions. Up to SMALL_LIST bytes they share one piece of memory, which is asked for
/// once (20 tensors of 2 MB: 23 us a call with memory for each, 14 like this); larger ones have their own, which
/// can be given back one by one.
constexpr int64_t SMALL_LIST = int64_t(16) << 20;
inline std::vector<at::Tensor> new_gradients(const std::vector<at::Tensor>& gradients) {
    constexpr int64_t ALIGNMENT = 256;
    auto bytes_of = [](const at::Tensor& t) {
        return (t.numel() * static_cast<int64_t>(t.element_size()) + ALIGNMENT - 1) / ALIGNMENT * ALIGNMENT;
    };
    int64_t bytes = 0;
    for (const at::Tensor& gradient : gradients) {
        bytes += bytes_of(gradient);
    }
    std::vector<at::Tensor> outputs;
    outputs.reserve(gradients.size());
    if (bytes > SMALL_LIST) {
        for (const at::Tensor& gradient : gradients) {
            outputs.push_back(gradient.is_contiguous() ? new_like(gradient) : at::empty_like(gradient));
        }
        return outputs;
    }
    const at::Tensor memory = at::detail::empty_cuda(
        {bytes}, at::kByte, c10::nullopt, gradients[0].device(), c10::nullopt, c10::nullopt
    );
    int64_t at = 0;
    for (const at::Tensor& gradient : gradients) {
        at::Tensor output = at::detail::make_tensor<c10::TensorImpl>(
            c10::Storage(memory.storage()), memory.key_set(), gradient.dtype()
        );
        c10::TensorImpl* const impl = output.unsafeGetTensorImpl();
        impl->set_storage_offset(at / static_cast<int64_t>(gradient.element_size()));
        impl->set_sizes_and_strides(gradient.sizes(), gradient.strides());
        outputs.push_back(std::move(output));
        at += bytes_of(gradient);
    }
    return outputs;
}
inline at::Tensor new_norm(const std::vector<at::Tensor>& gradients) {
    bool wide = false;
    for (const at::Tensor& gradient : gradients) {
        wide = wide || gradient.scalar_type() == at::kDouble;
    }
    return at::detail::empty_cuda(
        {}, wide ? at::kDouble : at::kFloat, c10::nullopt, gradients[0].device(), c10::nullopt, c10::nullopt
    );
}
inline std::vector<mops::Gradient> views_of(const std::vector<at::Tensor>& gradients) {
    std::vector<mops::Gradient> views;
    views.reserve(gradients.size());
    for (const at::Tensor& gradient : gradients) {
        const at::ScalarType type = gradient.scalar_type();
        views.push_back(mops::Gradient{
            gradient.data_ptr(), gradient.numel(),
            type == at::kFloat    ? mops::GradientType::F32
            : type == at::kDouble ? mops::GradientType::F64
            : type == at::kHalf   ? mops::GradientType::F16
                                  : mops::GradientType::BF16,
        });
    }
    return views;
}
inline void norm_of_gradients(const at::Tensor& norm, const std::vector<at::Tensor>& gradients) {
    const auto views = views_of(gradients);
    by_dtype(norm, [&](auto zero) {
        using T = decltype(zero);
        mops::cuda::gradient_norm<T>(mops::Tensor<T, 1>{norm.data_ptr<T>(), {1}}, views.data(), views.size());
    });
}
/// (outputs: the gradients themselves, in place)
inline void clip_gradients_to(
    const at::Tensor& norm, const std::vector<at::Tensor>& outputs, const std::vector<at::Tensor>& gradients,
    double max_norm
) {
    const auto to = views_of(outputs), from = views_of(gradients);
    by_dtype(norm, [&](auto zero) {
        using T = decltype(zero);
        mops::cuda::clip_gradients<T>(
            mops::Tensor<T, 1>{norm.data_ptr<T>(), {1}}, to.data(), from.data(), from.size(), max_norm
        );
    });
}

} // namespace mops::amd::torch_tensors

#endif
