// The norm of all gradients of a network together, and the gradients scaled so
// that it is at most max_norm:
//
//   norm = sqrt(sum over all tensors and numbers of g^2)
//   output = g min(1, max_norm / norm)
//
// Any number of tensors of any sizes and types goes through one launch per
// TENSORS of them: their addresses and sizes travel as kernel arguments (a
// captured launch keeps its own), and their numbers are cut into chunks that the
// workgroups take in turn. Squares are added up in 64 bits, where neither those
// of the largest 32-bit or bfloat16 number nor a sum of billions of them lose
// anything that matters; 64-bit numbers whose squares would leave the range have
// sums of their own, of squares at another scale (Squares). The order depends on
// the sizes only. Every workgroup of
// the second launch adds up the partial sums for itself, and goes through the
// chunks from the last one back: the caches still hold those.
//
// Bound by memory: the gradients are read once for the norm, read and written
// once to be scaled; in place and below max_norm nothing is read again.
#include "mops/layers.hpp"

#include <algorithm>
#include <cmath>
#include <limits>
#include <type_traits>
#include <vector>

#include "device_common.hpp"
#include "numbers.hpp"
#include "runtime.hpp"

namespace mops::amd::gradient_norm {
namespace {

using mops::Gradient;
using mops::GradientType;

constexpr int THREADS = 256;
constexpr int PIECES_EACH = 8;                                // of 16 bytes, of a thread and chunk
constexpr int64_t CHUNK_BYTES = int64_t(THREADS) * PIECES_EACH * 16;
constexpr int TENSORS = 64;                                   // of a launch: 2 KB of arguments
constexpr int64_t WORKGROUPS_PER_UNIT = 8;                    // all that a compute unit has room for

int64_t size_of(GradientType type) {
    return type == GradientType::F64 ? 8 : type == GradientType::F32 ? 4 : 2;
}
int64_t chunks_of(const Gradient& g) { return static_cast<int64_t>(ceil_div(g.size * size_of(g.type), CHUNK_BYTES)); }

struct Table {
    const void* from[TENSORS];
    void* to[TENSORS];
    int64_t size[TENSORS];
    int64_t end[TENSORS]; // chunks of the tensors up to this one
    GradientType type[TENSORS];
    int32_t count;

    __device__ __forceinline__ int64_t chunks() const { return end[count - 1]; }
    __device__ __forceinline__ int64_t begin_of(int32_t tensor) const { return tensor > 0 ? end[tensor - 1] : 0; }
    /// Which tensor has chunk `chunk`.
    __device__ __forceinline__ int32_t tensor_of(int64_t chunk) const {
        int32_t low = 0, high = count - 1;
        while (low < high) {
            const int32_t middle = (low + high) / 2;
            if (end[middle] > chunk) {
                high = middle;
            } else {
                low = middle + 1;
            }
        }
        return low;
    }
};

/// body(zero of the type).
template <typename Body> __device__ __forceinline__ void by_type(GradientType type, Body&& body) { // (uniform)
    if (type == GradientType::F32) {
        body(0.f);
    } else if (type == GradientType::BF16) {
        body(static_cast<__bf16>(0.f));
    } else if (type == GradientType::F16) {
        body(static_cast<_Float16>(0.f));
    } else {
        body(0.0);
    }
}

/// Consecutive chunks of a tensor, the workgroup's: numbers begin .. end - 1, whole chunks but for the tensor's last.
template <typename T> struct Part {
    static constexpr int COUNT = PIECE<T>;
    static constexpr int64_t NUMBERS = CHUNK_BYTES / sizeof(T);
    typedef Piece<T, COUNT> Numbers;
    int64_t begin, end;

    /// chunk(at, count) for every chunk, in order or from the last one back: the thread's first number in it, and how many of
    /// its pieces exist (compile-time PIECES_EACH in whole chunks). one(at) for numbers behind the last whole piece.
    template <bool BACK, typename OfChunk, typename One>
    __device__ __forceinline__ void go(OfChunk&& chunk, One&& one) const {
        const int64_t all = (end - begin) / NUMBERS;
        const int64_t rest = begin + all * NUMBERS, pieces = (end - rest) / COUNT;
        if (rest < end) { // (uniform)
            const int64_t mine = (pieces - threadIdx.x + THREADS - 1) / THREADS; // (none: 0 or less)
            chunk(rest + threadIdx.x * COUNT, static_cast<int>(mine));
            const int64_t at = rest + pieces * COUNT + threadIdx.x;
            if (at < end) {
                one(at);
            }
        }
        for (int64_t c = 0; c < all; c++) {
            chunk(
                begin + (BACK ? all - 1 - c : c) * NUMBERS + threadIdx.x * COUNT, std::integral_constant<int, PIECES_EACH>{}
            );
        }
    }
    static __device__ __forceinline__ int64_t of_piece(int i) { return static_cast<int64_t>(i) * THREADS * COUNT; }
};

/// Every workgroup has consecutive chunks of all tensors (it looks for the first one's tensor once, and the caches see
/// streams): body(zero of the type, tensor, its part), in order or from the last one back.
template <bool BACK, typename Body> __device__ __forceinline__ void for_parts(const Table& table, Body&& body) {
    const int64_t chunks = table.chunks();
    const int64_t first = chunks * blockIdx.x / gridDim.x, last = chunks * (blockIdx.x + 1) / gridDim.x;
    if (first >= last) {
        return;
    }
    for (int32_t tensor = table.tensor_of(BACK ? last - 1 : first);; tensor += BACK ? -1 : 1) {
        const int64_t begin = table.begin_of(tensor);
        by_type(table.type[tensor], [&](auto zero) {
            typedef decltype(zero) T;
            const int64_t from = max(first - begin, int64_t(0)), to = min(last, table.end[tensor]) - begin;
            body(zero, tensor, Part<T>{from * Part<T>::NUMBERS, min(to * Part<T>::NUMBERS, table.size[tensor])});
        });
        if (BACK ? begin <= first : table.end[tensor] >= last) {
            return;
        }
    }
}

/// Sums of squares. Of 64-bit numbers, those above LARGE and below SMALL have sums of their own, of the numbers times
/// 2^-SCALE and 2^SCALE: the squares of all others, 2^60 of them, and those of the scaled ones are ordinary numbers (three
/// sums by size: J. L. Blue, ACM Trans. Math. Software 4, 1978). Infinities are large, what is not a number is ordinary.
struct Squares {
    static constexpr double LARGE = 0x1p480, SMALL = 0x1p-480;
    static constexpr int SCALE = 600;
    double ordinary, large, small;

    __device__ __forceinline__ void add(double x) {
        const bool is_large = fabs(x) > LARGE, is_small = fabs(x) < SMALL;
        const double scaled = x * (is_large ? 0x1p-600 : is_small ? 0x1p600 : 1.0), square = scaled * scaled;
        large += is_large ? square : 0;
        small += is_small ? square : 0;
        ordinary += is_large || is_small ? 0 : square;
    }
};
/// A norm: `number` times a power of two.
struct Norm {
    double number;
    int exponent;

    /// (infinite beyond the range)
    __device__ __forceinline__ double rounded() const { return ldexp(number, exponent); }
    static __device__ __forceinline__ Norm of(const Squares& squares) {
        if (squares.large != 0) {
            return Norm{sqrt(squares.large + ldexp(squares.ordinary, -2 * Squares::SCALE)), Squares::SCALE};
        }
        return squares.ordinary != 0 ? Norm{sqrt(squares.ordinary + ldexp(squares.small, -2 * Squares::SCALE)), 0}
                                     : Norm{sqrt(squares.small), -Squares::SCALE};
    }
};

__device__ __forceinline__ double sum_of_wave(double sum) {
#pragma unroll
    for (int s = 1; s < WAVE; s *= 2) {
        sum += __shfl_xor(sum, s);
    }
    return sum;
}
/// The sum over the workgroup, in all threads.
__device__ __forceinline__ double sum_of_workgroup(double sum) {
    __shared__ double of_wave[THREADS / WAVE];
    sum = sum_of_wave(sum);
    __syncthreads(); // (of another sum in front)
    if (threadIdx.x % WAVE == 0) {
        of_wave[threadIdx.x / WAVE] = sum;
    }
    __syncthreads();
    sum = 0;
#pragma unroll
    for (int w = 0; w < THREADS / WAVE; w++) {
        sum += of_wave[w];
    }
    return sum;
}

/// The partial sums of all workgroups in memory: [count] ordinary ones, and with 64-bit numbers among the gradients [count]
/// large and [count] small ones behind them.
struct Parts {
    int32_t count;
    bool of_doubles;

    size_t bytes() const { return align256(std::max<size_t>((of_doubles ? 3 : 1) * static_cast<size_t>(count), 1) * sizeof(double)); }
    __device__ __forceinline__ void store(double* partial, int32_t i, const Squares& squares) const {
        partial[i] = squares.ordinary;
        if (of_doubles) { // (uniform)
            partial[count + i] = squares.large;
            partial[2 * count + i] = squares.small;
        }
    }
};

/// KEPT: the gradients are read again, and the caches should have what they can (616 million bfloat16 numbers, squares and
/// scaling: 205 + 430 us; streamed past the caches 179 + 478). For the norm alone they stream past (260 million: 77 us, 6.8
/// TB/s).
template <bool KEPT>
__global__ __launch_bounds__(THREADS) void squares_kernel(double* __restrict__ partial, Parts parts, int32_t first, const Table table) {
    double sums[2] = {0, 0};
    Squares of_double{0, 0, 0};
    for_parts<false>(table, [&](auto zero, int32_t tensor, const auto& part) {
        typedef decltype(zero) T;
        typedef typename Part<T>::Numbers Numbers;
        const T* const from = static_cast<const T*>(table.from[tensor]);
        auto add_one = [&](double x, int e) {
            if constexpr (std::is_same_v<T, double>) {
                of_double.add(x);
            } else {
                sums[e % 2] += x * x;
            }
        };
        auto add = [&](const Numbers& numbers) {
#pragma unroll
            for (int e = 0; e < PIECE<T>; e++) {
                add_one(static_cast<double>(numbers.get(e)), e);
            }
        };
        part.template go<false>(
            [&](int64_t at, auto count) {
                Numbers numbers[PIECES_EACH]{};
#pragma unroll
                for (int i = 0; i < PIECES_EACH; i++) {
                    if (i < count) {
                        const T* const piece = from + at + part.of_piece(i);
                        numbers[i] = KEPT ? Numbers::load(piece) : Numbers::stream(piece);
                    }
                }
#pragma unroll
                for (int i = 0; i < PIECES_EACH; i++) {
                    add(numbers[i]);
                }
            },
            [&](int64_t at) { add_one(static_cast<double>(from[at]), 0); }
        );
    });
    const Squares all{
        sum_of_workgroup(sums[0] + sums[1] + of_double.ordinary), parts.of_doubles ? sum_of_workgroup(of_double.large) : 0,
        parts.of_doubles ? sum_of_workgroup(of_double.small) : 0
    };
    if (threadIdx.x == 0) {
        parts.store(partial, first + static_cast<int32_t>(blockIdx.x), all);
    }
}

/// The norm, from the partial sums of all workgroups, in all threads.
__device__ __forceinline__ Norm norm_of(const double* partial, const Parts& parts) {
    Squares sums{0, 0, 0};
#pragma unroll 4
    for (int32_t i = threadIdx.x; i < parts.count; i += THREADS) {
        sums.ordinary += partial[i];
    }
    sums.ordinary = sum_of_workgroup(sums.ordinary);
    if (parts.of_doubles) { // (uniform)
        for (int32_t i = threadIdx.x; i < parts.count; i += THREADS) {
            sums.large += partial[parts.count + i];
            sums.small += partial[2 * parts.count + i];
        }
        sums.large = sum_of_workgroup(sums.large);
        sums.small = sum_of_workgroup(sums.small);
    }
    return Norm::of(sums);
}

template <typename Sum>
__global__ __launch_bounds__(THREADS) void norm_kernel(Sum* __restrict__ norm, const double* __restrict__ partial, Parts parts) {
    const Norm all = norm_of(partial, parts);
    if (threadIdx.x == 0) {
        *norm = static_cast<Sum>(all.rounded());
    }
}

/// min(1, max_norm / norm) as `digits` (0.5 to 1) times a power of two: it can be far below the smallest number of its type
/// where numbers times it are ordinary ones (bfloat16 numbers of 3e38 that are clipped to a norm of 1e-3).
struct Factor {
    double digits;
    int exponent;
};
/// (a norm that is none, or infinite, makes of the gradients what the formula does)
__device__ __forceinline__ Factor factor_of(const Norm& norm, double max_norm) {
    if (norm.rounded() <= max_norm) {
        return Factor{1, 0};
    }
    int of_max = 0, of_norm = 0;
    const double ratio = frexp(max_norm, &of_max) / frexp(norm.number, &of_norm); // (0.5 to 2)
    const int more = ratio > 1 ? 1 : 0;
    return Factor{more > 0 ? 0.5 * ratio : ratio, of_max - of_norm - norm.exponent + more};
}
/// A number times the factor, rounded once. 16 bits: a factor of 32 bits is exact enough, 2^-24 beside the result's 2^-9. SMALL:
/// a factor that is no ordinary number of its type (an instruction more for each number: 616 million in bfloat16, 643 us
/// instead of 637). 32 bits: in 64, whose range no factor leaves that makes a number.
template <typename T, bool SMALL> struct Scaling {
    typedef std::conditional_t<sizeof(T) == 2, float, double> Wide;
    Wide factor;
    int exponent;

    __device__ __forceinline__ explicit Scaling(const Factor& f)
        : factor(static_cast<Wide>(SMALL ? f.digits : ldexp(f.digits, f.exponent))), exponent(f.exponent) {}
    __device__ __forceinline__ T operator()(T number) const {
        const Wide product = static_cast<Wide>(number) * factor;
        return static_cast<T>(SMALL ? ldexp(product, exponent) : product);
    }
};
/// body(the scaling).
template <typename T, typename Body> __device__ __forceinline__ void with_scaling(const Factor& factor, Body&& body) {
    constexpr int LEAST = std::numeric_limits<typename Scaling<T, false>::Wide>::min_exponent;
    if (sizeof(T) == 4 || factor.exponent >= LEAST) { // (uniform)
        body(Scaling<T, false>(factor));
    } else {
        body(Scaling<T, true>(factor));
    }
}

/// norm: null in all launches but one.
template <typename Sum>
__global__ __launch_bounds__(THREADS) void scale_kernel(
    Sum* __restrict__ norm, const double* __restrict__ partial, Parts parts, double max_norm, bool in_place, const Table table
) {
    const Norm all = norm_of(partial, parts);
    if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) {
        *norm = static_cast<Sum>(all.rounded());
    }
    if (in_place && all.rounded() <= max_norm) {
        return; // (uniform)
    }
    const Factor factor = factor_of(all, max_norm);
    for_parts<true>(table, [&](auto zero, int32_t tensor, const auto& part) {
        typedef decltype(zero) T;
        typedef typename Part<T>::Numbers Numbers;
        const T* const from = static_cast<const T*>(table.from[tensor]);
        T* const to = static_cast<T*>(table.to[tensor]);
        with_scaling<T>(factor, [&](const auto& by) {
            auto scaled = [&](const Numbers& numbers) {
                Numbers result;
#pragma unroll
                for (int e = 0; e < PIECE<T>; e++) {
                    result.v[e] = by(numbers.v[e]);
                }
                return result;
            };
            part.template go<true>(
                [&](int64_t at, auto count) {
                    Numbers numbers[PIECES_EACH];
#pragma unroll
                    for (int i = 0; i < PIECES_EACH; i++) {
                        if (i < count) {
                            numbers[i] = Numbers::stream(from + at + part.of_piece(i));
                        }
                    }
#pragma unroll
                    for (int i = 0; i < PIECES_EACH; i++) {
                        if (i < count) {
                            scaled(numbers[i]).stream_to(to + at + part.of_piece(i));
                        }
                    }
                },
                [&](int64_t at) { to[at] = by(from[at]); }
            );
        });
    });
}

/// The gradients in tables of TENSORS, those without numbers left out.
std::vector<Table> tables_of(const Gradient* outputs, const Gradient* gradients, size_t n) {
    std::vector<Table> tables;
    for (size_t i = 0; i < n; i++) {
        if (gradients[i].size == 0) {
            continue;
        }
        if (tables.empty() || tables.back().count == TENSORS) {
            tables.emplace_back();
            tables.back().count = 0;
        }
        Table& table = tables.back();
        const int32_t at = table.count++;
        table.from[at] = gradients[i].data;
        table.to[at] = outputs != nullptr ? outputs[i].data : nullptr;
        table.size[at] = gradients[i].size;
        table.type[at] = gradients[i].type;
        table.end[at] = (at > 0 ? table.end[at - 1] : 0) + chunks_of(gradients[i]);
    }
    return tables;
}
unsigned workgroups_of(const Table& table) {
    return static_cast<unsigned>(std::min<int64_t>(table.end[table.count - 1], WORKGROUPS_PER_UNIT * compute_units()));
}

/// The partial sums, in the thread's scratch memory, and what there is of them.
template <bool KEPT> double* sum_squares(const std::vector<Table>& tables, Parts& parts, hipStream_t stream) {
    parts = Parts{0, false};
    for (const Table& table : tables) {
        parts.count += static_cast<int32_t>(workgroups_of(table));
        parts.of_doubles = parts.of_doubles || std::find(table.type, table.type + table.count, GradientType::F64) != table.type + table.count;
    }
    double* const partial = static_cast<double*>(scratch(parts.bytes()));
    int32_t first = 0;
    for (const Table& table : tables) {
        squares_kernel<KEPT><<<workgroups_of(table), THREADS, 0, stream>>>(partial, parts, first, table);
        MOPS_HIP_CHECK(hipGetLastError());
        first += static_cast<int32_t>(workgroups_of(table));
    }
    return partial;
}

void check(const Gradient* gradients, size_t n, const char* what, const char* operation) {
    if (gradients == nullptr && n > 0) {
        throw std::runtime_error(std::string("there are no ") + what + " in " + operation);
    }
    for (size_t i = 0; i < n; i++) {
        const std::string name = std::string(what) + "[" + std::to_string(i) + "]";
        const int32_t type = static_cast<int32_t>(gradients[i].type);
        if (type < 0 || type > static_cast<int32_t>(GradientType::F16)) {
            throw std::runtime_error(name + " has no known type in " + operation);
        }
        if (gradients[i].size < 0 || (gradients[i].size > 0 && gradients[i].data == nullptr)) {
            throw std::runtime_error(name + " has no memory, or a negative size, in " + operation);
        }
    }
}

/// Every output is its own gradient's memory, or shares none with anything else; the norm shares none with anything (it is
/// written while gradients are read).
template <typename Sum> void check_memory(const Sum* norm, const Gradient* outputs, const Gradient* gradients, size_t n) {
    struct Span {
        const char *begin, *end;
    };
    auto span = [](const Gradient& g) {
        const char* const begin = static_cast<const char*>(g.data);
        return Span{begin, begin + g.size * size_of(g.type)};
    };
    std::vector<Span> written;
    for (size_t i = 0; i < n; i++) {
        if (outputs[i].size > 0) {
            written.push_back(span(outputs[i]));
        }
    }
    std::sort(written.begin(), written.end(), [](const Span& a, const Span& b) { return a.begin < b.begin; });
    for (size_t i = 1; i < written.size(); i++) {
        if (written[i].begin < written[i - 1].end) {
            throw std::runtime_error("outputs must not share memory with each other in clip_gradients");
        }
    }
    for (size_t i = 0; i < n; i++) {
        const Span read = span(gradients[i]);
        if (read.begin == read.end || outputs[i].data == gradients[i].data) {
            continue; // (others that write there would share memory with this output)
        }
        auto after = std::lower_bound(written.begin(), written.end(), read.end, [](const Span& a, const char* at) {
            return a.begin < at;
        });
        if (after != written.begin() && std::prev(after)->end > read.begin) {
            throw std::runtime_error(
                "an output must be its own gradient's memory, or share none with any gradient, in clip_gradients"
            );
        }
    }
    const Span of_norm{reinterpret_cast<const char*>(norm), reinterpret_cast<const char*>(norm + 1)};
    for (size_t i = 0; i < n; i++) {
        for (const Span& other : {span(gradients[i]), span(outputs[i])}) {
            if (other.begin != other.end && other.begin < of_norm.end && of_norm.begin < other.end) {
                throw std::runtime_error("norm must not share memory with a gradient or an output in clip_gradients");
            }
        }
    }
}

template <typename Sum, typename Norm> Sum* check_norm(const Norm& norm, const char* operation) {
    if (norm.shape[0] != 1) {
        throw std::runtime_error(std::string("norm must have one element in ") + operation);
    }
    if (norm.data == nullptr) {
        throw std::runtime_error(std::string("norm has no memory in ") + operation);
    }
    return norm.data;
}

} // namespace
} // namespace mops::amd::gradient_norm

namespace mops::cuda {

using namespace mops::amd;

template <typename sum_t>
void gradient_norm(Tensor<sum_t, 1> norm, const Gradient* gradients, size_t n_gradients) {
    namespace own = mops::amd::gradient_norm;
    sum_t* const to = own::check_norm<sum_t>(norm, "gradient_norm");
    own::check(gradients, n_gradients, "gradients", "gradient_norm");
    const auto tables = own::tables_of(nullptr, gradients, n_gradients);
    const hipStream_t stream = current_stream();
    own::Parts parts{};
    const double* const partial = own::sum_squares<false>(tables, parts, stream);
    own::norm_kernel<sum_t><<<1, own::THREADS, 0, stream>>>(to, partial, parts);
    finish_call("gradient_norm");
}

template <typename sum_t>
void clip_gradients(
    Tensor<sum_t, 1> norm, const Gradient* outputs, const Gradient* gradients, size_t n_gradients, double max_norm
) {
    namespace own = mops::amd::gradient_norm;
    sum_t* const to = own::check_norm<sum_t>(norm, "clip_gradients");
    if (!(max_norm >= 0)) {
        throw std::runtime_error("max_norm must be a number that is not negative in clip_gradients");
    }
    own::check(gradients, n_gradients, "gradients", "clip_gradients");
    own::check(outputs, n_gradients, "outputs", "clip_gradients");
    for (size_t i = 0; i < n_gradients; i++) {
        if (outputs[i].size != gradients[i].size || outputs[i].type != gradients[i].type) {
            throw std::runtime_error(
                "outputs[" + std::to_string(i) + "] must have the size and the type of its gradient in clip_gradients"
            );
        }
    }
    own::check_memory(to, outputs, gradients, n_gradients);
    const auto tables = own::tables_of(outputs, gradients, n_gradients);
    const hipStream_t stream = current_stream();
    own::Parts parts{};
    const double* const partial = own::sum_squares<true>(tables, parts, stream);
    if (tables.empty()) {
        own::norm_kernel<sum_t><<<1, own::THREADS, 0, stream>>>(to, partial, parts);
    }
    // the last tensors first (the caches hold those), the norm with the last launch
    for (size_t i = tables.size(); i-- > 0;) {
        const own::Table& table = tables[i];
        bool in_place = true;
        for (int32_t t = 0; t < table.count; t++) {
            in_place = in_place && table.to[t] == table.from[t];
        }
        own::scale_kernel<sum_t><<<own::workgroups_of(table), own::THREADS, 0, stream>>>(
            i == 0 ? to : nullptr, partial, parts, max_norm, in_place, table
        );
        MOPS_HIP_CHECK(hipGetLastError());
    }
    finish_call("clip_gradients");
}

#define MOPS_GRADIENT_NORM_INSTANTIATE(T)                                                          \
    template void gradient_norm<T>(Tensor<T, 1>, const Gradient*, size_t);                         \
    template void clip_gradients<T>(Tensor<T, 1>, const Gradient*, const Gradient*, size_t, double);
MOPS_GRADIENT_NORM_INSTANTIATE(float)
MOPS_GRADIENT_NORM_INSTANTIATE(double)

} // namespace mops::cuda
