// The first half of a gated feed-forward block, by group:
//
//   gate = A[r, :] W[g, :, :L],  up = A[r, :] W[g, :, L:]
//   output[r, :] = act(gate) up                          for the rows r of group g
//
// and its gradients, with c = grad_output[r, :]:
//
//   s[r, :] = (c up act'(gate), c act(gate))             (2 L numbers)
//   grad_A[r, :] = s[r, :] W[g, :, :]^T,   grad_W[g, :, :] = sum over the rows of A[r, :]^T s[r, :]
//
// Both projections are one product: a tile of grouped_tiles.hpp takes columns of
// W's two halves in turn, block by block, so that a lane ends with the gate and
// the up of the same numbers in registers. The activation and the product are
// its finish; the projections never reach memory. The gradients compute them
// again (nothing is kept from the forward call), make s of them in the same
// way, and hand s to the products that grouped_matrix_product's gradients are:
// s is the one intermediate in memory, 2 L numbers of T per row. Rounding it
// to T is what the matrix instructions take: an operand is T in any case, and
// the error of a number is that of an input of the operator.
#ifndef MOPS_AMD_GATED_PRODUCT_KERNELS_HPP
#define MOPS_AMD_GATED_PRODUCT_KERNELS_HPP

#include <type_traits>

#include "gated_product.hpp"
#include "grouped_launch.hpp"
#include "grouped_tiles.hpp"
#include "numbers.hpp"
#include "runtime.hpp"

namespace mops::amd::gated_product {

using namespace grouped_product;

// ------------------------------------------------------------ activations --
__device__ __forceinline__ float exponential(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }
__device__ __forceinline__ double exponential(double x) { return exp(x); }
__device__ __forceinline__ float inverse(float x) { return __builtin_amdgcn_rcpf(x); }
__device__ __forceinline__ double inverse(double x) { return 1 / x; }

/// 1 / (1 + e^-x) and what is left to 1. In 32 bits either is off by up to (16 + 2 |x|) 2^-24 of itself: the exponent x log2(e) is
/// rounded, as x has been in front of it (a sum of products; 80 is off by 4e-6, and so is e^-80). (e^-x infinite: 0 and 1; what
/// is below the smallest ordinary number, from -87.4 down, is 0)
template <typename Wide> struct Sigmoid {
    Wide value, rest;

    __device__ __forceinline__ explicit Sigmoid(Wide x) {
        const Wide power = exponential(-x);
        value = inverse(1 + power);
        rest = x < 0 ? 1 - value : power * value;
    }
};

/// The normal distribution's integral up to x and its density: with z = |x| / sqrt(2), half the complementary error function
/// of z is e^(-z^2) times a function that falls slowly from 1/2 to 0, which a polynomial in t = 1 / (1 + 0.35 z), times t,
/// gives to 1.0e-8 of itself (coefficients: least squares, weighted until the relative error is the same everywhere,
/// 0 <= z <= 14; 1 + erf has lost its digits where x is far below zero). The rounded exponent x^2 / 2 costs more than the
/// polynomial, up to (16 + 2 x^2) 2^-24 of the whole (5e-6 at -6, 1e-5 at -10). No branches: the error function of the mathematical
/// library took a third of a tile's time (20011 rows of 24 groups, 1280 x 2 x 1000, bfloat16, projections with their
/// gradients: 171 us, 153 like this).
template <typename Wide> struct Normal {
    Wide below, density;

    __device__ __forceinline__ explicit Normal(float x) {
        const float size = fabsf(x), t = inverse(1 + 0.35f * 0.707106781186547524f * size);
        const float power = exponential(-0.5f * x * x);
        float q = 0.04184640198945999f;
        q = fmaf(q, t, -0.17791077494621277f);
        q = fmaf(q, t, 0.22679196298122406f);
        q = fmaf(q, t, -0.08916350454092026f);
        q = fmaf(q, t, 0.1390409767627716f);
        q = fmaf(q, t, 0.11759191751480103f);
        q = fmaf(q, t, 0.1612173467874527f);
        q = fmaf(q, t, 0.18570789694786072f);
        q = fmaf(q, t, 0.19740821421146393f);
        q = fmaf(q, t, 0.1974695771932602f);
        const float beyond = 0.5f * power * t * q;
        below = x < 0 ? beyond : 1 - beyond;
        density = 0.398942280401432678f * power;
    }
    __device__ __forceinline__ explicit Normal(double x) {
        below = 0.5 * erfc(x * -0.70710678118654752440);
        density = 0.39894228040143267794 * exp(-0.5 * x * x);
    }
};

/// act(x) and act'(x) (that of a slope that nobody reads is not computed).
template <Activation WHICH, typename Wide> __device__ __forceinline__ void activate(Wide x, Wide& value, Wide& slope) {
    if constexpr (WHICH == Activation::GELU) {
        const Normal<Wide> normal(x);
        value = x * normal.below;
        slope = normal.below + x * normal.density;
    } else {
        const Sigmoid<Wide> s(x);
        value = WHICH == Activation::SIGMOID ? s.value : x * s.value;
        slope = WHICH == Activation::SIGMOID ? s.value * s.rest : s.value + x * (s.value * s.rest);
    }
}
template <Activation WHICH, typename Wide> __device__ __forceinline__ Wide activated(Wide x) {
    Wide value, slope;
    activate<WHICH>(x, value, slope);
    return value;
}
template <typename Body> __device__ __forceinline__ void with_activation(Activation which, Body&& body) { // (uniform)
    if (which == Activation::GELU) {
        body(std::integral_constant<Activation, Activation::GELU>{});
    } else if (which == Activation::SIGMOID) {
        body(std::integral_constant<Activation, Activation::SIGMOID>{});
    } else {
        body(std::integral_constant<Activation, Activation::SILU>{});
    }
}

// ---------------------------------------------------------------- finishes --
/// Shares of k: [split][row][2 n_size], the gates' sums in front.
template <int LDS_BYTES, typename T, int BM, int BN, int WM, int WN>
__device__ __forceinline__ void store_shares(const Product<T>& g, const TileOf<T, BM, BN, WM, WN>& t) {
    typedef wide_t<T> Wide;
#pragma unroll
    for (int half = 0; half < 2; half++) {
        turn_over<Wide, TileOf<T, BM, BN, WM, WN>::NB / 2, LDS_BYTES>(
            t, [&](int i, int j, int e) { return t.sums[i][2 * j + half][e]; },
            [&](int row, int column, const typename Packed<Wide>::Numbers& numbers) {
                const size_t of_split = static_cast<size_t>(t.split) * g.groups.n_rows;
                Wide* const to = row < t.unit.count
                                     ? g.partial + (of_split + t.rows[row]) * 2 * g.n_size + half * g.n_size
                                     : nullptr;
                store_piece<false, Wide>(to, t.n0 + column, g.n_size, numbers);
            }
        );
    }
}

/// output[r, n] = act(gate) up.
template <typename T> struct StoreGated {
    static constexpr bool PAIRS = true, RESTS = true;
    template <int BM, int BN> static constexpr bool ONCE = BM == 32; // (few rows per group)
    Activation activation;

    template <bool MAY_SPLIT, int LDS_BYTES, int BM, int BN, int WM, int WN>
    __device__ __forceinline__ void operator()(const Product<T>& g, const TileOf<T, BM, BN, WM, WN>& t) const {
        if constexpr (MAY_SPLIT) {
            if (g.splits > 1) { // (uniform)
                store_shares<LDS_BYTES>(g, t);
                return;
            }
        }
        with_activation(activation, [&](auto which) {
            turn_over<T, TileOf<T, BM, BN, WM, WN>::NB / 2, LDS_BYTES>(
                t,
                [&](int i, int j, int e) {
                    return activated<decltype(which)::value, wide_t<T>>(t.sums[i][2 * j][e]) * t.sums[i][2 * j + 1][e];
                },
                [&](int row, int column, const typename Packed<T>::Numbers& numbers) {
                    T* const to = row < t.unit.count ? g.out + static_cast<size_t>(t.rows[row]) * g.n_size : nullptr;
                    store_piece<true, T>(to, t.n0 + column, g.n_size, numbers);
                }
            );
        });
    }
};

/// s in rows of `stride` numbers, whole pieces: the gates' n_size, the ups', zeros.
template <typename T> struct Slopes {
    T* s;
    int32_t stride;
    const T* grad_output;
    Activation activation;

    /// `COUNT` numbers of T in memory at any address.
    template <int COUNT> struct Some {
        typedef T Anywhere __attribute__((ext_vector_type(COUNT), aligned(sizeof(T))));
    };
    /// grad_output's numbers n .. of row `row`, zeros behind its end.
    template <int COUNT>
    __device__ __forceinline__ typename Some<COUNT>::Anywhere cotangents(size_t row, int32_t n, int32_t n_size) const {
        typename Some<COUNT>::Anywhere numbers{};
        const T* const c = grad_output + row * n_size + n;
        if (n + COUNT <= n_size) {
            numbers = *reinterpret_cast<const typename Some<COUNT>::Anywhere*>(c);
        } else {
#pragma unroll
            for (int r = 0; r < COUNT; r++) {
                if (n + r < n_size) {
                    numbers[r] = c[r];
                }
            }
        }
        return numbers;
    }
    /// Numbers n .. of row `row` of s (those that exist), from their gates and ups.
    template <Activation WHICH, int COUNT>
    __device__ __forceinline__ void make(
        size_t row, int32_t n, int32_t n_size, const typename Some<COUNT>::Anywhere& c, const wide_t<T> (&gate)[COUNT],
        const wide_t<T> (&up)[COUNT]
    ) const {
        typedef typename Some<COUNT>::Anywhere Anywhere;
        T* const to = s + row * stride + n;
        Anywhere of_gate, of_up;
#pragma unroll
        for (int r = 0; r < COUNT; r++) {
            wide_t<T> value, slope;
            activate<WHICH>(gate[r], value, slope);
            const wide_t<T> cotangent = static_cast<wide_t<T>>(c[r]);
            of_gate[r] = static_cast<T>(cotangent * up[r] * slope);
            of_up[r] = static_cast<T>(cotangent * value);
        }
        if (n + COUNT <= n_size) {
            *reinterpret_cast<Anywhere*>(to) = of_gate;
            *reinterpret_cast<Anywhere*>(to + n_size) = of_up;
        } else {
#pragma unroll
            for (int r = 0; r < COUNT; r++) {
                if (n + r < n_size) {
                    to[r] = of_gate[r];
                    to[n_size + r] = of_up[r];
                }
            }
        }
        if (n + COUNT >= n_size) { // (the row's last numbers)
            for (int32_t at = 2 * n_size; at < stride; at++) {
                s[row * stride + at] = static_cast<T>(0.f);
            }
        }
    }
};

/// Through LDS as pairs of sums, so that grad_output is read and s written in whole pieces.
template <typename T> struct StoreSlopes : Slopes<T> {
    static constexpr bool PAIRS = true, RESTS = false;
    template <int BM, int BN> static constexpr bool ONCE = BM == 32;

    template <bool MAY_SPLIT, int LDS_BYTES, int BM, int BN, int WM, int WN>
    __device__ __forceinline__ void operator()(const Product<T>& g, const TileOf<T, BM, BN, WM, WN>& t) const {
        if constexpr (MAY_SPLIT) {
            if (g.splits > 1) { // (uniform)
                store_shares<LDS_BYTES>(g, t);
                return;
            }
        }
        typedef wide_t<T> Wide;
        typedef TileOf<T, BM, BN, WM, WN> Tile;
        typedef TurnedOver<T, Wide, Tile::NB> Turned;
        constexpr int BLOCK = Tile::BLOCK, COUNT = Packed<T>::COUNT, OF_PIECE = Turned::OF_PIECE;
        constexpr int OUT_PIECES = Tile::NB / 2 * BLOCK / COUNT, OF_BLOCK = BLOCK / COUNT; // of a wavefront's row of s
        static_assert(Turned::BYTES * WM * WN <= LDS_BYTES, "");
        const Turned turned{t.lds + t.wave * Turned::BYTES, t.lane};
        constexpr int TURNS = BLOCK * OUT_PIECES / WAVE; // pieces of a lane and block of rows
        auto row_of = [&](int i, int turn) { return t.wave_m + i * BLOCK + (turn * WAVE + t.lane) / OUT_PIECES; };
        auto piece_of = [&](int turn) { return (turn * WAVE + t.lane) % OUT_PIECES; };
        auto column_of = [&](int turn) { return t.n0 + (t.across() * OUT_PIECES + piece_of(turn)) * COUNT; };
        auto exists = [&](int i, int turn) { return row_of(i, turn) < t.unit.count && column_of(turn) < g.n_size; };
        // (all of grad_output is asked for in front of the first store, which it might overlap for all the compiler knows)
        typename Slopes<T>::template Some<COUNT>::Anywhere cotangents[Tile::MB][TURNS];
#pragma unroll
        for (int i = 0; i < Tile::MB; i++) {
#pragma unroll
            for (int turn = 0; turn < TURNS; turn++) {
                if (exists(i, turn)) {
                    cotangents[i][turn] =
                        this->template cotangents<COUNT>(t.rows[row_of(i, turn)], column_of(turn), g.n_size);
                }
            }
        }
        with_activation(this->activation, [&](auto which) {
#pragma unroll
            for (int i = 0; i < Tile::MB; i++) {
                turned.write([&](int j, int e) { return t.sums[i][j][e]; });
#pragma unroll
                for (int turn = 0; turn < TURNS; turn++) {
                    const int row = (turn * WAVE + t.lane) / OUT_PIECES, piece = piece_of(turn);
                    // (block 2 j has the gates of the wavefront's columns j BLOCK .., block 2 j + 1 the ups)
                    const int first = (piece / OF_BLOCK * 2 * BLOCK + piece % OF_BLOCK * COUNT) / OF_PIECE;
                    Wide gate[COUNT], up[COUNT];
#pragma unroll
                    for (int p = 0; p < COUNT / OF_PIECE; p++) {
                        const auto gates = turned.read(row, first + p), ups = turned.read(row, first + BLOCK / OF_PIECE + p);
#pragma unroll
                        for (int r = 0; r < OF_PIECE; r++) {
                            gate[p * OF_PIECE + r] = gates[r];
                            up[p * OF_PIECE + r] = ups[r];
                        }
                    }
                    if (exists(i, turn)) {
                        this->template make<decltype(which)::value, COUNT>(
                            t.rows[row_of(i, turn)], column_of(turn), g.n_size, cotangents[i][turn], gate, up
                        );
                    }
                }
                Turned::settle();
            }
        });
    }
};

/// The sum of the shares of k, finished: a thread per number. What is in no group was not shared (Slopes), and nobody reads
/// what is made of it.
template <typename T, typename Finish>
__global__ __launch_bounds__(JOIN_THREADS) void join_shares_kernel(Product<T> g, Finish finish) {
    typedef wide_t<T> Wide;
    const size_t i = blockIdx.x * static_cast<size_t>(JOIN_THREADS) + threadIdx.x;
    const size_t rows = g.groups.n_rows;
    if (i >= rows * g.n_size) {
        return;
    }
    const size_t row = i / g.n_size;
    const int32_t n = static_cast<int32_t>(i % g.n_size);
    const Wide* from = g.partial + row * 2 * g.n_size + n;
    Wide gate[1] = {0}, up[1] = {0};
#pragma unroll 4
    for (int32_t s = 0; s < g.splits; s++, from += rows * 2 * g.n_size) {
        gate[0] += from[0];
        up[0] += from[g.n_size];
    }
    with_activation(finish.activation, [&](auto which) {
        if constexpr (std::is_same_v<Finish, StoreGated<T>>) {
            g.out[i] = static_cast<T>(activated<decltype(which)::value, Wide>(gate[0]) * up[0]);
        } else {
            finish.template make<decltype(which)::value, 1>(
                row, n, g.n_size, finish.template cotangents<1>(row, n, g.n_size), gate, up
            );
        }
    });
}

// -------------------------------------------------------------------- host --
/// Columns of the result in a tile: half of those of W (WIDE_COLUMNS for the tiles of few rows).
inline int columns_of(int tile) { return std::max(tile, WIDE_COLUMNS) / 2; }

/// The projections and their finish.
template <typename T> class Projections {
public:
    explicit Projections(const Inputs<T>& inputs)
        : A_{inputs.A, static_cast<size_t>(inputs.groups.n_rows), inputs.k_size},
          W_{inputs.W, static_cast<size_t>(inputs.groups.n_groups) * inputs.k_size * 2, inputs.columns} {
        g_.groups = inputs.groups;
        g_.n_size = inputs.columns;
        g_.k_size = inputs.k_size;
        choose(worth_copying(A_, W_, 4.0 * A_.n_rows * g_.k_size * g_.n_size));
    }
    size_t bytes() const { return copies_ + 2 * split_bytes(g_); }
    bool copies() const { return copies_ > 0; }
    void do_without_copies() { choose(false); }

    /// `out`: of StoreGated.
    template <typename Finish> void run(T* out, const Finish& finish, char* workspace, hipStream_t stream) const {
        Product<T> g = g_;
        g.out = out;
        g.partial = reinterpret_cast<wide_t<T>*>(workspace + copies_);
        char* room = copies_ > 0 ? workspace : nullptr;
        g.q = place(A_, room, stream);
        g.p = place(W_, room, stream);
        if (tile_ <= 64 && g.in_place) {
            launch_wide<T, Form::FORWARD>(g, tile_, columns_of(tile_), stream, finish);
        } else {
            const unsigned workgroups = set_tiles<Form::FORWARD>(g, tile_, columns_of(tile_));
            with_tile<T>(tile_, g.in_place, [&](auto size, auto m, auto n, auto in_place) {
                constexpr int BM = decltype(size)::value, BN = BM == 64 ? WIDE_COLUMNS : BM;
                constexpr int WM = decltype(m)::value, WN = decltype(n)::value;
                constexpr bool ALIGNED = decltype(in_place)::value;
                if constexpr (BM > 64 || !ALIGNED) { // (the others are wide ones)
                    tiles_kernel<T, Form::FORWARD, BM, BN, WM, WN, DEEP, STAGES_OF<BM, ALIGNED>, ALIGNED, Finish>
                        <<<workgroups, WM * WN * WAVE, 0, stream>>>(g, finish);
                }
            });
            MOPS_HIP_CHECK(hipGetLastError());
        }
        if (g.splits > 1) {
            const size_t blocks = ceil_div(static_cast<size_t>(g.groups.n_rows) * g.n_size, JOIN_THREADS);
            join_shares_kernel<T, Finish><<<static_cast<unsigned>(blocks), JOIN_THREADS, 0, stream>>>(g, finish);
            MOPS_HIP_CHECK(hipGetLastError());
        }
    }

private:
    void choose(bool copied) {
        copies_ = copied ? A_.copied_bytes() + W_.copied_bytes() : 0;
        g_.in_place = copied || (A_.in_place() && W_.in_place());
        // (as tile_of_rows)
        const size_t rows = A_.n_rows, groups = static_cast<size_t>(g_.groups.n_groups);
        auto fits = [&](int tile) {
            return exists<T>(tile, g_.in_place) && rows >= tile / 2 * groups && filled(tile, 2 * g_.n_size) &&
                   ceil_div(rows, tile) * tiles(g_.n_size, columns_of(tile)) >= static_cast<size_t>(compute_units());
        };
        tile_ = fits(256) ? 256 : fits(128) ? 128 : 64;
        share_k(g_, tile_);
        if (tile_ == 64 && g_.in_place && rows <= 16 * groups) {
            tile_ = LEAST_ROWS<T>;
        }
    }

    const Matrices<T> A_, W_;
    Product<T> g_{};
    int tile_ = 64;
    size_t copies_ = 0;
};

template <typename T> void forward(const Inputs<T>& inputs, T* output, hipStream_t stream) {
    Projections<T> projections(inputs);
    char* workspace = projections.copies() ? static_cast<char*>(scratch_or_null(projections.bytes())) : nullptr;
    if (workspace == nullptr) {
        projections.do_without_copies();
        workspace = projections.bytes() > 0 ? static_cast<char*>(scratch(projections.bytes())) : nullptr;
    }
    projections.run(output, StoreGated<T>{inputs.activation}, workspace, stream);
}

template <typename T>
void gradients(const Inputs<T>& inputs, const T* grad_output, T* grad_A, T* grad_W, hipStream_t stream) {
    const size_t rows = inputs.groups.n_rows;
    const int32_t width = 2 * inputs.columns;
    const int32_t stride = static_cast<int32_t>(ceil_div(static_cast<size_t>(width), PIECE<T>)) * PIECE<T>;
    const size_t slope_bytes = align256(rows * stride * sizeof(T));
    Projections<T> projections(inputs);
    Product<T> sums{}, of_rows{};
    sums.out = grad_W;
    sums.groups = inputs.groups;
    sums.m_size = inputs.k_size;
    sums.n_size = width;
    of_rows.out = grad_A;
    of_rows.groups = inputs.groups;
    of_rows.n_size = inputs.k_size;
    of_rows.k_size = width;
    // (where s lies depends on nothing but its size)
    auto products_of = [&](T* s) {
        return Gradients<T>(
            sums, of_rows, Matrices<T>{s, rows, width, stride}, Matrices<T>{inputs.A, rows, inputs.k_size},
            Matrices<T>{inputs.W, static_cast<size_t>(inputs.groups.n_groups) * inputs.k_size, width}
        );
    };
    Gradients<T> products = products_of(nullptr);
    auto bytes = [&] { return slope_bytes + std::max(projections.bytes(), products.bytes()); };
    char* workspace =
        projections.copies() || products.copies() ? static_cast<char*>(scratch_or_null(bytes())) : nullptr;
    const bool copied = workspace != nullptr;
    if (!copied) {
        projections.do_without_copies();
        products.do_without_copies();
        workspace = static_cast<char*>(scratch(bytes()));
    }
    T* const s = reinterpret_cast<T*>(workspace);
    projections.run(
        static_cast<T*>(nullptr), StoreSlopes<T>{{s, stride, grad_output, inputs.activation}}, workspace + slope_bytes,
        stream
    );
    products = products_of(s);
    if (!copied) {
        products.do_without_copies();
    }
    products.run(workspace + slope_bytes, stream);
}

} // namespace mops::amd::gated_product

#endif
