// A linear layer to many classes and the cross entropy of its softmax:
//
//   x[r, v] = A[r, :] . W[v, :],   s[r] = log(sum over v of exp(x[r, v]))
//   losses[r] = s[r] - x[r, targets[r]]
//
// and its gradients, from g = grad_losses[r] and h = grad_log_sums[r]:
//
//   d[r, v] = (g + h) exp(x[r, v] - s[r]) - (v = targets[r] ? g : 0)
//   grad_A[r, :] = sum over v of d[r, v] W[v, :],   grad_W[v, :] = sum over r of d[r, v] A[r, :]
//
// The logits x never reach memory. A tile of grouped_tiles.hpp ends with a
// row's logits in registers, and its finish makes of them the row's largest one
// and the sum of the powers below it (two numbers per row and tile, joined
// afterwards, a piece of the classes at a time where those of all would take too
// much memory), or the numbers d, rounded to T (what the matrix instructions
// take; 16-bit types scaled, and in two parts for few rows: SCALED, IN_TWO_PARTS). Of d, a piece of the classes is in
// memory at a time, and both products with it follow while the caches hold what
// they can of it; grad_A is summed up over the pieces in 32 bits.
//
// Rows without a target in range are in no group (rows_with_targets): they cost
// nothing, and whatever they hold reaches nothing.
#ifndef MOPS_AMD_CROSS_ENTROPY_KERNELS_HPP
#define MOPS_AMD_CROSS_ENTROPY_KERNELS_HPP

#include <limits>
#include <numeric>
#include <tuple>
#include <type_traits>

#include "cross_entropy.hpp"
#include "grouped_launch.hpp"
#include "grouped_tiles.hpp"
#include "numbers.hpp"
#include "runtime.hpp"

namespace mops::amd::cross_entropy {

using namespace grouped_product;

/// Powers and logarithms of two: a logit enters an exponent as (x - what it is relative to) log2(e). The difference comes
/// first: it is exact where the two are close, so that the power of a class that is all but certain is off by its own rounding
/// and not by that of a product as large as the logit (x log2(e) - base, one instruction instead of two, is off by 6e-8 |x|,
/// 4e-6 at 60, and so was the loss of such a row, and p - 1; the losses of 4001 rows of 32003 classes, K = 1000, float16, take
/// 261 us like this, 258 like that).
constexpr double LOG2_E = 1.44269504088896340736, LN_2 = 0.69314718055994530942;
__device__ __forceinline__ float power(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ double power(double x) { return exp2(x); }
__device__ __forceinline__ float logarithm(float x) { return log2f(x); }
__device__ __forceinline__ double logarithm(double x) { return log2(x); }
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double larger(double a, double b) { return fmax(a, b); }
/// e^(x - base)
template <typename Wide> __device__ __forceinline__ Wide power_of(Wide x, Wide base) {
    return power((x - base) * static_cast<Wide>(LOG2_E));
}

/// The largest of some logits, and the sum of the powers relative to it. (Not-a-number is never the largest;
/// it makes the sum one.)
template <typename Wide> struct Sum {
    Wide most, sum;

    static __device__ __forceinline__ Wide lowest() { return -std::numeric_limits<Wide>::infinity(); }
    /// What the powers are taken relative to: no difference of infinities where there is nothing.
    static __device__ __forceinline__ Wide base(Wide most) { return most == lowest() ? Wide(0) : most; }
    /// Of a single logit.
    static __device__ __forceinline__ Sum of(Wide x) {
        const Wide most = x == x ? x : lowest();
        return Sum{most, x == x ? power_of(x, base(most)) : x};
    }
    __device__ __forceinline__ void join(const Sum& other) {
        const Wide both = larger(most, other.most), from = base(both);
        sum = sum * power_of(most, from) + other.sum * power_of(other.most, from);
        most = both;
    }
    /// log(sum of the powers of e), less x.
    __device__ __forceinline__ Wide logarithm_above(Wide x) const {
        return most - x + static_cast<Wide>(LN_2) * logarithm(sum);
    }
};

// ----------------------------------------------------------- sums by tiles --
/// partial[tile of classes][place]; target_logits[row], where the tile has the row's target. The classes are those from
/// `first_class` on.
template <typename T> struct StorePartialSums {
    typedef wide_t<T> Wide;
    static constexpr bool PAIRS = false, RESTS = false;
    template <int BM, int BN> static constexpr bool ONCE = BM != BN; // (wide tiles: launch_logits)
    Sum<Wide>* partial;
    Wide* target_logits;
    const int32_t* targets;
    int32_t first_class;

    template <bool MAY_SPLIT, int LDS_BYTES, int BM, int BN, int WM, int WN>
    __device__ __forceinline__ void operator()(const Product<T>& g, const TileOf<T, BM, BN, WM, WN>& t) const {
        typedef TileOf<T, BM, BN, WM, WN> Tile;
        if constexpr (MAY_SPLIT) {
            if (g.splits > 1) { // (uniform)
                StoreSums<T, Form::GRAD_ROWS>{}.template operator()<MAY_SPLIT, LDS_BYTES>(g, t);
                return;
            }
        }
        static_assert(WN * BM * sizeof(Sum<Wide>) <= LDS_BYTES, "");
        Sum<Wide>* const shared = reinterpret_cast<Sum<Wide>*>(t.lds);
        constexpr int COLUMNS = Tile::NB * Tile::BLOCK;
        const int32_t first = t.n0 + t.across() * COLUMNS; // class of the wavefront's first column
        if (t.n0 + BN > g.n_size) { // (uniform) nothing where there is no class
            t.for_each([&](int i, int j, int e) {
                if (first + j * Tile::BLOCK + t.column(e) >= g.n_size) {
                    t.sums[i][j][e] = Sum<Wide>::lowest();
                }
            });
        }
#pragma unroll
        for (int i = 0; i < Tile::MB; i++) {
            const int32_t row = t.rows[min(t.row(i), t.unit.count - 1)];
            // (any target: the difference wraps around, but never to one of the columns)
            const int32_t target = static_cast<int32_t>(static_cast<uint32_t>(targets[row]) - (first_class + first));
            // (few wavefronts have a target of their rows among their columns; one lane of all tiles has its logit)
            if (__any(target >= 0 && target < COLUMNS)) {
#pragma unroll
                for (int j = 0; j < Tile::NB; j++) {
#pragma unroll
                    for (int e = 0; e < Tile::HELD; e++) {
                        if (j * Tile::BLOCK + t.column(e) == target && t.row(i) < t.unit.count) {
                            target_logits[row] = t.sums[i][j][e];
                        }
                    }
                }
            }
            Wide most = Sum<Wide>::lowest();
#pragma unroll
            for (int j = 0; j < Tile::NB; j++) {
#pragma unroll
                for (int e = 0; e < Tile::HELD; e++) {
                    most = larger(most, t.sums[i][j][e]);
                }
            }
#pragma unroll
            for (int s = Tile::BLOCK; s < WAVE; s *= 2) {
                most = larger(most, __shfl_xor(most, s));
            }
            const Wide base = Sum<Wide>::base(most);
            Wide sum[2] = {0, 0};
#pragma unroll
            for (int j = 0; j < Tile::NB; j++) {
#pragma unroll
                for (int e = 0; e < Tile::HELD; e++) {
                    sum[e % 2] += power_of(t.sums[i][j][e], base);
                }
            }
            sum[0] += sum[1];
#pragma unroll
            for (int s = Tile::BLOCK; s < WAVE; s *= 2) {
                sum[0] += __shfl_xor(sum[0], s);
            }
            if (t.lane < Tile::BLOCK) {
                shared[t.across() * BM + t.row(i)] = Sum<Wide>{most, sum[0]};
            }
        }
        __syncthreads();
        for (int m = threadIdx.x; m < t.unit.count; m += Tile::THREADS) {
            Sum<Wide> all = shared[m];
#pragma unroll
            for (int w = 1; w < WN; w++) {
                all.join(shared[w * BM + m]);
            }
            partial[static_cast<size_t>(t.n0 / BN) * g.groups.n_rows + t.unit.begin + m] = all;
        }
    }
};

/// losses and log_sums of ROWS places per workgroup, as many threads each as there are for them, from the sums of `parts`
/// tiles; zeros for the rows without a target. running[place]: the sums of the pieces of classes in front (not in the first
/// one) and up to this one (not in the last).
constexpr int JOIN_SUM_THREADS = 256;
template <typename T, int ROWS>
__global__ __launch_bounds__(JOIN_SUM_THREADS) void join_sums_kernel(
    wide_t<T>* __restrict__ losses, wide_t<T>* __restrict__ log_sums, const Sum<wide_t<T>>* __restrict__ partial,
    Sum<wide_t<T>>* __restrict__ running, const wide_t<T>* __restrict__ target_logits, const int32_t* __restrict__ targets,
    RowGroups groups, int32_t parts, int32_t classes, bool first, bool last
) {
    typedef wide_t<T> Wide;
    constexpr int LANES = JOIN_SUM_THREADS / ROWS;
    __shared__ Sum<Wide> shared[LANES][ROWS];
    const int in_block = threadIdx.x % ROWS, lane = threadIdx.x / ROWS;
    const int32_t place = blockIdx.x * ROWS + in_block, kept = groups.end_of(0, groups.begin_of(0));
    Sum<Wide> all{Sum<Wide>::lowest(), 0};
    if (place < kept) {
        if (!first && lane == 0) {
            all = running[place];
        }
#pragma unroll 4
        for (int32_t p = lane; p < parts; p += LANES) {
            all.join(partial[static_cast<size_t>(p) * groups.n_rows + place]);
        }
    }
    shared[lane][in_block] = all;
#pragma unroll
    for (int half = LANES / 2; half > 0; half /= 2) {
        __syncthreads();
        if (lane < half) {
            all.join(shared[lane + half][in_block]);
            shared[lane][in_block] = all;
        }
    }
    if (!last) { // (uniform)
        if (lane == 0 && place < kept) {
            running[place] = all;
        }
    } else if (lane == 0 && place < groups.n_rows) {
        const int32_t row = groups.row_at(place);
        const bool has_target = place < kept && in_bounds(targets[row], classes);
        losses[row] = has_target ? all.logarithm_above(target_logits[row]) : Wide(0);
        log_sums[row] = has_target ? all.logarithm_above(0) : Wide(0);
    }
}

/// The same where k is shared (few rows, few classes): a workgroup per place adds up its logits, [split][row][class].
constexpr int ROW_THREADS = 256;
template <typename T>
__global__ __launch_bounds__(ROW_THREADS) void join_shared_sums_kernel(
    wide_t<T>* __restrict__ losses, wide_t<T>* __restrict__ log_sums, const int32_t* __restrict__ targets, Product<T> g
) {
    typedef wide_t<T> Wide;
    __shared__ Sum<Wide> shared[ROW_THREADS / WAVE];
    __shared__ Wide target_logit;
    const int32_t place = blockIdx.x, kept = g.groups.end_of(0, g.groups.begin_of(0)), row = g.groups.row_at(place);
    if (place >= kept || !in_bounds(targets[row], g.n_size)) { // (uniform)
        if (threadIdx.x == 0) {
            losses[row] = 0;
            log_sums[row] = 0;
        }
        return;
    }
    const size_t size = static_cast<size_t>(g.groups.n_rows) * g.n_size;
    Sum<Wide> all{Sum<Wide>::lowest(), 0};
    for (int32_t v = threadIdx.x; v < g.n_size; v += ROW_THREADS) {
        Wide x = 0;
#pragma unroll 4
        for (int32_t s = 0; s < g.splits; s++) {
            x += g.partial[s * size + static_cast<size_t>(row) * g.n_size + v];
        }
        if (v == targets[row]) {
            target_logit = x;
        }
        all.join(Sum<Wide>::of(x));
    }
#pragma unroll
    for (int s = 1; s < WAVE; s *= 2) {
        all.join(Sum<Wide>{__shfl_xor(all.most, s), __shfl_xor(all.sum, s)});
    }
    if (threadIdx.x % WAVE == 0) {
        shared[threadIdx.x / WAVE] = all;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < ROW_THREADS / WAVE; w++) {
            all.join(shared[w]);
        }
        losses[row] = all.logarithm_above(target_logit);
        log_sums[row] = all.logarithm_above(0);
    }
}

// ---------------------------------------------------------------- gradients --
/// 16-bit types: d is stored relative to the weight of the first row with a target (its digits: a number in [1, 2)), and the
/// sums are multiplied by it again, in 32 bits. The largest numbers of d are a weight times something just below one, and
/// in the loss of a mean all weights are the same: rounded as they are, they would all be off by the same part, up to 2^-9
/// of the gradients in bfloat16, and those would be off by it however many rows they sum up. 16-bit floats have five bits of
/// exponent as well, and d, most of whose numbers are a probability times a weight (of a mean: one in the number of rows),
/// would lose most of its bits: a power of two brings the largest weight of the call to 2^13 .. 2^14 (twice that is the
/// most d can be: below 65504). The other types need neither.
template <typename T> constexpr bool SCALED = sizeof(T) == 2;
/// Up to so many rows the 16-bit types have d in two parts, what it is rounded to and what that leaves (as rows of their own,
/// behind the others): a gradient of few rows consists of few numbers d, each times many numbers, and whether their errors
/// are above or below the average is chance (3 rows of 38982 classes, K = 1127, bfloat16: errors of 2.8e-3 of the result,
/// 1.7e-3 in two parts, which is what the result's own rounding makes). Rows cost little where the classes have to be
/// read and their gradients written anyway: 256 rows of 50000 classes, K = 2048, are 505 us (257 in one part
/// 437), of 38982, K = 1127, 351 (301), of 32000, K = 512, 118 (113). 512 rows would be 928 (776), 632 (424) and 204 (161).
/// The error, against a single rounding of the results, is 1.00 in two parts and 1.3 to 1.5 in one, at 257 rows as at 1024 (50000 x
/// 2048, 13112 x 50, 94 x 128, 4000 x 512, bfloat16 and float16; up to 1.6 where a few frequent classes have most of the
/// rows): the border is where the second part begins to cost, the error is the same behind it.
constexpr int32_t IN_TWO_PARTS = 256;
/// Up to so many rows of d, grad_A takes as long as the classes take to be read, and two shares of them per compute unit have
/// more on their way than one (rows of 50000 classes, K = 2048, bfloat16, one / two / three, us, all of the gradients: 3
/// rows 249 / 214 / 209, 64 rows 307 / 288 / 261, 256 rows 592 / 510 / 527; of 32000, K = 512: 62 / 58 / 61, 73 / 75 / 75,
/// 131 / 121 / 127; of 20000, K = 1127, float: 204 / 166 / 164, 500 rows 879 / 783 / 732).
constexpr int32_t FEW_ROWS_OF_D = 512;
template <typename T> struct Unscale {
    float* scale; // and its inverse (SCALED; null: one)

    __device__ __forceinline__ wide_t<T> factor() const {
        if constexpr (SCALED<T>) {
            return scale != nullptr ? scale[0] : 1;
        }
        return 1;
    }
    __device__ __forceinline__ wide_t<T> operator()(wide_t<T> sum) const {
        if constexpr (SCALED<T>) {
            return scale != nullptr ? sum * scale[1] : sum;
        }
        return sum;
    }
};

/// How d is made of logits.
template <typename T> struct Weights {
    typedef wide_t<T> Wide;
    const Wide *grad_losses, *grad_log_sums, *log_sums;
    const int32_t* targets;
    int32_t first; // class of the piece's first column
    Unscale<T> scale;

    struct OfRow {
        Wide base, of_power, of_target; // base: of the powers, log_sums
        int32_t target;

        __device__ __forceinline__ Wide at_others(Wide x) const { return of_power * power_of(x, base); }
        __device__ __forceinline__ Wide make(Wide x, int32_t n) const {
            return at_others(x) - (n == target ? of_target : Wide(0));
        }
    };
    __device__ __forceinline__ OfRow of_row(int32_t row) const {
        const Wide g = grad_losses != nullptr ? grad_losses[row] : Wide(0);
        const Wide h = grad_log_sums != nullptr ? grad_log_sums[row] : Wide(0);
        return OfRow{log_sums[row], (g + h) * scale.factor(), g * scale.factor(), targets[row] - first};
    }
};

/// What the rounding to T leaves (nothing of what is infinite).
template <typename T> __device__ __forceinline__ wide_t<T> rest_of(wide_t<T> x) {
    const wide_t<T> rest = x - static_cast<wide_t<T>>(static_cast<T>(x));
    return rest == rest ? rest : wide_t<T>(0);
}

/// d[row, 0 .. stride - 1], whole pieces with zeros behind n_size; what the rounding leaves of it in rows of their own.
template <typename T> struct StoreGradients : Weights<T> {
    typedef wide_t<T> Wide;
    static constexpr bool PAIRS = false, RESTS = false;
    template <int BM, int BN> static constexpr bool ONCE = BM != BN; // (wide tiles: launch_logits)
    T* d;
    int32_t stride;
    size_t rest_at; // numbers from a row to the row of what is left of it (0: nowhere)

    template <bool MAY_SPLIT, int LDS_BYTES, int BM, int BN, int WM, int WN>
    __device__ __forceinline__ void operator()(const Product<T>& g, const TileOf<T, BM, BN, WM, WN>& t) const {
        typedef TileOf<T, BM, BN, WM, WN> Tile;
        if constexpr (MAY_SPLIT) {
            if (g.splits > 1) { // (uniform)
                StoreSums<T, Form::GRAD_ROWS>{}.template operator()<MAY_SPLIT, LDS_BYTES>(g, t);
                return;
            }
        }
        constexpr int COLUMNS = Tile::NB * Tile::BLOCK;
        const int32_t first = t.n0 + t.across() * COLUMNS;
#pragma unroll
        for (int i = 0; i < Tile::MB; i++) {
            const auto of = this->of_row(t.rows[min(t.row(i), t.unit.count - 1)]);
#pragma unroll
            for (int j = 0; j < Tile::NB; j++) {
#pragma unroll
                for (int e = 0; e < Tile::HELD; e++) {
                    t.sums[i][j][e] = of.at_others(t.sums[i][j][e]);
                }
            }
            // (few wavefronts have a target of their rows among their columns)
            if (__any(of.target >= first && of.target < first + COLUMNS)) {
#pragma unroll
                for (int j = 0; j < Tile::NB; j++) {
#pragma unroll
                    for (int e = 0; e < Tile::HELD; e++) {
                        t.sums[i][j][e] -= first + j * Tile::BLOCK + t.column(e) == of.target ? of.of_target : Wide(0);
                    }
                }
            }
        }
        if (t.n0 + BN > g.n_size) { // (uniform) zeros where there is no class
            t.for_each([&](int i, int j, int e) {
                if (first + j * Tile::BLOCK + t.column(e) >= g.n_size) {
                    t.sums[i][j][e] = 0;
                }
            });
        }
        auto store = [&](T* rows) {
            turn_over<T, Tile::NB, LDS_BYTES>(
                t, [&](int i, int j, int e) { return t.sums[i][j][e]; },
                [&](int row, int column, const typename Packed<T>::Numbers& numbers) {
                    T* const to = row < t.unit.count ? rows + static_cast<size_t>(t.rows[row]) * stride : nullptr;
                    store_piece<false, T>(to, t.n0 + column, stride, numbers);
                }
            );
        };
        store(d);
        if (sizeof(T) == 2 && rest_at > 0) { // (uniform)
            t.for_each([&](int i, int j, int e) { t.sums[i][j][e] = rest_of<T>(t.sums[i][j][e]); });
            store(d + rest_at);
        }
    }
};

/// The same from shares of k, [split][row][n_size]: a thread per number. (What rows without a target get, nobody reads.)
template <typename T>
__global__ __launch_bounds__(JOIN_THREADS) void join_shared_gradients_kernel(Product<T> g, StoreGradients<T> finish) {
    const size_t size = static_cast<size_t>(g.groups.n_rows) * g.n_size;
    const size_t i = blockIdx.x * static_cast<size_t>(JOIN_THREADS) + threadIdx.x;
    const size_t row = i / finish.stride;
    const int32_t n = static_cast<int32_t>(i % finish.stride);
    if (row >= static_cast<size_t>(g.groups.n_rows)) {
        return;
    }
    wide_t<T> x = 0;
    if (n < g.n_size) {
#pragma unroll 4
        for (int32_t s = 0; s < g.splits; s++) {
            x += g.partial[s * size + row * g.n_size + n];
        }
        x = finish.of_row(static_cast<int32_t>(row)).make(x, n);
    }
    finish.d[i] = static_cast<T>(x);
    if (sizeof(T) == 2 && finish.rest_at > 0) {
        finish.d[finish.rest_at + i] = static_cast<T>(rest_of<T>(x));
    }
}

/// The plans of few rows, of d in two parts and the scale of it, in one launch (50 rows of 63 classes, K = 4, float16,
/// losses and gradients: 31.8 us; 37.1 in launches of their own). Rows n_rows .. 2 n_rows - 1 of A are rows
/// 0 .. n_rows - 1 again, in whole pieces with zeros behind them; the places are those of the rows with a target, of what
/// is left of them, and of the others.
constexpr int TWICE_THREADS = IN_TWO_PARTS; // (a row each in the first workgroup)
struct PlanOfTwice {
    int32_t *order, *offsets;             // of the rows: as rows_with_targets
    int32_t *twice_order, *twice_offsets; // of the rows of d
    float* scale;                         // (null: none)
};
template <typename T>
__global__ __launch_bounds__(TWICE_THREADS) void twice_kernel(
    T* __restrict__ to, Operand<T> from, int32_t width, int32_t pieces, PlanOfTwice plan, const int32_t* __restrict__ targets,
    const float* __restrict__ grad_losses, const float* __restrict__ grad_log_sums, int32_t rows, int32_t classes
) {
    constexpr int32_t COUNT = Matrix<T>::COUNT;
    const uint32_t i = blockIdx.x * TWICE_THREADS + threadIdx.x; // (of up to IN_TWO_PARTS rows: below 2^31)
    if (i < static_cast<uint32_t>(rows) * pieces) {
        const size_t row = i / pieces, piece = i % pieces;
        const int32_t first = static_cast<int32_t>(piece) * COUNT;
        const T* const at = from.data + row * from.stride + first;
        const Numbers<T> numbers =
            first + COUNT <= width ? load_numbers<T>(at) : load_some_numbers<T>(at, width - first);
        *reinterpret_cast<Numbers<T>*>(to + (row * pieces + piece) * COUNT) = numbers;
        *reinterpret_cast<Numbers<T>*>(to + ((row + rows) * pieces + piece) * COUNT) = numbers;
    }
    if (blockIdx.x > 0) { // (uniform)
        return;
    }
    constexpr int WAVES = TWICE_THREADS / WAVE;
    __shared__ int32_t counts[WAVES];
    __shared__ float largest[WAVES];
    const int32_t row = threadIdx.x;
    const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
    const bool kept = row < rows && in_bounds(targets[row], classes);
    const float g = kept && grad_losses != nullptr ? grad_losses[row] : 0;
    const float h = kept && grad_log_sums != nullptr ? grad_log_sums[row] : 0;
    float most = weight_of(g, h);
#pragma unroll
    for (int s = 1; s < WAVE; s *= 2) {
        most = fmaxf(most, __shfl_xor(most, s));
    }
    const uint64_t of_lanes = __ballot(kept);
    if (lane == 0) {
        counts[wave] = __popcll(of_lanes);
        largest[wave] = most;
    }
    __syncthreads();
    int32_t before = __popcll(of_lanes & ((uint64_t(1) << lane) - 1)), all = 0; // of the kept rows
#pragma unroll
    for (int w = 0; w < WAVES; w++) {
        before += w < wave ? counts[w] : 0;
        all += counts[w];
        most = fmaxf(most, largest[w]);
    }
    if (row < rows) {
        const int32_t at = kept ? before : 2 * all + row - before;
        plan.order[kept ? before : all + row - before] = row;
        plan.twice_order[at] = row;
        plan.twice_order[at + (kept ? all : rows - all)] = row + rows;
    }
    if (threadIdx.x == 0) {
        plan.offsets[0] = plan.twice_offsets[0] = 0;
        plan.offsets[1] = all;
        plan.twice_offsets[1] = 2 * all;
    }
    if (plan.scale != nullptr && (kept ? before == 0 : all == 0 && threadIdx.x == 0)) {
        set_scale(plan.scale, g, h, most);
    }
}

/// grad_A, summed up over the pieces of the classes in `sums` [row][n_size] (only where there are several), or as partial
/// results where d is in two parts.
template <typename T> struct AddRows {
    typedef wide_t<T> Wide;
    static constexpr bool PAIRS = false, RESTS = true;
    template <int BM, int BN> static constexpr bool ONCE = false;
    Wide* sums;
    bool first, last, twice;
    Unscale<T> scale;

    template <bool MAY_SPLIT, int LDS_BYTES, int BM, int BN, int WM, int WN>
    __device__ __forceinline__ void operator()(const Product<T>& g, const TileOf<T, BM, BN, WM, WN>& t) const {
        typedef TileOf<T, BM, BN, WM, WN> Tile;
        const bool alone = first && last;
        const bool rest = t.unit.group == g.groups.n_groups;
        if ((MAY_SPLIT && g.splits > 1) || (alone && !twice)) { // (uniform)
            StoreSums<T, Form::FORWARD, Unscale<T>>{scale}.template operator()<MAY_SPLIT, LDS_BYTES>(g, t);
            return;
        }
        if constexpr (sizeof(T) == 2) {
            if (twice) { // (uniform)
                turn_over<Wide, Tile::NB, LDS_BYTES>(
                    t, [&](int i, int j, int e) { return scale(t.sums[i][j][e]); },
                    [&](int row, int column, const typename Packed<Wide>::Numbers& numbers) {
                        Wide* const to =
                            row < t.unit.count ? g.partial + static_cast<size_t>(t.rows[row]) * g.n_size : nullptr;
                        store_piece<false, Wide>(to, t.n0 + column, g.n_size, numbers);
                    }
                );
                return;
            }
        }
        if (rest && !last) { // (uniform)
            return;
        }
        typedef typename Packed<Wide>::Anywhere Anywhere;
        constexpr int COUNT = Packed<Wide>::COUNT;
        typedef T Narrow __attribute__((ext_vector_type(COUNT), aligned(sizeof(T))));
        turn_over<Wide, Tile::NB, LDS_BYTES>(
            t, [&](int i, int j, int e) { return scale(t.sums[i][j][e]); },
            [&](int row, int column, const typename Packed<Wide>::Numbers& numbers) {
                const int32_t n = t.n0 + column;
                if (row >= t.unit.count || n >= g.n_size) {
                    return;
                }
                const size_t at = static_cast<size_t>(t.rows[row]) * g.n_size + n;
                Anywhere total{};
                const bool before = !first && !rest;
                if (n + COUNT <= g.n_size) {
                    if (before) {
                        total = *reinterpret_cast<const Anywhere*>(sums + at);
                    }
                    Narrow narrow;
#pragma unroll
                    for (int r = 0; r < COUNT; r++) {
                        total[r] += numbers[r];
                        narrow[r] = static_cast<T>(total[r]);
                    }
                    if (last) {
                        *reinterpret_cast<Narrow*>(g.out + at) = narrow;
                    } else {
                        *reinterpret_cast<Anywhere*>(sums + at) = total;
                    }
                } else {
#pragma unroll
                    for (int r = 0; r < COUNT; r++) {
                        if (n + r < g.n_size) {
                            const Wide one = (before ? sums[at + r] : Wide(0)) + numbers[r];
                            if (last) {
                                g.out[at + r] = static_cast<T>(one);
                            } else {
                                sums[at + r] = one;
                            }
                        }
                    }
                }
            }
        );
    }
};

/// The same from shares of k and from both parts of d (which are scaled already): a thread per number.
template <typename T> __global__ __launch_bounds__(JOIN_THREADS) void add_shares_kernel(Product<T> g, AddRows<T> finish) {
    const size_t size = static_cast<size_t>(g.groups.n_rows) * g.n_size; // (of a share)
    const size_t results = finish.twice ? size / 2 : size;
    const size_t i = blockIdx.x * static_cast<size_t>(JOIN_THREADS) + threadIdx.x;
    if (i < results) {
        wide_t<T> sum = finish.first ? wide_t<T>(0) : finish.sums[i];
        const int32_t splits = max(g.splits, 1);
#pragma unroll 8
        for (int32_t s = 0; s < splits; s++) {
            sum += g.partial[s * size + i];
        }
        if (finish.twice) { // (uniform)
#pragma unroll 8
            for (int32_t s = 0; s < splits; s++) {
                sum += g.partial[s * size + results + i];
            }
        }
        if (finish.last) {
            g.out[i] = static_cast<T>(sum);
        } else {
            finish.sums[i] = sum;
        }
    }
}

// -------------------------------------------------------------------- host --
/// Rows of which a workgroup joins two, so that there are enough workgroups (64 rows, 391 tiles: 10.8 us with 16 of them in
/// each of four workgroups, 4.7 like this).
constexpr unsigned FEW_JOINED = 2048;
/// Up to so many rows the losses are computed of all of them and those without a target left out at the end: a launch less,
/// and they are one row of tiles whatever they hold.
constexpr int32_t FEW_ROWS = 256;

/// The plan of a call's rows, in its workspace.
struct Plan {
    int32_t *order = nullptr, *offsets = nullptr, *counts = nullptr;

    static size_t bytes(int32_t rows) { return align256(static_cast<size_t>(rows) * 4) + 256 + align256(row_chunks(rows) * 4); }
    Plan() = default;
    Plan(char*& room, int32_t rows) {
        order = reinterpret_cast<int32_t*>(room);
        offsets = reinterpret_cast<int32_t*>(room + align256(static_cast<size_t>(rows) * 4));
        counts = offsets + 64;
        room += bytes(rows);
    }
};

/// What the two directions have in common.
template <typename T> class Call {
protected:
    explicit Call(const Inputs<T>& inputs)
        : in_(inputs), A_{inputs.A, static_cast<size_t>(inputs.rows), inputs.k_size},
          W_{inputs.W, static_cast<size_t>(inputs.classes), inputs.k_size} {
        logits_.groups = RowGroups{nullptr, nullptr, 1, inputs.rows};
        logits_.k_size = inputs.k_size;
    }
    double operations() const { return 2.0 * in_.rows * in_.classes * in_.k_size; }
    void choose_logits(bool copied, int32_t classes) {
        copied_ = copied;
        logits_.in_place = copied || (A_.in_place() && W_.in_place());
        logits_.n_size = classes;
        of_logits_ = tile_of_rows(logits_);
        share_k(logits_, of_logits_);
        // (classes are read once for few rows: wide tiles, where there are enough to keep the compute units busy)
        wide_ = logits_.in_place && in_.rows <= 64 && tiles(classes, WIDE_COLUMNS) >= static_cast<unsigned>(compute_units());
        if (wide_) {
            of_logits_ = WIDE_COLUMNS;
            logits_.splits = 1;
        }
    }
    template <typename Finish> void launch_logits(const Product<T>& g, hipStream_t stream, const Finish& finish) const {
        if (wide_) {
            launch_wide<T, Form::GRAD_ROWS>(g, in_.rows <= LEAST_ROWS<T> ? LEAST_ROWS<T> : 64, WIDE_COLUMNS, stream, finish);
        } else {
            launch<T, Form::GRAD_ROWS>(g, of_logits_, stream, finish);
        }
    }
    size_t copied_bytes() const { return copied_ ? A_.copied_bytes() + W_.copied_bytes() : 0; }
    /// The operands, the plan (if `planned`) and the groups of everything.
    RowGroups begin(char*& room, bool planned, hipStream_t stream) {
        plan_ = Plan(room, in_.rows);
        if (planned) {
            rows_with_targets(plan_.order, plan_.offsets, plan_.counts, in_.targets, in_.rows, in_.classes, stream);
        }
        char* none = nullptr;
        of_A_ = place(A_, copied_ ? room : none, stream);
        of_W_ = place(W_, copied_ ? room : none, stream);
        return planned ? RowGroups{plan_.offsets, plan_.order, 1, in_.rows} : RowGroups{nullptr, nullptr, 1, in_.rows};
    }

    const Inputs<T> in_;
    const Matrices<T> A_, W_;
    Operand<T> of_A_{}, of_W_{};
    Product<T> logits_{};
    Plan plan_;
    int of_logits_ = 64; // columns of a tile of logits
    bool wide_ = false, copied_ = false;
};

/// Bytes of partial sums that are in memory at a time, at most (but for those of one tile of classes): two numbers per row and
/// tile, 25 MB for 8192 rows and 100003 classes. Less where the device has not as much (forward).
constexpr size_t MOST_SUMS = size_t(1) << 29, LEAST_SUMS = size_t(1) << 17;

template <typename T> class Forward : Call<T> {
public:
    explicit Forward(const Inputs<T>& inputs) : Call<T>(inputs) {
        choose(worth_copying(this->A_, this->W_, this->operations()), MOST_SUMS);
    }
    void choose(bool copied, size_t most_bytes) {
        this->choose_logits(copied, this->in_.classes);
        const size_t most = std::max<size_t>(most_bytes / (std::max(this->in_.rows, 1) * sizeof(Sum<wide_t<T>>)), 1);
        // (where k is shared, there are few rows and few classes, and logits instead)
        each_ = this->logits_.splits > 1 || parts(this->in_.classes) <= most ? this->in_.classes
                                                                             : static_cast<int32_t>(most * this->of_logits_);
    }
    size_t bytes() const {
        return Plan::bytes(this->in_.rows) + this->copied_bytes() + target_bytes() + running_bytes() + partial_bytes();
    }
    void run(wide_t<T>* losses, wide_t<T>* log_sums, char* room, hipStream_t stream) {
        typedef wide_t<T> Wide;
        Product<T> g = this->logits_;
        g.groups = this->begin(room, this->in_.rows > FEW_ROWS, stream);
        g.q = this->of_A_;
        Wide* const target_logits = reinterpret_cast<Wide*>(room);
        room += target_bytes();
        Sum<Wide>* const running = reinterpret_cast<Sum<Wide>*>(room);
        room += running_bytes();
        Sum<Wide>* const partial = reinterpret_cast<Sum<Wide>*>(room);
        g.partial = reinterpret_cast<Wide*>(room);
        const unsigned rows = static_cast<unsigned>(this->in_.rows);
        // (without classes: one piece of none, for the zeros)
        bool last = false;
        for (int64_t at = 0; !last; at += each_) {
            const int32_t first = static_cast<int32_t>(at);
            last = this->in_.classes - first <= each_;
            g.n_size = last ? this->in_.classes - first : each_;
            g.p = Operand<T>{this->of_W_.data + static_cast<size_t>(first) * this->of_W_.stride, this->of_W_.stride};
            if (g.n_size > 0) {
                this->launch_logits(g, stream, StorePartialSums<T>{partial, target_logits, this->in_.targets, first});
            }
            auto join = [&](auto each) {
                constexpr int ROWS = decltype(each)::value;
                join_sums_kernel<T, ROWS><<<static_cast<unsigned>(ceil_div(rows, ROWS)), JOIN_SUM_THREADS, 0, stream>>>(
                    losses, log_sums, partial, running, target_logits, this->in_.targets, g.groups,
                    static_cast<int32_t>(parts(g.n_size)), this->in_.classes, first == 0, last
                );
            };
            if (g.splits > 1) {
                join_shared_sums_kernel<T><<<rows, ROW_THREADS, 0, stream>>>(losses, log_sums, this->in_.targets, g);
            } else if (rows <= FEW_JOINED) {
                join(std::integral_constant<int, 2>{});
            } else {
                join(std::integral_constant<int, 16>{});
            }
            MOPS_HIP_CHECK(hipGetLastError());
        }
    }

private:
    size_t target_bytes() const { return align256(static_cast<size_t>(this->in_.rows) * sizeof(wide_t<T>)); }
    size_t parts(int32_t classes) const { return tiles(classes, this->of_logits_); }
    size_t running_bytes() const {
        return each_ < this->in_.classes ? align256(static_cast<size_t>(this->in_.rows) * sizeof(Sum<wide_t<T>>)) : 0;
    }
    size_t partial_bytes() const {
        return this->logits_.splits > 1 ? split_bytes(this->logits_)
                                        : align256(parts(each_) * this->in_.rows * sizeof(Sum<wide_t<T>>));
    }

    int32_t each_ = 0; // classes per piece
};

template <typename T>
void forward(const Inputs<T>& inputs, wide_t<T>* losses, wide_t<T>* log_sums, hipStream_t stream) {
    Forward<T> call(inputs);
    char* workspace = static_cast<char*>(scratch_or_null(call.bytes()));
    // (as much as there is: smaller pieces of the classes do as well, and so do operands that are not copied)
    for (size_t most = MOST_SUMS; workspace == nullptr && most >= LEAST_SUMS; most /= 4) {
        call.choose(false, most);
        workspace = static_cast<char*>(scratch_or_null(call.bytes()));
    }
    if (workspace == nullptr) {
        workspace = static_cast<char*>(scratch(call.bytes()));
    }
    call.run(losses, log_sums, workspace, stream);
}

/// Bytes of d that are in memory at a time, at most (but for the smallest piece): fewer and larger pieces of the classes read
/// grad_A's sums less often and have more rounds of tiles. Less where the device has not as much (gradients).
constexpr size_t MOST_BYTES = size_t(1) << 29, LEAST_BYTES = size_t(1) << 23;
constexpr size_t SMALLEST_PIECE = 256;

template <typename T> class Backward : Call<T> {
public:
    Backward(const Inputs<T>& inputs, T* grad_A, T* grad_W) : Call<T>(inputs), grad_A_(grad_A), grad_W_(grad_W) {
        twice_ = sizeof(T) == 2 && inputs.rows <= IN_TWO_PARTS;
        sums_.groups = last_sums_.groups = rows_.groups = RowGroups{nullptr, nullptr, 1, rows_of_d()};
        sums_.n_size = last_sums_.n_size = rows_.n_size = inputs.k_size;
        choose(worth_copying(this->A_, this->W_, 3 * this->operations()), MOST_BYTES);
    }
    void choose(bool copied, size_t most_bytes) {
        const size_t classes = this->in_.classes, row_bytes = std::max<size_t>(rows_of_d(), 1) * sizeof(T);
        const size_t most = std::max(most_bytes / row_bytes / SMALLEST_PIECE * SMALLEST_PIECE, SMALLEST_PIECE);
        // Tiles of grad_W in whole rounds of all compute units, where a piece has room for one (8192 rows, 100003 classes, K =
        // 2048, bfloat16: 10.3 ms; in four pieces of the same size, 3.06 rounds each, 11.2).
        constexpr size_t TILE = sizeof(T) == 2 ? 256 : 128;
        const size_t units = static_cast<size_t>(compute_units());
        const size_t round = TILE * (units / std::gcd(units, std::max<size_t>(tiles(this->in_.k_size, TILE), 1)));
        each_ = classes <= most ? classes : round <= most ? most / round * round : most;
        stride_ = static_cast<int32_t>(ceil_div(each_, PIECE<T>)) * PIECE<T>;
        this->choose_logits(copied, static_cast<int32_t>(each_));
        sums_.in_place = last_sums_.in_place = copied || twice_ || this->A_.in_place();
        rows_.in_place = copied || this->W_.in_place();
        sums_.m_size = rows_.k_size = static_cast<int32_t>(each_);
        // (the last piece may be a small one, whose rows are shared out further)
        last_sums_.m_size = static_cast<int32_t>(each_ > 0 ? this->in_.classes - (ceil_div(this->in_.classes, each_) - 1) * each_ : 0);
        of_sums_ = choose_sums(sums_);
        of_last_sums_ = choose_sums(last_sums_);
        of_rows_ = tile_of_rows(rows_);
        share_k(rows_, of_rows_, rows_.groups.n_rows <= FEW_ROWS_OF_D ? 2 : 1);
    }
    bool copies() const { return this->copied_bytes() > 0; }
    size_t bytes() const {
        return Plan::bytes(this->in_.rows) + this->copied_bytes() + 256 + twice_bytes() + d_bytes() + total_bytes() +
               std::max(split_bytes(this->logits_), row_bytes() + sum_bytes());
    }
    void run(
        const wide_t<T>* grad_losses, const wide_t<T>* grad_log_sums, const wide_t<T>* log_sums, char* room,
        hipStream_t stream
    ) {
        typedef wide_t<T> Wide;
        const Inputs<T>& in = this->in_;
        RowGroups groups = this->begin(room, !twice_, stream), groups_of_d = groups;
        // (numbers in two parts are as good at any scale that their type holds)
        const bool scaled = SCALED<T> && (std::is_same_v<T, _Float16> || !twice_);
        const Unscale<T> scale{scaled ? reinterpret_cast<float*>(room) : nullptr};
        room += 256;
        Operand<T> A = this->of_A_;
        if constexpr (SCALED<T>) {
            if (twice_) {
                std::tie(groups, groups_of_d, A) = twice(scale.scale, grad_losses, grad_log_sums, room, stream);
            } else {
                find_scale(
                    scale.scale, grad_losses, grad_log_sums, in.targets, groups, in.classes,
                    std::is_same_v<T, _Float16>, stream
                );
            }
        }
        T* const d = reinterpret_cast<T*>(room);
        room += d_bytes();
        Wide* const totals = reinterpret_cast<Wide*>(room);
        room += total_bytes();
        // (without classes: one piece of none, for the zeros of grad_A)
        bool last = false;
        for (size_t first = 0; !last; first += each_) {
            const int32_t count = static_cast<int32_t>(std::min(each_, static_cast<size_t>(in.classes) - first));
            last = first + each_ >= static_cast<size_t>(in.classes);
            const size_t W_at = first * this->of_W_.stride;
            Product<T> g = this->logits_;
            g.groups = groups;
            g.n_size = count;
            g.q = this->of_A_;
            g.p = Operand<T>{this->of_W_.data + W_at, this->of_W_.stride};
            g.partial = reinterpret_cast<Wide*>(room);
            const StoreGradients<T> make{
                {grad_losses, grad_log_sums, log_sums, in.targets, static_cast<int32_t>(first), scale}, d, stride_,
                twice_ ? static_cast<size_t>(in.rows) * stride_ : 0
            };
            if (count > 0) {
                this->launch_logits(g, stream, make);
            }
            if (count > 0 && g.splits > 1) {
                const size_t blocks = ceil_div(static_cast<size_t>(in.rows) * stride_, JOIN_THREADS);
                join_shared_gradients_kernel<T><<<static_cast<unsigned>(blocks), JOIN_THREADS, 0, stream>>>(g, make);
                MOPS_HIP_CHECK(hipGetLastError());
            }
            Product<T> sums = last ? last_sums_ : sums_, rows = rows_;
            sums.groups = rows.groups = groups_of_d;
            sums.out = grad_W_ != nullptr ? grad_W_ + first * in.k_size : nullptr;
            rows.k_size = count;
            sums.q = rows.q = Operand<T>{d, stride_};
            sums.p = A;
            rows.out = grad_A_;
            rows.p = g.p;
            rows.partial = reinterpret_cast<Wide*>(room);
            sums.partial = reinterpret_cast<Wide*>(room + row_bytes());
            multiply(sums, last ? of_last_sums_ : of_sums_, rows, StoreSums<T, Form::GRAD_SUMS, Unscale<T>>{scale}, AddRows<T>{totals, first == 0, last, twice_, scale}, stream);
        }
    }

private:
    int32_t rows_of_d() const { return this->in_.rows * (twice_ ? 2 : 1); }
    size_t d_bytes() const { return align256(static_cast<size_t>(rows_of_d()) * stride_ * sizeof(T)); }
    size_t plan_of_d_bytes() const { return 256 + align256(static_cast<size_t>(rows_of_d()) * 4); }
    size_t twice_bytes() const {
        return twice_ ? plan_of_d_bytes() + align256(static_cast<size_t>(rows_of_d()) * this->A_.pieces() * 16) : 0;
    }
    /// The plans of the rows and of both parts of d, and the rows of A twice.
    std::tuple<RowGroups, RowGroups, Operand<T>> twice(
        float* scale, const float* grad_losses, const float* grad_log_sums, char*& room, hipStream_t stream
    ) const {
        const Inputs<T>& in = this->in_;
        int32_t *const offsets = reinterpret_cast<int32_t*>(room), *const order = offsets + 64;
        T* const to = reinterpret_cast<T*>(room + plan_of_d_bytes());
        const int32_t pieces = this->A_.pieces();
        const size_t blocks = std::max<size_t>(ceil_div(static_cast<size_t>(in.rows) * pieces, TWICE_THREADS), 1);
        twice_kernel<T><<<static_cast<unsigned>(blocks), TWICE_THREADS, 0, stream>>>(
            to, this->of_A_, in.k_size, pieces, PlanOfTwice{this->plan_.order, this->plan_.offsets, order, offsets, scale},
            in.targets, grad_losses, grad_log_sums, in.rows, in.classes
        );
        MOPS_HIP_CHECK(hipGetLastError());
        room += twice_bytes();
        return {
            RowGroups{this->plan_.offsets, this->plan_.order, 1, in.rows}, RowGroups{offsets, order, 1, rows_of_d()},
            Operand<T>{to, pieces * PIECE<T>}
        };
    }
    size_t total_bytes() const { // (of grad_A over the pieces)
        return grad_A_ != nullptr && each_ < static_cast<size_t>(this->in_.classes)
                   ? align256(static_cast<size_t>(this->in_.rows) * this->in_.k_size * sizeof(wide_t<T>))
                   : 0;
    }
    size_t row_bytes() const {
        const size_t of_share = align256(static_cast<size_t>(rows_of_d()) * rows_.n_size * sizeof(wide_t<T>));
        return grad_A_ == nullptr ? 0 : twice_ && rows_.splits <= 1 ? of_share : split_bytes(rows_);
    }
    size_t sum_bytes() const {
        auto of = [](const Product<T>& sums) {
            return sums.most_slots * partial_size(sums.m_size, sums.n_size) * sizeof(wide_t<T>);
        };
        return grad_W_ != nullptr ? std::max(of(sums_), of(last_sums_)) : 0;
    }
    static int choose_sums(Product<T>& sums) {
        const int tile = tile_of_sums(sums);
        share_rows(sums);
        sums.most_slots = most_split_units(sums.groups.n_rows, sums.step);
        return tile;
    }
    /// Smaller units than all rows ask for, for rows of which most may have no target: an eighth, or what partial results of
    /// MOST_PARTIAL bytes allow (200000 rows, 30000 with a target, 94 classes, K = 128, float: 32 us, 63 without).
    static void share_rows(Product<T>& sums) {
        constexpr size_t MOST_PARTIAL = size_t(1) << 25;
        const size_t of_unit = partial_size(sums.m_size, sums.n_size) * sizeof(wide_t<T>);
        const int32_t least = std::max(sums.step / 8, 256);
        for (;;) {
            const int32_t half = static_cast<int32_t>(ceil_div(static_cast<size_t>(sums.step) / 2, 64) * 64);
            if (half < least || half == sums.step || most_split_units(sums.groups.n_rows, half) * of_unit > MOST_PARTIAL) {
                return;
            }
            sums.step = half;
        }
    }
    /// Both products with a piece of d, in one launch where their tiles are the same.
    void multiply(
        Product<T>& sums, int of_sums, Product<T>& rows, const StoreSums<T, Form::GRAD_SUMS, Unscale<T>>& finish_sums,
        const AddRows<T>& finish_rows, hipStream_t stream
    ) {
        const bool of_W = sums.out != nullptr, of_A = rows.out != nullptr;
        if (of_W && of_A && of_sums == of_rows_ && sums.in_place == rows.in_place) {
            const unsigned for_sums = set_tiles<Form::GRAD_SUMS>(sums, of_sums);
            const unsigned for_rows = set_tiles<Form::FORWARD>(rows, of_rows_);
            with_tile<T>(of_sums, sums.in_place, [&](auto size, auto m, auto n, auto is_aligned) {
                constexpr int TILE = decltype(size)::value, WM = decltype(m)::value, WN = decltype(n)::value;
                constexpr bool ALIGNED = decltype(is_aligned)::value;
                gradients_kernel<
                    T, TILE, TILE, WM, WN, DEEP, STAGES_OF<TILE, ALIGNED>, ALIGNED, Form::FORWARD,
                    StoreSums<T, Form::GRAD_SUMS, Unscale<T>>, AddRows<T>>
                    <<<for_sums + for_rows, WM * WN * WAVE, 0, stream>>>(sums, rows, for_sums, finish_sums, finish_rows);
            });
            MOPS_HIP_CHECK(hipGetLastError());
        } else {
            if (of_W) {
                launch<T, Form::GRAD_SUMS>(sums, of_sums, stream, finish_sums);
            }
            if (of_A) {
                launch<T, Form::FORWARD>(rows, of_rows_, stream, finish_rows);
            }
        }
        if (of_A && (rows.splits > 1 || (twice_ && this->in_.rows > 0 && rows.n_size > 0))) {
            const size_t blocks = ceil_div(static_cast<size_t>(this->in_.rows) * rows.n_size, JOIN_THREADS); // (of numbers of grad_A)
            add_shares_kernel<T><<<static_cast<unsigned>(blocks), JOIN_THREADS, 0, stream>>>(rows, finish_rows);
            MOPS_HIP_CHECK(hipGetLastError());
        }
        if (of_W && sums.most_slots > 0) {
            const unsigned workgroups = 4 * static_cast<unsigned>(compute_units());
            join_units_kernel<T><<<workgroups, JOIN_WAVES * WAVE, 0, stream>>>(sums);
            MOPS_HIP_CHECK(hipGetLastError());
        }
    }

    T *const grad_A_, *const grad_W_;
    bool twice_; // d is in two parts
    size_t each_; // classes per piece
    int32_t stride_;
    Product<T> sums_{}, last_sums_{}, rows_{};
    int of_sums_ = 64, of_last_sums_ = 64, of_rows_ = 64;
};

template <typename T>
void gradients(
    const Inputs<T>& inputs, const wide_t<T>* grad_losses, const wide_t<T>* grad_log_sums, const wide_t<T>* log_sums,
    T* grad_A, T* grad_W, hipStream_t stream
) {
    Backward<T> call(inputs, grad_A, grad_W);
    // (as much as there is: smaller pieces of the classes do as well, and so do operands that are not copied)
    char* workspace = static_cast<char*>(scratch_or_null(call.bytes()));
    for (size_t most = MOST_BYTES; workspace == nullptr && most >= LEAST_BYTES; most /= 4) {
        call.choose(false, most);
        workspace = static_cast<char*>(scratch_or_null(call.bytes()));
    }
    if (workspace == nullptr) {
        workspace = static_cast<char*>(scratch(call.bytes()));
    }
    call.run(grad_losses, grad_log_sums, log_sums, workspace, stream);
}

} // namespace mops::amd::cross_entropy

#endif
