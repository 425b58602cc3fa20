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
// afterwards), or the numbers d, rounded to T (what the matrix instructions
// take; 16-bit floats scaled, see Unscale). Of d, a piece of the classes is in
// memory at a time, and both products with it follow while the caches hold what
// they can of it; grad_A is summed up over the pieces in 32 bits.
//
// Rows without a target in range are in no group (rows_with_targets): they cost
// nothing, and whatever they hold reaches nothing.
#ifndef MOPS_AMD_CROSS_ENTROPY_KERNELS_HPP
#define MOPS_AMD_CROSS_ENTROPY_KERNELS_HPP

#include <limits>
#include <type_traits>

#include "cross_entropy.hpp"
#include "grouped_launch.hpp"
#include "grouped_tiles.hpp"
#include "numbers.hpp"
#include "runtime.hpp"

namespace mops::amd::cross_entropy {

using namespace grouped_product;

__device__ __forceinline__ float power(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }
__device__ __forceinline__ double power(double x) { return exp(x); }
__device__ __forceinline__ float logarithm(float x) { return logf(x); }
__device__ __forceinline__ double logarithm(double x) { return log(x); }
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double larger(double a, double b) { return fmax(a, b); }

/// The largest of some logits and the sum of exp(x - largest). (Not-a-number is never the largest; it makes the sum one.)
template <typename Wide> struct Sum {
    Wide most, sum;

    static __device__ __forceinline__ Wide lowest() { return -std::numeric_limits<Wide>::infinity(); }
    /// What the powers are taken relative to: no difference of infinities where there is nothing.
    static __device__ __forceinline__ Wide base(Wide most) { return most == lowest() ? Wide(0) : most; }
    __device__ __forceinline__ void join(const Sum& other) {
        const Wide both = larger(most, other.most);
        sum = sum * power(most - base(both)) + other.sum * power(other.most - base(both));
        most = both;
    }
    __device__ __forceinline__ Wide logarithm_of_sum() const { return most + logarithm(sum); }
};

// ----------------------------------------------------------- sums by tiles --
/// partial[tile of classes][place]; target_logits[row], where the tile has the row's target.
template <typename T> struct StorePartialSums {
    typedef wide_t<T> Wide;
    static constexpr bool PAIRS = false, RESTS = false;
    Sum<Wide>* partial;
    Wide* target_logits;
    const int32_t* targets;

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
        const int32_t first = t.n0 + t.across() * Tile::NB * Tile::BLOCK; // class of the wavefront's first column
        const bool whole = t.n0 + BN <= g.n_size; // (uniform)
#pragma unroll
        for (int i = 0; i < Tile::MB; i++) {
            const int32_t row = t.rows[min(t.row(i), t.unit.count - 1)];
            const int32_t target = targets[row] - first;
            Sum<Wide> all{Sum<Wide>::lowest(), 0};
            Wide of_target = 0;
#pragma unroll
            for (int j = 0; j < Tile::NB; j++) {
#pragma unroll
                for (int e = 0; e < Tile::HELD; e++) {
                    const int at = j * Tile::BLOCK + t.column(e);
                    const Wide x = t.sums[i][j][e];
                    all.most = larger(all.most, whole || first + at < g.n_size ? x : Sum<Wide>::lowest());
                    of_target = at == target ? x : of_target;
                }
            }
#pragma unroll
            for (int s = Tile::BLOCK; s < WAVE; s *= 2) {
                all.most = larger(all.most, __shfl_xor(all.most, s));
            }
            const Wide base = Sum<Wide>::base(all.most);
#pragma unroll
            for (int j = 0; j < Tile::NB; j++) {
#pragma unroll
                for (int e = 0; e < Tile::HELD; e++) {
                    const int at = j * Tile::BLOCK + t.column(e);
                    const Wide one = power(t.sums[i][j][e] - base);
                    all.sum += whole || first + at < g.n_size ? one : Wide(0);
                }
            }
#pragma unroll
            for (int s = Tile::BLOCK; s < WAVE; s *= 2) {
                all.sum += __shfl_xor(all.sum, s);
            }
            if (t.lane < Tile::BLOCK) {
                shared[t.across() * BM + t.row(i)] = all;
            }
            // (one lane of all tiles has the target's column)
            bool mine = false;
#pragma unroll
            for (int j = 0; j < Tile::NB; j++) {
#pragma unroll
                for (int e = 0; e < Tile::HELD; e++) {
                    mine = mine || j * Tile::BLOCK + t.column(e) == target;
                }
            }
            if (mine && t.row(i) < t.unit.count) {
                target_logits[row] = of_target;
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

/// losses and log_sums of JOINED_ROWS places per workgroup, JOIN_LANES threads each, from the sums of `parts` tiles; zeros
/// for the rows without a target.
constexpr int JOINED_ROWS = 16, JOIN_LANES = 16;
template <typename T>
__global__ __launch_bounds__(JOINED_ROWS* JOIN_LANES) void join_sums_kernel(
    wide_t<T>* __restrict__ losses, wide_t<T>* __restrict__ log_sums, const Sum<wide_t<T>>* __restrict__ partial,
    const wide_t<T>* __restrict__ target_logits, RowGroups groups, int32_t parts
) {
    typedef wide_t<T> Wide;
    __shared__ Sum<Wide> shared[JOIN_LANES][JOINED_ROWS];
    const int in_block = threadIdx.x % JOINED_ROWS, lane = threadIdx.x / JOINED_ROWS;
    const int32_t place = blockIdx.x * JOINED_ROWS + in_block, kept = groups.end_of(0, groups.begin_of(0));
    Sum<Wide> all{Sum<Wide>::lowest(), 0};
    if (place < kept) {
        for (int32_t p = lane; p < parts; p += JOIN_LANES) {
            all.join(partial[static_cast<size_t>(p) * groups.n_rows + place]);
        }
    }
    shared[lane][in_block] = all;
    __syncthreads();
    if (lane == 0 && place < groups.n_rows) {
        const int32_t row = groups.row_at(place);
        Wide loss = 0, log_sum = 0;
        if (place < kept) {
            for (int l = 1; l < JOIN_LANES; l++) {
                all.join(shared[l][in_block]);
            }
            log_sum = all.logarithm_of_sum();
            loss = all.most - target_logits[row] + logarithm(all.sum);
        }
        losses[row] = loss;
        log_sums[row] = log_sum;
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
    if (place >= kept) { // (uniform)
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
        all.join(Sum<Wide>{x == x ? x : Sum<Wide>::lowest(), x == x ? power(x - Sum<Wide>::base(x)) : x});
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
        losses[row] = all.most - target_logit + logarithm(all.sum);
        log_sums[row] = all.logarithm_of_sum();
    }
}

// ---------------------------------------------------------------- gradients --
/// 16-bit floats have five bits of exponent: d, most of whose numbers are a probability times a weight (of a mean: one in
/// the number of rows), would lose most of its bits. It is stored times a power of two that brings the largest weight of
/// the call to 2^13 .. 2^14 (twice that is the most d can be: below 65504), and the sums are divided by it again before they
/// are rounded, which is exact. The other types have the exponents of `wide` or more than the weights need.
template <typename T> constexpr bool SCALED = std::is_same_v<T, _Float16>;
template <typename T> struct Unscale {
    const float* scale; // and its inverse (SCALED)

    __device__ __forceinline__ wide_t<T> factor() const {
        if constexpr (SCALED<T>) {
            return scale[0];
        }
        return 1;
    }
    __device__ __forceinline__ wide_t<T> operator()(wide_t<T> sum) const {
        if constexpr (SCALED<T>) {
            return sum * scale[1];
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
        Wide log_sum, of_power, of_target;
        int32_t target;

        __device__ __forceinline__ Wide make(Wide x, int32_t n) const {
            return of_power * power(x - log_sum) - (n == target ? of_target : Wide(0));
        }
    };
    __device__ __forceinline__ OfRow of_row(int32_t row) const {
        const Wide g = grad_losses != nullptr ? grad_losses[row] : Wide(0);
        const Wide h = grad_log_sums != nullptr ? grad_log_sums[row] : Wide(0);
        return OfRow{log_sums[row], (g + h) * scale.factor(), g * scale.factor(), targets[row] - first};
    }
};

/// d[row, 0 .. stride - 1], whole pieces with zeros behind n_size.
template <typename T> struct StoreGradients : Weights<T> {
    typedef wide_t<T> Wide;
    static constexpr bool PAIRS = false, RESTS = false;
    T* d;
    int32_t stride;

    template <bool MAY_SPLIT, int LDS_BYTES, int BM, int BN, int WM, int WN>
    __device__ __forceinline__ void operator()(const Product<T>& g, const TileOf<T, BM, BN, WM, WN>& t) const {
        typedef TileOf<T, BM, BN, WM, WN> Tile;
        if constexpr (MAY_SPLIT) {
            if (g.splits > 1) { // (uniform)
                StoreSums<T, Form::GRAD_ROWS>{}.template operator()<MAY_SPLIT, LDS_BYTES>(g, t);
                return;
            }
        }
        typename Weights<T>::OfRow of[Tile::MB];
#pragma unroll
        for (int i = 0; i < Tile::MB; i++) {
            of[i] = this->of_row(t.rows[min(t.row(i), t.unit.count - 1)]);
        }
        const int32_t first = t.n0 + t.across() * Tile::NB * Tile::BLOCK;
        const bool whole = t.n0 + BN <= g.n_size; // (uniform)
        turn_over<T, Tile::NB, LDS_BYTES>(
            t,
            [&](int i, int j, int e) {
                const int32_t n = first + j * Tile::BLOCK + t.column(e);
                const Wide made = of[i].make(t.sums[i][j][e], n);
                return whole || n < g.n_size ? made : Wide(0);
            },
            [&](int row, int column, const typename Packed<T>::Numbers& numbers) {
                T* const to = row < t.unit.count ? d + static_cast<size_t>(t.rows[row]) * stride : nullptr;
                store_piece<false, T>(to, t.n0 + column, stride, numbers);
            }
        );
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
}

/// grad_A, summed up over the pieces of the classes in `sums` [row][n_size] (only where there are several).
template <typename T> struct AddRows {
    typedef wide_t<T> Wide;
    static constexpr bool PAIRS = false, RESTS = true;
    Wide* sums;
    bool first, last;
    Unscale<T> scale;

    template <bool MAY_SPLIT, int LDS_BYTES, int BM, int BN, int WM, int WN>
    __device__ __forceinline__ void operator()(const Product<T>& g, const TileOf<T, BM, BN, WM, WN>& t) const {
        typedef TileOf<T, BM, BN, WM, WN> Tile;
        const bool alone = first && last;
        const bool rest = t.unit.group == g.groups.n_groups;
        if ((MAY_SPLIT && g.splits > 1) || alone) { // (uniform)
            StoreSums<T, Form::FORWARD, Unscale<T>>{scale}.template operator()<MAY_SPLIT, LDS_BYTES>(g, t);
            return;
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

/// The same from shares of k (which are scaled already): a thread per number.
template <typename T> __global__ __launch_bounds__(JOIN_THREADS) void add_shares_kernel(Product<T> g, AddRows<T> finish) {
    const size_t size = static_cast<size_t>(g.groups.n_rows) * g.n_size;
    const size_t i = blockIdx.x * static_cast<size_t>(JOIN_THREADS) + threadIdx.x;
    if (i < size) {
        wide_t<T> sum = finish.first ? wide_t<T>(0) : finish.sums[i];
#pragma unroll 8
        for (int32_t s = 0; s < g.splits; s++) {
            sum += g.partial[s * size + i];
        }
        if (finish.last) {
            g.out[i] = static_cast<T>(sum);
        } else {
            finish.sums[i] = sum;
        }
    }
}

// -------------------------------------------------------------------- host --
/// The plan of a call's rows, in its workspace.
struct Plan {
    int32_t *order, *offsets, *counts;

    static size_t bytes(int32_t rows) { return align256(static_cast<size_t>(rows) * 4) + 256 + align256(row_chunks(rows) * 4); }
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
    }
    size_t copied_bytes() const { return copied_ ? A_.copied_bytes() + W_.copied_bytes() : 0; }
    /// The operands, the plan and the groups of everything.
    RowGroups begin(char*& room, hipStream_t stream) {
        const Plan plan(room, in_.rows);
        rows_with_targets(plan.order, plan.offsets, plan.counts, in_.targets, in_.rows, in_.classes, stream);
        char* none = nullptr;
        of_A_ = place(A_, copied_ ? room : none, stream);
        of_W_ = place(W_, copied_ ? room : none, stream);
        return RowGroups{plan.offsets, plan.order, 1, in_.rows};
    }

    const Inputs<T> in_;
    const Matrices<T> A_, W_;
    Operand<T> of_A_{}, of_W_{};
    Product<T> logits_{};
    int of_logits_ = 64;
    bool copied_ = false;
};

template <typename T> class Forward : Call<T> {
public:
    explicit Forward(const Inputs<T>& inputs) : Call<T>(inputs) { choose(worth_copying(this->A_, this->W_, this->operations())); }
    void choose(bool copied) { this->choose_logits(copied, this->in_.classes); }
    bool copies() const { return this->copied_bytes() > 0; }
    size_t bytes() const { return Plan::bytes(this->in_.rows) + this->copied_bytes() + target_bytes() + partial_bytes(); }
    void run(wide_t<T>* losses, wide_t<T>* log_sums, char* room, hipStream_t stream) {
        typedef wide_t<T> Wide;
        Product<T> g = this->logits_;
        g.groups = this->begin(room, stream);
        g.q = this->of_A_;
        g.p = this->of_W_;
        Wide* const target_logits = reinterpret_cast<Wide*>(room);
        room += target_bytes();
        Sum<Wide>* const partial = reinterpret_cast<Sum<Wide>*>(room);
        g.partial = reinterpret_cast<Wide*>(room);
        if (g.n_size > 0) {
            launch<T, Form::GRAD_ROWS>(
                g, this->of_logits_, stream, StorePartialSums<T>{partial, target_logits, this->in_.targets}
            );
        }
        const unsigned rows = static_cast<unsigned>(this->in_.rows);
        if (g.splits > 1) {
            join_shared_sums_kernel<T><<<rows, ROW_THREADS, 0, stream>>>(losses, log_sums, this->in_.targets, g);
        } else {
            join_sums_kernel<T>
                <<<static_cast<unsigned>(ceil_div(rows, JOINED_ROWS)), JOINED_ROWS * JOIN_LANES, 0, stream>>>(
                    losses, log_sums, partial, target_logits, g.groups, static_cast<int32_t>(parts())
                );
        }
        MOPS_HIP_CHECK(hipGetLastError());
    }

private:
    size_t target_bytes() const { return align256(static_cast<size_t>(this->in_.rows) * sizeof(wide_t<T>)); }
    size_t parts() const { return tiles(this->in_.classes, this->of_logits_); }
    size_t partial_bytes() const {
        return this->logits_.splits > 1 ? split_bytes(this->logits_)
                                        : align256(parts() * this->in_.rows * sizeof(Sum<wide_t<T>>));
    }
};

template <typename T>
void forward(const Inputs<T>& inputs, wide_t<T>* losses, wide_t<T>* log_sums, hipStream_t stream) {
    Forward<T> call(inputs);
    char* workspace = call.copies() ? static_cast<char*>(scratch_or_null(call.bytes())) : nullptr;
    if (workspace == nullptr) {
        call.choose(false);
        workspace = static_cast<char*>(scratch(call.bytes()));
    }
    call.run(losses, log_sums, workspace, stream);
}

/// Bytes of d that are in memory at a time, at most (but for the smallest piece).
constexpr size_t MOST_BYTES = size_t(1) << 29;
constexpr size_t SMALLEST_PIECE = 256;

template <typename T> class Backward : Call<T> {
public:
    Backward(const Inputs<T>& inputs, T* grad_A, T* grad_W) : Call<T>(inputs), grad_A_(grad_A), grad_W_(grad_W) {
        const size_t classes = inputs.classes, rows = inputs.rows;
        const size_t pieces = std::max<size_t>(ceil_div(rows * classes * sizeof(T), MOST_BYTES), 1);
        each_ = std::min(ceil_div(ceil_div(classes, pieces), SMALLEST_PIECE) * SMALLEST_PIECE, classes);
        stride_ = static_cast<int32_t>(ceil_div(each_, PIECE<T>)) * PIECE<T>;
        sums_.groups = rows_.groups = this->logits_.groups;
        sums_.n_size = rows_.n_size = inputs.k_size;
        choose(worth_copying(this->A_, this->W_, 3 * this->operations()));
    }
    void choose(bool copied) {
        this->choose_logits(copied, static_cast<int32_t>(each_));
        sums_.in_place = copied || this->A_.in_place();
        rows_.in_place = copied || this->W_.in_place();
        sums_.m_size = rows_.k_size = static_cast<int32_t>(each_);
        of_sums_ = tile_of_sums(sums_);
        sums_.most_slots = most_split_units(sums_.groups.n_rows, sums_.step);
        of_rows_ = tile_of_rows(rows_);
        share_k(rows_, of_rows_);
    }
    bool copies() const { return this->copied_bytes() > 0; }
    size_t bytes() const {
        return Plan::bytes(this->in_.rows) + this->copied_bytes() + 256 + d_bytes() + total_bytes() +
               std::max(split_bytes(this->logits_), row_bytes() + sum_bytes());
    }
    void run(
        const wide_t<T>* grad_losses, const wide_t<T>* grad_log_sums, const wide_t<T>* log_sums, char* room,
        hipStream_t stream
    ) {
        typedef wide_t<T> Wide;
        const Inputs<T>& in = this->in_;
        const RowGroups groups = this->begin(room, stream);
        const Unscale<T> scale{reinterpret_cast<float*>(room)};
        if constexpr (SCALED<T>) {
            find_scale(
                reinterpret_cast<float*>(room), grad_losses, grad_log_sums, in.targets, in.rows, in.classes, stream
            );
        }
        room += 256;
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
                {grad_losses, grad_log_sums, log_sums, in.targets, static_cast<int32_t>(first), scale}, d, stride_
            };
            if (count > 0) {
                launch<T, Form::GRAD_ROWS>(g, this->of_logits_, stream, make);
            }
            if (count > 0 && g.splits > 1) {
                const size_t blocks = ceil_div(static_cast<size_t>(in.rows) * stride_, JOIN_THREADS);
                join_shared_gradients_kernel<T><<<static_cast<unsigned>(blocks), JOIN_THREADS, 0, stream>>>(g, make);
                MOPS_HIP_CHECK(hipGetLastError());
            }
            Product<T> sums = sums_, rows = rows_;
            sums.groups = rows.groups = groups;
            sums.out = grad_W_ != nullptr ? grad_W_ + first * in.k_size : nullptr;
            sums.m_size = rows.k_size = count;
            sums.q = rows.q = Operand<T>{d, stride_};
            sums.p = this->of_A_;
            rows.out = grad_A_;
            rows.p = g.p;
            rows.partial = reinterpret_cast<Wide*>(room);
            sums.partial = reinterpret_cast<Wide*>(room + row_bytes());
            multiply(sums, rows, StoreSums<T, Form::GRAD_SUMS, Unscale<T>>{scale}, AddRows<T>{totals, first == 0, last, scale}, stream);
        }
    }

private:
    size_t d_bytes() const { return align256(static_cast<size_t>(this->in_.rows) * stride_ * sizeof(T)); }
    size_t total_bytes() const { // (of grad_A over the pieces)
        return grad_A_ != nullptr && each_ < static_cast<size_t>(this->in_.classes)
                   ? align256(static_cast<size_t>(this->in_.rows) * this->in_.k_size * sizeof(wide_t<T>))
                   : 0;
    }
    size_t row_bytes() const { return grad_A_ != nullptr ? split_bytes(rows_) : 0; }
    size_t sum_bytes() const {
        return grad_W_ != nullptr ? sums_.most_slots * partial_size(sums_.m_size, sums_.n_size) * sizeof(wide_t<T>) : 0;
    }
    /// Both products with a piece of d, in one launch where their tiles are the same.
    void multiply(
        Product<T>& sums, Product<T>& rows, const StoreSums<T, Form::GRAD_SUMS, Unscale<T>>& finish_sums,
        const AddRows<T>& finish_rows, hipStream_t stream
    ) {
        const bool of_W = sums.out != nullptr, of_A = rows.out != nullptr;
        if (of_W && of_A && of_sums_ == of_rows_ && sums.in_place == rows.in_place) {
            const unsigned for_sums = set_tiles<Form::GRAD_SUMS>(sums, of_sums_);
            const unsigned for_rows = set_tiles<Form::FORWARD>(rows, of_rows_);
            with_tile<T>(of_sums_, sums.in_place, [&](auto size, auto m, auto n, auto is_aligned) {
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
                launch<T, Form::GRAD_SUMS>(sums, of_sums_, stream, finish_sums);
            }
            if (of_A) {
                launch<T, Form::FORWARD>(rows, of_rows_, stream, finish_rows);
            }
        }
        if (of_A && rows.splits > 1) {
            const size_t blocks = ceil_div(static_cast<size_t>(rows.groups.n_rows) * rows.n_size, JOIN_THREADS);
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
    size_t each_; // classes per piece
    int32_t stride_;
    Product<T> sums_{}, rows_{};
    int of_sums_ = 64, of_rows_ = 64;
};

template <typename T>
void gradients(
    const Inputs<T>& inputs, const wide_t<T>* grad_losses, const wide_t<T>* grad_log_sums, const wide_t<T>* log_sums,
    T* grad_A, T* grad_W, hipStream_t stream
) {
    Backward<T> call(inputs, grad_A, grad_W);
    char* workspace = call.copies() ? static_cast<char*>(scratch_or_null(call.bytes())) : nullptr;
    if (workspace == nullptr) {
        call.choose(false);
        workspace = static_cast<char*>(scratch(call.bytes()));
    }
    call.run(grad_losses, grad_log_sums, log_sums, workspace, stream);
}

} // namespace mops::amd::cross_entropy

#endif
