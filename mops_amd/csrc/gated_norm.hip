// The residual update around a block, with the norm behind the block and the
// norm in front of the next one:
//
//   norm(x) = x / sqrt(mean(x^2) + epsilon)              (row by row)
//   state   = residual + s gate norm(block) weight_block
//   next    = norm(state) weight_next
//
// and its gradients. Everything is bound by memory: a row is read once, held in
// registers (a team of lanes per row, up to four pieces of 16 bytes per lane),
// and its results are written once. Rows of more than 2048 pieces (the
// gradients of 16-bit rows: 1024) are read three times instead (`wide` kernels).
//
// Gradients. With b = block, y = norm(b) = b rb, a = s gate y weight_block,
// t = residual + a, rt = 1 / sqrt(mean(t^2) + epsilon), h = grad_next weight_next:
//
//   d  = grad_state + rt (h - t c),  c = rt^2 mean(h t)         (= grad_residual)
//   grad_gate  = s d y weight_block
//   grad_block = rb (k - y mean(k y)),  k = s d gate weight_block
//   grad_weight_block = sum over rows of s d gate y
//   grad_weight_next  = sum over rows of grad_next t rt
//
// k y = d a, so mean(k y) follows from sums that need no d:
//   sum(d a) = sum(grad_state a) + rt (sum(h a) - c sum(t a)),
// which leaves two rounds of sums per row (b^2; then t^2, h t, grad_state a, h a,
// t a) instead of three. Sums over the rows: every workgroup keeps its own in
// registers over the rows it walks and leaves them in scratch memory, where a
// second launch adds them up in a fixed order.
#include "mops/layers.hpp"

#include <algorithm>

#include "checks.hpp"
#include "device_common.hpp"
#include "numbers.hpp"
#include "runtime.hpp"

namespace mops::amd {
namespace gated_norm {
namespace {

template <typename T> struct Forward {
    T *state, *next;
    const T *residual, *block, *gate, *weight_block, *weight_next;
    int32_t n_rows;
    PiecesOfRow row;
    bool gate_per_row;
    wide_t<T> scale, epsilon;
};

template <typename T> struct Gradients {
    T *grad_residual, *grad_block, *grad_gate;
    const T *grad_state, *grad_next; // (null: zero)
    const T *residual, *block, *gate, *weight_block, *weight_next;
    wide_t<T>* sums;  // [workgroup][which][columns]: weight_block, weight_next, gate (of one row); null: not wanted
    wide_t<T>* of_row; // [row][3], `wide` kernels: rb, rt, c
    int32_t n_rows;
    PiecesOfRow row;
    bool gate_per_row;
    wide_t<T> scale, epsilon;
};

/// 1 / sqrt(x) to the last bits of the type (the hardware's single-precision estimate is good to one).
__device__ __forceinline__ float inverse_root(float x) { return rsqrtf(x); }
__device__ __forceinline__ double inverse_root(double x) { return 1.0 / sqrt(x); }

/// The sums over the TEAM lanes of a row, in all of them. Teams of more than a wavefront: all threads
/// of the workgroup call it, `room` holds COUNT numbers per wavefront.
template <int TEAM, int COUNT, typename W> __device__ __forceinline__ void sum_over_team(W (&sum)[COUNT], W* room) {
#pragma unroll
    for (int step = 1; step < (TEAM < WAVE ? TEAM : WAVE); step *= 2) {
#pragma unroll
        for (int i = 0; i < COUNT; i++) {
            sum[i] += __shfl_xor(sum[i], step);
        }
    }
    if constexpr (TEAM > WAVE) {
        constexpr int WAVES = TEAM / WAVE;
        const int wave = threadIdx.x / WAVE, lane = threadIdx.x & (WAVE - 1);
        if (lane == 0) {
#pragma unroll
            for (int i = 0; i < COUNT; i++) {
                room[i * WAVES + wave] = sum[i];
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < COUNT; i++) {
            sum[i] = 0;
#pragma unroll
            for (int w = 0; w < WAVES; w++) {
                sum[i] += room[i * WAVES + w];
            }
        }
    }
}

/// A lane's pieces of a row: piece p * TEAM + lane, p < P. The last piece of the row repeats columns of the one
/// before (PiecesOfRow): `fresh` says from which of its columns on a piece counts in sums over the row.
template <int TEAM, int P, int N> struct Columns {
    int32_t at[P], fresh[P];

    __device__ __forceinline__ Columns(const PiecesOfRow& row, int lane) {
#pragma unroll
        for (int p = 0; p < P; p++) {
            const int32_t piece = p * TEAM + lane;
            at[p] = row.start<N>(min(piece, row.pieces - 1));
            fresh[p] = piece < row.pieces ? piece * N - at[p] : N;
        }
    }
    __device__ __forceinline__ bool holds(int p) const { return fresh[p] < N; }
};

/// Threads of a workgroup whose teams have TEAM lanes.
template <int TEAM> constexpr int THREADS_OF = TEAM > 256 ? TEAM : 256;

/// Both results, bound by memory: three reads and two writes per number (four with a shared gate), 16 384 rows of 4096
/// bfloat16 with a gate each in 101 us, 6.6 TB/s. What is read once streams past the caches (127 us through them).
template <typename T, int TEAM, int P, int N>
__global__ __launch_bounds__(THREADS_OF<TEAM>) void forward_kernel(Forward<T> f) {
    typedef wide_t<T> W;
    typedef Piece<T, N> Row;
    constexpr int TEAMS = THREADS_OF<TEAM> / TEAM;
    __shared__ W room[2][2][TEAM > WAVE ? TEAM / WAVE : 1];
    const int lane = threadIdx.x & (TEAM - 1);
    const Columns<TEAM, P, N> column(f.row, lane);
    const W of_columns = W(1) / f.row.columns;
    Row weight_block[P], weight_next[P], shared_gate[P];
#pragma unroll
    for (int p = 0; p < P; p++) {
        weight_block[p] = Row::load(f.weight_block + column.at[p]);
        weight_next[p] = Row::load(f.weight_next + column.at[p]);
        shared_gate[p] = Row::load(f.gate + column.at[p]);
    }
    // (the number of steps is the same for all teams of a workgroup: they meet in sum_over_team)
    int parity = 0;
    for (int32_t base = blockIdx.x * TEAMS; base < f.n_rows; base += gridDim.x * TEAMS, parity ^= 1) {
        const int32_t row = base + static_cast<int32_t>(threadIdx.x) / TEAM;
        const size_t begin = static_cast<size_t>(min(row, f.n_rows - 1)) * f.row.columns;
        Row block[P], residual[P], gate[P];
#pragma unroll
        for (int p = 0; p < P; p++) {
            block[p] = Row::stream(f.block + begin + column.at[p]);
            residual[p] = Row::stream(f.residual + begin + column.at[p]);
            gate[p] = f.gate_per_row ? Row::stream(f.gate + begin + column.at[p]) : shared_gate[p];
        }
        W sum[1] = {0};
#pragma unroll
        for (int p = 0; p < P; p++) {
#pragma unroll
            for (int j = 0; j < N; j++) {
                const W b = block[p].get(j);
                sum[0] += j >= column.fresh[p] ? b * b : W(0);
            }
        }
        sum_over_team<TEAM, 1>(sum, &room[parity][0][0]);
        const W inverse_block = inverse_root(sum[0] * of_columns + f.epsilon) * f.scale;
        W state[P][N];
        sum[0] = 0;
#pragma unroll
        for (int p = 0; p < P; p++) {
#pragma unroll
            for (int j = 0; j < N; j++) {
                state[p][j] = residual[p].get(j) +
                              gate[p].get(j) * (block[p].get(j) * inverse_block) * weight_block[p].get(j);
                sum[0] += j >= column.fresh[p] ? state[p][j] * state[p][j] : W(0);
            }
        }
        sum_over_team<TEAM, 1>(sum, &room[parity][1][0]);
        const W inverse_state = inverse_root(sum[0] * of_columns + f.epsilon);
        if (row < f.n_rows) {
#pragma unroll
            for (int p = 0; p < P; p++) {
                if (column.holds(p)) {
                    Row to_state, to_next;
#pragma unroll
                    for (int j = 0; j < N; j++) {
                        to_state.set(j, state[p][j]);
                        to_next.set(j, state[p][j] * inverse_state * weight_next[p].get(j));
                    }
                    to_state.store(f.state + begin + column.at[p]);
                    to_next.store(f.next + begin + column.at[p]);
                }
            }
        }
    }
}

/// All gradients of a row in one pass, bound by memory: five reads and three writes per number, 16 384 rows of 4096 bfloat16
/// in 188 us, 5.7 TB/s; 50 021 rows of 384 floats with a shared gate in 86, 5.4 TB/s. The sums over the rows stay in
/// registers, which is what limits the lanes' pieces.
template <typename T, int TEAM, int P, int N>
__global__ __launch_bounds__(THREADS_OF<TEAM>) void gradient_kernel(Gradients<T> g) {
    typedef wide_t<T> W;
    typedef Piece<T, N> Row;
    constexpr int THREADS = THREADS_OF<TEAM>, TEAMS = THREADS / TEAM;
    __shared__ W room[2][6][TEAM > WAVE ? TEAM / WAVE : 1];
    __shared__ W joined[TEAMS > 1 ? THREADS * N : 1];
    const int lane = threadIdx.x & (TEAM - 1);
    const Columns<TEAM, P, N> column(g.row, lane);
    const W of_columns = W(1) / g.row.columns;
    Row weight_block[P], weight_next[P], shared_gate[P];
    W for_block[P][N], for_next[P][N], for_gate[P][N];
#pragma unroll
    for (int p = 0; p < P; p++) {
        weight_block[p] = Row::load(g.weight_block + column.at[p]);
        weight_next[p] = Row::load(g.weight_next + column.at[p]);
        shared_gate[p] = Row::load(g.gate + column.at[p]);
#pragma unroll
        for (int j = 0; j < N; j++) {
            for_block[p][j] = for_next[p][j] = for_gate[p][j] = 0;
        }
    }
    int parity = 0;
    for (int32_t base = blockIdx.x * TEAMS; base < g.n_rows; base += gridDim.x * TEAMS, parity ^= 1) {
        const int32_t row = base + static_cast<int32_t>(threadIdx.x) / TEAM;
        const bool valid = row < g.n_rows;
        const size_t begin = static_cast<size_t>(min(row, g.n_rows - 1)) * g.row.columns;
        Row block[P], residual[P], gate[P], grad_state[P], grad_next[P];
#pragma unroll
        for (int p = 0; p < P; p++) {
            const size_t at = begin + column.at[p];
            block[p] = Row::stream(g.block + at);
            residual[p] = Row::stream(g.residual + at);
            gate[p] = g.gate_per_row ? Row::stream(g.gate + at) : shared_gate[p];
            grad_state[p] = g.grad_state != nullptr ? Row::stream(g.grad_state + at) : Row{};
            grad_next[p] = g.grad_next != nullptr ? Row::stream(g.grad_next + at) : Row{};
        }
        W sum[1] = {0};
#pragma unroll
        for (int p = 0; p < P; p++) {
#pragma unroll
            for (int j = 0; j < N; j++) {
                const W b = block[p].get(j);
                sum[0] += j >= column.fresh[p] ? b * b : W(0);
            }
        }
        sum_over_team<TEAM, 1>(sum, &room[parity][0][0]);
        const W rb = inverse_root(sum[0] * of_columns + g.epsilon);
        W sums[5] = {0, 0, 0, 0, 0};
#pragma unroll
        for (int p = 0; p < P; p++) {
#pragma unroll
            for (int j = 0; j < N; j++) {
                const W a = g.scale * gate[p].get(j) * (block[p].get(j) * rb) * weight_block[p].get(j);
                const W t = residual[p].get(j) + a;
                const W h = grad_next[p].get(j) * weight_next[p].get(j);
                if (j >= column.fresh[p]) {
                    sums[0] += t * t;
                    sums[1] += h * t;
                    sums[2] += grad_state[p].get(j) * a;
                    sums[3] += h * a;
                    sums[4] += t * a;
                }
            }
        }
        sum_over_team<TEAM, 5>(sums, &room[parity][1][0]);
        const W rt = inverse_root(sums[0] * of_columns + g.epsilon);
        const W c = rt * rt * (sums[1] * of_columns);
        const W mean_ky = (sums[2] + rt * (sums[3] - c * sums[4])) * of_columns;
#pragma unroll
        for (int p = 0; p < P; p++) {
            Row to_residual, to_block, to_gate;
#pragma unroll
            for (int j = 0; j < N; j++) {
                const W y = block[p].get(j) * rb, wb = weight_block[p].get(j), gj = gate[p].get(j);
                const W t = residual[p].get(j) + g.scale * gj * y * wb;
                const W gn = grad_next[p].get(j);
                const W d = grad_state[p].get(j) + rt * (gn * weight_next[p].get(j) - t * c);
                const W through = g.scale * d * gj, on_gate = g.scale * d * y * wb;
                to_residual.set(j, d);
                to_block.set(j, rb * (through * wb - y * mean_ky));
                to_gate.set(j, on_gate);
                if (valid) {
                    for_block[p][j] += through * y;
                    for_next[p][j] += gn * t * rt;
                    for_gate[p][j] += on_gate;
                }
            }
            if (valid && column.holds(p)) {
                const size_t at = begin + column.at[p];
                if (g.grad_residual != nullptr) {
                    to_residual.stream_to(g.grad_residual + at);
                }
                if (g.grad_block != nullptr) {
                    to_block.stream_to(g.grad_block + at);
                }
                if (g.grad_gate != nullptr) {
                    to_gate.stream_to(g.grad_gate + at);
                }
            }
        }
    }
    if (g.sums == nullptr) {
        return;
    }
    // what this workgroup has of the sums over the rows (columns that two pieces hold are the same in both)
    const int which = g.gate_per_row ? 2 : 3;
    for (int w = 0; w < which; w++) {
#pragma unroll
        for (int p = 0; p < P; p++) {
            W total[N];
#pragma unroll
            for (int j = 0; j < N; j++) {
                total[j] = w == 0 ? for_block[p][j] : w == 1 ? for_next[p][j] : for_gate[p][j];
            }
            if constexpr (TEAMS > 1) {
                __syncthreads();
#pragma unroll
                for (int j = 0; j < N; j++) {
                    joined[j * THREADS + threadIdx.x] = total[j];
                }
                __syncthreads();
                if (static_cast<int>(threadIdx.x) < TEAM) {
                    for (int t = 1; t < TEAMS; t++) {
#pragma unroll
                        for (int j = 0; j < N; j++) {
                            total[j] += joined[j * THREADS + t * TEAM + threadIdx.x];
                        }
                    }
                }
            }
            if (static_cast<int>(threadIdx.x) < TEAM && column.holds(p)) {
                W* to = g.sums + (static_cast<size_t>(blockIdx.x) * which + w) * g.row.columns + column.at[p];
#pragma unroll
                for (int j = 0; j < N; j++) {
                    to[j] = total[j];
                }
            }
        }
    }
}

/// to[column] := the sum over the workgroups of what they have (512 of them and 4096 columns of two sums: 17 MB, read from the
/// caches, 6 us): 16 lanes side by side for 16 columns, and 16 shares of
/// the workgroups.
constexpr int JOIN_COLUMNS = 16, JOIN_SHARES = 16;
template <typename T>
__global__ __launch_bounds__(JOIN_COLUMNS* JOIN_SHARES) void join_kernel(
    T* __restrict__ grad_weight_block, T* __restrict__ grad_weight_next, T* __restrict__ grad_gate,
    const wide_t<T>* __restrict__ sums, int32_t workgroups, int32_t which, int32_t columns
) {
    __shared__ wide_t<T> shared[JOIN_SHARES][JOIN_COLUMNS + 1];
    T* const to = blockIdx.y == 0 ? grad_weight_block : blockIdx.y == 1 ? grad_weight_next : grad_gate;
    if (to == nullptr) {
        return; // (uniform)
    }
    const int32_t of = threadIdx.x & (JOIN_COLUMNS - 1), share = threadIdx.x / JOIN_COLUMNS;
    const int32_t column = blockIdx.x * JOIN_COLUMNS + of;
    wide_t<T> sum = 0;
    if (column < columns) {
#pragma unroll 8
        for (int32_t b = share; b < workgroups; b += JOIN_SHARES) {
            sum += sums[(static_cast<size_t>(b) * which + blockIdx.y) * columns + column];
        }
    }
    shared[share][of] = sum;
    __syncthreads();
    if (share == 0 && column < columns) {
        for (int s = 1; s < JOIN_SHARES; s++) {
            sum += shared[s][of];
        }
        to[column] = static_cast<T>(sum);
    }
}

// Rows that do not fit the registers of a workgroup: read again for every step, number by number, from the caches (3300
// rows of 20 000 bfloat16: 270 us, 2.0 TB/s of what has to move; gradients 624, 1.7).
constexpr int WIDE_THREADS = 1024;

template <typename T> __global__ __launch_bounds__(WIDE_THREADS) void wide_forward_kernel(Forward<T> f) {
    typedef wide_t<T> W;
    __shared__ W room[2][WIDE_THREADS / WAVE];
    const size_t begin = static_cast<size_t>(blockIdx.x) * f.row.columns;
    const T* gate = f.gate_per_row ? f.gate + begin : f.gate;
    W sum[1] = {0};
    for (int32_t i = threadIdx.x; i < f.row.columns; i += WIDE_THREADS) {
        const W b = static_cast<W>(f.block[begin + i]);
        sum[0] += b * b;
    }
    sum_over_team<WIDE_THREADS, 1>(sum, room[0]);
    const W rb = inverse_root(sum[0] / f.row.columns + f.epsilon) * f.scale;
    auto state_at = [&](int32_t i) {
        return static_cast<W>(f.residual[begin + i]) +
               static_cast<W>(gate[i]) * (static_cast<W>(f.block[begin + i]) * rb) * static_cast<W>(f.weight_block[i]);
    };
    sum[0] = 0;
    for (int32_t i = threadIdx.x; i < f.row.columns; i += WIDE_THREADS) {
        const W t = state_at(i);
        sum[0] += t * t;
    }
    sum_over_team<WIDE_THREADS, 1>(sum, room[1]);
    const W rt = inverse_root(sum[0] / f.row.columns + f.epsilon);
    for (int32_t i = threadIdx.x; i < f.row.columns; i += WIDE_THREADS) {
        const W t = state_at(i);
        f.state[begin + i] = static_cast<T>(t);
        f.next[begin + i] = static_cast<T>(t * rt * static_cast<W>(f.weight_next[i]));
    }
}

/// What the gradient has at a column of a row: shared by the two `wide` kernels.
template <typename T> struct AtColumn {
    wide_t<T> y, wb, gate, t, gn, h, gs;

    __device__ __forceinline__ AtColumn(const Gradients<T>& g, size_t begin, int32_t i, wide_t<T> rb) {
        typedef wide_t<T> W;
        y = static_cast<W>(g.block[begin + i]) * rb;
        wb = static_cast<W>(g.weight_block[i]);
        gate = static_cast<W>(g.gate[g.gate_per_row ? begin + i : i]);
        t = static_cast<W>(g.residual[begin + i]) + g.scale * gate * y * wb;
        gn = g.grad_next != nullptr ? static_cast<W>(g.grad_next[begin + i]) : W(0);
        h = gn * static_cast<W>(g.weight_next[i]);
        gs = g.grad_state != nullptr ? static_cast<W>(g.grad_state[begin + i]) : W(0);
    }
};

template <typename T> __global__ __launch_bounds__(WIDE_THREADS) void wide_gradient_kernel(Gradients<T> g) {
    typedef wide_t<T> W;
    __shared__ W room[6][WIDE_THREADS / WAVE];
    const size_t begin = static_cast<size_t>(blockIdx.x) * g.row.columns;
    W sum[1] = {0};
    for (int32_t i = threadIdx.x; i < g.row.columns; i += WIDE_THREADS) {
        const W b = static_cast<W>(g.block[begin + i]);
        sum[0] += b * b;
    }
    sum_over_team<WIDE_THREADS, 1>(sum, room[0]);
    const W rb = inverse_root(sum[0] / g.row.columns + g.epsilon);
    W sums[5] = {0, 0, 0, 0, 0};
    for (int32_t i = threadIdx.x; i < g.row.columns; i += WIDE_THREADS) {
        const AtColumn<T> v(g, begin, i, rb);
        const W a = g.scale * v.gate * v.y * v.wb;
        sums[0] += v.t * v.t;
        sums[1] += v.h * v.t;
        sums[2] += v.gs * a;
        sums[3] += v.h * a;
        sums[4] += v.t * a;
    }
    sum_over_team<WIDE_THREADS, 5>(sums, room[1]);
    const W rt = inverse_root(sums[0] / g.row.columns + g.epsilon);
    const W c = rt * rt * (sums[1] / g.row.columns);
    const W mean_ky = (sums[2] + rt * (sums[3] - c * sums[4])) / g.row.columns;
    if (threadIdx.x == 0 && g.of_row != nullptr) {
        W* to = g.of_row + 3 * static_cast<size_t>(blockIdx.x);
        to[0] = rb;
        to[1] = rt;
        to[2] = c;
    }
    for (int32_t i = threadIdx.x; i < g.row.columns; i += WIDE_THREADS) {
        const AtColumn<T> v(g, begin, i, rb);
        const W d = v.gs + rt * (v.h - v.t * c);
        if (g.grad_residual != nullptr) {
            g.grad_residual[begin + i] = static_cast<T>(d);
        }
        if (g.grad_block != nullptr) {
            g.grad_block[begin + i] = static_cast<T>(rb * (g.scale * d * v.gate * v.wb - v.y * mean_ky));
        }
        if (g.grad_gate != nullptr) {
            g.grad_gate[begin + i] = static_cast<T>(g.scale * d * v.y * v.wb);
        }
    }
}

/// The sums over the rows of a column, by a lane, for a share of the rows per workgroup.
constexpr int WIDE_COLUMNS = 256;
template <typename T> __global__ __launch_bounds__(WIDE_COLUMNS) void wide_sums_kernel(Gradients<T> g) {
    typedef wide_t<T> W;
    const int32_t i = blockIdx.x * WIDE_COLUMNS + threadIdx.x;
    if (i >= g.row.columns) {
        return;
    }
    W for_block = 0, for_next = 0, for_gate = 0;
    for (int32_t row = blockIdx.y; row < g.n_rows; row += gridDim.y) {
        const W* of_row = g.of_row + 3 * static_cast<size_t>(row);
        const W rb = of_row[0], rt = of_row[1], c = of_row[2];
        const AtColumn<T> v(g, static_cast<size_t>(row) * g.row.columns, i, rb);
        const W d = v.gs + rt * (v.h - v.t * c);
        for_block += g.scale * d * v.gate * v.y;
        for_next += v.gn * v.t * rt;
        for_gate += g.scale * d * v.y * v.wb;
    }
    const int which = g.gate_per_row ? 2 : 3;
    W* to = g.sums + static_cast<size_t>(blockIdx.y) * which * g.row.columns + i;
    to[0] = for_block;
    to[g.row.columns] = for_next;
    if (which == 3) {
        to[2 * static_cast<size_t>(g.row.columns)] = for_gate;
    }
}

/// A row has the lanes that its pieces fill, and as few pieces per lane as that takes: rows of up to 1024 pieces fit the registers of 256 or 512 lanes. Gradients of 67 million numbers of
/// bfloat16: 183 us in rows of 256 (32 lanes; with 64, half of them idle, 307), 187 of 1024 (64 lanes with two pieces),
/// 191 of 4096 (256 with two), 245 of 8192 (512 with two; 256 with four, one workgroup per compute unit, 290).
/// body(TEAM, P, N): the lanes per row and pieces per lane that hold a row; false: none does, or it has more than MOST
/// pieces.
template <typename T, int MOST, typename Body> bool by_columns(int32_t columns, Body&& body) {
    auto with = [&](auto team, auto pieces, auto width) {
        body(team, pieces, width);
        return true;
    };
    constexpr int N = PIECE<T>;
    const int32_t pieces = (columns + N - 1) / N;
    std::integral_constant<int, 1> one;
    std::integral_constant<int, 2> two;
    std::integral_constant<int, 4> four;
    std::integral_constant<int, 16> lanes16;
    std::integral_constant<int, 32> lanes32;
    std::integral_constant<int, 64> lanes64;
    std::integral_constant<int, 256> lanes256;
    std::integral_constant<int, 512> lanes512;
    std::integral_constant<int, N> n;
    if (columns < N) {
        return with(lanes16, one, one);
    }
    if (pieces <= 16) {
        return with(lanes16, one, n);
    }
    if (pieces <= 32) {
        return with(lanes32, one, n);
    }
    if (pieces <= 64) {
        return with(lanes64, one, n);
    }
    if (pieces <= 128) {
        return with(lanes64, two, n);
    }
    if (pieces <= 256) {
        return with(lanes256, one, n);
    }
    if (pieces <= 512) {
        return with(lanes256, two, n);
    }
    if (pieces <= 1024) {
        return with(lanes512, two, n);
    }
    if constexpr (MOST >= 2048) {
        if (pieces <= 2048) {
            return with(lanes512, four, n);
        }
    }
    return false;
}

/// Workgroups that walk over the rows: enough for every compute unit to have `resident` of them.
unsigned workgroups(int32_t n_rows, int teams, int resident) {
    const size_t wanted = ceil_div(static_cast<size_t>(n_rows), static_cast<size_t>(teams));
    return static_cast<unsigned>(std::min<size_t>(wanted, static_cast<size_t>(compute_units()) * resident));
}

template <typename T> void forward(Forward<T> f, int32_t columns, hipStream_t stream) {
    const bool held = by_columns<T, 2048>(columns, [&](auto team, auto pieces, auto width) {
        constexpr int TEAM = decltype(team)::value, P = decltype(pieces)::value, N = decltype(width)::value;
        f.row = PiecesOfRow::make<N>(columns);
        const int resident = 2048 / THREADS_OF<TEAM>;
        forward_kernel<T, TEAM, P, N>
            <<<workgroups(f.n_rows, THREADS_OF<TEAM> / TEAM, resident), THREADS_OF<TEAM>, 0, stream>>>(f);
    });
    if (!held) {
        f.row = PiecesOfRow::make<1>(columns);
        wide_forward_kernel<T><<<static_cast<unsigned>(f.n_rows), WIDE_THREADS, 0, stream>>>(f);
    }
    MOPS_HIP_CHECK(hipGetLastError());
}

template <typename T>
void gradients(
    Gradients<T> g, T* grad_weight_block, T* grad_weight_next, T* grad_gate_of_all, int32_t columns, hipStream_t stream
) {
    const bool wants_sums =
        grad_weight_block != nullptr || grad_weight_next != nullptr || grad_gate_of_all != nullptr;
    const int which = g.gate_per_row ? 2 : 3;
    auto sums_bytes = [&](unsigned groups) {
        return wants_sums ? align256(static_cast<size_t>(groups) * which * columns * sizeof(wide_t<T>)) : 0;
    };
    unsigned groups = 0;
    // (four pieces of eight numbers do not fit the registers with all that the gradients keep of them: 4096 rows of
    // 16 384 bfloat16 would be 851 us with 768 bytes of spilled registers per lane, number by number they are 587)
    constexpr int MOST = sizeof(T) == 2 ? 1024 : 2048;
    const bool held = by_columns<T, MOST>(columns, [&](auto team, auto pieces, auto width) {
        constexpr int TEAM = decltype(team)::value, P = decltype(pieces)::value, N = decltype(width)::value;
        g.row = PiecesOfRow::make<N>(columns);
        // (two workgroups of 256 per compute unit: 16 384 rows of 4096 bfloat16 are 195 us, with three of them, which do
        // not all fit, 223 us, with four 198)
        groups = workgroups(g.n_rows, THREADS_OF<TEAM> / TEAM, 512 / THREADS_OF<TEAM>);
        g.sums = wants_sums ? static_cast<wide_t<T>*>(scratch(sums_bytes(groups))) : nullptr;
        gradient_kernel<T, TEAM, P, N><<<groups, THREADS_OF<TEAM>, 0, stream>>>(g);
    });
    if (!held) {
        g.row = PiecesOfRow::make<1>(columns);
        groups = static_cast<unsigned>(std::min(g.n_rows, 64));
        if (wants_sums) {
            char* workspace = static_cast<char*>(
                scratch(sums_bytes(groups) + 3 * static_cast<size_t>(g.n_rows) * sizeof(wide_t<T>))
            );
            g.sums = reinterpret_cast<wide_t<T>*>(workspace);
            g.of_row = reinterpret_cast<wide_t<T>*>(workspace + sums_bytes(groups));
        }
        wide_gradient_kernel<T><<<static_cast<unsigned>(g.n_rows), WIDE_THREADS, 0, stream>>>(g);
        if (wants_sums) {
            const unsigned blocks = static_cast<unsigned>(ceil_div(static_cast<size_t>(columns), WIDE_COLUMNS));
            wide_sums_kernel<T><<<dim3(blocks, groups), WIDE_COLUMNS, 0, stream>>>(g);
        }
    }
    if (wants_sums) {
        const unsigned blocks = static_cast<unsigned>(ceil_div(static_cast<size_t>(columns), JOIN_COLUMNS));
        join_kernel<T><<<dim3(blocks, which), JOIN_COLUMNS * JOIN_SHARES, 0, stream>>>(
            grad_weight_block, grad_weight_next, grad_gate_of_all, g.sums, static_cast<int32_t>(groups), which, columns
        );
    }
    MOPS_HIP_CHECK(hipGetLastError());
}

template <typename T> __global__ void zero_kernel(T* __restrict__ data, int32_t count) {
    const int32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i < count) {
        data[i] = static_cast<T>(0.f);
    }
}

} // namespace
} // namespace gated_norm
} // namespace mops::amd

namespace mops::cuda {

using namespace mops::amd;

namespace {

template <typename scalar_t>
void check_update(
    const checks::Validator& check, Tensor<scalar_t, 2> residual, Tensor<scalar_t, 2> block, Tensor<scalar_t, 2> gate,
    Tensor<scalar_t, 1> weight_block, Tensor<scalar_t, 1> weight_next
) {
    using checks::axis_of;
    check.same_extent(axis_of(block, "block", 0), axis_of(residual, "residual", 0));
    check.same_extent(axis_of(block, "block", 1), axis_of(residual, "residual", 1));
    check.same_extent(axis_of(gate, "gate", 1), axis_of(residual, "residual", 1));
    check.same_extent(axis_of(weight_block, "weight_block", 0), axis_of(residual, "residual", 1));
    check.same_extent(axis_of(weight_next, "weight_next", 0), axis_of(residual, "residual", 1));
    if (gate.shape[0] != 1 && gate.shape[0] != residual.shape[0]) {
        throw std::runtime_error(
            "gate must have one row or as many rows as residual (" + std::to_string(residual.shape[0]) + ") in " +
            check.operation() + ", got " + std::to_string(gate.shape[0])
        );
    }
}

template <typename scalar_t>
void check_like(
    const checks::Validator& check, Tensor<scalar_t, 2> tensor, const char* name, Tensor<scalar_t, 2> like,
    const char* like_name
) {
    if (tensor.data != nullptr) {
        check.same_extent(checks::axis_of(tensor, name, 0), checks::axis_of(like, like_name, 0));
        check.same_extent(checks::axis_of(tensor, name, 1), checks::axis_of(like, like_name, 1));
    }
}

} // namespace

template <typename scalar_t>
void gated_residual_norm(
    Tensor<scalar_t, 2> state, Tensor<scalar_t, 2> next, Tensor<scalar_t, 2> residual, Tensor<scalar_t, 2> block,
    Tensor<scalar_t, 2> gate, Tensor<scalar_t, 1> weight_block, Tensor<scalar_t, 1> weight_next,
    double residual_scale, double epsilon
) {
    typedef device_t<scalar_t> T;
    const checks::Validator check("gated_residual_norm");
    check_update(check, residual, block, gate, weight_block, weight_next);
    check.same_extent(checks::axis_of(state, "state", 0), checks::axis_of(residual, "residual", 0));
    check.same_extent(checks::axis_of(state, "state", 1), checks::axis_of(residual, "residual", 1));
    check.same_extent(checks::axis_of(next, "next", 0), checks::axis_of(residual, "residual", 0));
    check.same_extent(checks::axis_of(next, "next", 1), checks::axis_of(residual, "residual", 1));
    const int32_t n_rows = count_i32(residual.shape[0], "number of rows");
    const int32_t columns = count_i32(residual.shape[1], "number of columns");
    if (n_rows > 0 && columns > 0) {
        gated_norm::Forward<T> f{};
        f.state = data_of(state);
        f.next = data_of(next);
        f.residual = data_of(residual);
        f.block = data_of(block);
        f.gate = data_of(gate);
        f.weight_block = data_of(weight_block);
        f.weight_next = data_of(weight_next);
        f.n_rows = n_rows;
        f.gate_per_row = gate.shape[0] != 1;
        f.scale = static_cast<wide_t<T>>(residual_scale);
        f.epsilon = static_cast<wide_t<T>>(epsilon);
        gated_norm::forward(f, columns, current_stream());
    }
    finish_call("gated_residual_norm");
}

template <typename scalar_t>
void gated_residual_norm_vjp(
    Tensor<scalar_t, 2> grad_residual, Tensor<scalar_t, 2> grad_block, Tensor<scalar_t, 2> grad_gate,
    Tensor<scalar_t, 1> grad_weight_block, Tensor<scalar_t, 1> grad_weight_next, Tensor<scalar_t, 2> grad_state,
    Tensor<scalar_t, 2> grad_next, Tensor<scalar_t, 2> residual, Tensor<scalar_t, 2> block, Tensor<scalar_t, 2> gate,
    Tensor<scalar_t, 1> weight_block, Tensor<scalar_t, 1> weight_next, double residual_scale, double epsilon
) {
    typedef device_t<scalar_t> T;
    const checks::Validator check("gated_residual_norm_vjp");
    check_update(check, residual, block, gate, weight_block, weight_next);
    check_like(check, grad_state, "grad_state", residual, "residual");
    check_like(check, grad_next, "grad_next", residual, "residual");
    check_like(check, grad_residual, "grad_residual", residual, "residual");
    check_like(check, grad_block, "grad_block", residual, "residual");
    check_like(check, grad_gate, "grad_gate", gate, "gate");
    if (grad_weight_block.data != nullptr) {
        check.same_extent(
            checks::axis_of(grad_weight_block, "grad_weight_block", 0), checks::axis_of(residual, "residual", 1)
        );
    }
    if (grad_weight_next.data != nullptr) {
        check.same_extent(
            checks::axis_of(grad_weight_next, "grad_weight_next", 0), checks::axis_of(residual, "residual", 1)
        );
    }
    const int32_t n_rows = count_i32(residual.shape[0], "number of rows");
    const int32_t columns = count_i32(residual.shape[1], "number of columns");
    const bool gate_per_row = gate.shape[0] != 1;
    if (columns > 0) {
        if (n_rows > 0) {
            gated_norm::Gradients<T> g{};
            g.grad_residual = data_of(grad_residual);
            g.grad_block = data_of(grad_block);
            g.grad_gate = gate_per_row ? data_of(grad_gate) : nullptr;
            g.grad_state = data_of(grad_state);
            g.grad_next = data_of(grad_next);
            g.residual = data_of(residual);
            g.block = data_of(block);
            g.gate = data_of(gate);
            g.weight_block = data_of(weight_block);
            g.weight_next = data_of(weight_next);
            g.n_rows = n_rows;
            g.gate_per_row = gate_per_row;
            g.scale = static_cast<wide_t<T>>(residual_scale);
            g.epsilon = static_cast<wide_t<T>>(epsilon);
            gated_norm::gradients(
                g, data_of(grad_weight_block), data_of(grad_weight_next), gate_per_row ? nullptr : data_of(grad_gate),
                columns, current_stream()
            );
        } else { // sums over no rows
            T* const sums[3] = {
                data_of(grad_weight_block), data_of(grad_weight_next), gate_per_row ? nullptr : data_of(grad_gate)
            };
            for (T* to : sums) {
                if (to != nullptr) {
                    const unsigned blocks = static_cast<unsigned>(ceil_div(static_cast<size_t>(columns), 256));
                    gated_norm::zero_kernel<T><<<blocks, 256, 0, current_stream()>>>(to, columns);
                }
            }
        }
    }
    finish_call("gated_residual_norm_vjp");
}

#define MOPS_GATED_NORM_INSTANTIATE(T)                                                             \
    template void gated_residual_norm<T>(                                                          \
        Tensor<T, 2>, Tensor<T, 2>, Tensor<T, 2>, Tensor<T, 2>, Tensor<T, 2>, Tensor<T, 1>, Tensor<T, 1>, double, double \
    );                                                                                             \
    template void gated_residual_norm_vjp<T>(                                                      \
        Tensor<T, 2>, Tensor<T, 2>, Tensor<T, 2>, Tensor<T, 1>, Tensor<T, 1>, Tensor<T, 2>, Tensor<T, 2>, Tensor<T, 2>, \
        Tensor<T, 2>, Tensor<T, 2>, Tensor<T, 1>, Tensor<T, 1>, double, double                     \
    );
MOPS_GATED_NORM_INSTANTIATE(float)
MOPS_GATED_NORM_INSTANTIATE(double)
MOPS_GATED_NORM_INSTANTIATE(bfloat16)
MOPS_GATED_NORM_INSTANTIATE(float16)

} // namespace mops::cuda
