// A table looked up by an index, times a constant, and its gradient:
//
//   output[i, :]     = scale * table[indices[i], :]
//   grad_table[v, :] = scale * sum_{i: indices[i] = v} grad_output[i, :]
//
// Both only move memory. Forward: a team of lanes per row, a lane per 16 bytes
// of it, several rows on their way at once (32 768 rows of 2048 bfloat16: 44 us,
// 6.1 TB/s; 64 rows: 3.6, the launch). Gradient: the rows are put in the
// order of their index first (order_all_by_group, or the caller's plan); then
// every row of the table is the sum over consecutive places of that order, by
// the one team that stores it: no atomics, and an order of summation that
// depends on the indices only. A row of the table that very many rows name (a
// frequent word, an abundant element) would be one team's work of thousands of
// steps: a launch before sums up every whole chunk of places that lies inside
// one row of the table, by workgroups that are spread over the GPU, and its
// owner adds those sums and the places at either end.
#include "mops/layers.hpp"

#include <algorithm>

#include "checks.hpp"
#include "device_common.hpp"
#include "numbers.hpp"
#include "plan_bounds.hpp"
#include "runtime.hpp"
#include "sender_buckets.hpp"
#include "wave_sort.hpp"

namespace mops::amd {
namespace embedding {
namespace {

constexpr int THREADS = 256;
constexpr int AHEAD = 8;            // rows that a team has on their way
// Places of a chunk: a multiple of CHUNK_PLACES that makes some CHUNKS chunks, and no more than PLACES_EACH per team. (So 32
// for rows as wide as a workgroup, where a chunk is one team's work: 32 768 tokens of 100 003, 2048 bfloat16: 122 us, with
// 64 places 124; 4386 rows of 1024, 2500 float16: 25 and 35; 20 000 rows of 94, 2048 bfloat16: 35 and 31. Chunks of 32 are
// summed also inside rows of 33 to 64 places, whose teams do not read them: where such rows are left out, all of these
// take the same time.)
constexpr int32_t PLACES_EACH = 32;
constexpr int32_t CHUNKS = 1024;
constexpr int32_t CHUNK_PLACES = 64;
// Places that a team sums up by itself (with 32, 64 and 128, a plan given: 32 768 tokens of 100 003, 2048 bfloat16: 90, 90 and
// 134 us; 44 721 rows of 33 749, 223 float16: 19, 26 and 42; 65 536 of 50 000, 512 bfloat16, skewed: 40, 50 and 66).
constexpr int32_t ALONE = 64;
// Rows per table row from which on a workgroup has one table row (with 4, 16 and 64, a plan given: 30 000 rows of 5000, 256
// floats: 12.2, 8.5 and 8.0 us; 200 000 of them: 34, 34 and 37; 20 000 rows of 1000, 64 floats, skewed: 8.3, 8.8 and 10.8;
// 12 000 of them: 7.7, 10.3 and 10.2; 80 000 of 2000, 8 floats, skewed: 8.8, 8.4 and 12.8).
constexpr int32_t FEW = 16;
constexpr int32_t ROWS_PER_TEAM = 8; // at most
// Table rows of a workgroup, at most: their places in LDS (few_rows_kernel). They matter where rows are a few numbers wide
// (200 rows of 3 000 000, 2 floats: 15.0 us, with 256 of them 18.3; 18 050 of 1 000 000, 3 float16: 11.5 and 11.2).
constexpr int32_t TABLE_ROWS = 1024;

/// How a row's pieces are shared out: `team` lanes (a power of two) hold a piece each.
struct Teams {
    PiecesOfRow row;
    int32_t team, teams; // lanes per team, teams per workgroup
    unsigned tiles;      // workgroups beside each other that hold a row

    template <int N> static Teams make(int32_t columns, int32_t most_lanes = THREADS) {
        Teams t;
        t.row = PiecesOfRow::make<N>(columns);
        t.team = 1;
        while (t.team < most_lanes && t.team < t.row.pieces) {
            t.team *= 2;
        }
        t.teams = THREADS / t.team;
        t.tiles = static_cast<unsigned>(ceil_div(static_cast<size_t>(t.row.pieces), static_cast<size_t>(t.team)));
        return t;
    }
};

template <typename T, int N, int ROWS>
__global__ __launch_bounds__(THREADS) void lookup_kernel(
    T* __restrict__ output, const T* __restrict__ table, const int32_t* __restrict__ indices, int32_t n_rows,
    int32_t table_rows, Teams teams, wide_t<T> scale
) {
    const int32_t piece = blockIdx.y * teams.team + (threadIdx.x & (teams.team - 1));
    const int32_t first = (blockIdx.x * teams.teams + threadIdx.x / teams.team) * ROWS;
    if (piece >= teams.row.pieces) {
        return;
    }
    const int32_t column = teams.row.start<N>(piece);
    const size_t columns = teams.row.columns;
    int32_t index[ROWS];
    Piece<T, N> value[ROWS];
#pragma unroll
    for (int u = 0; u < ROWS; u++) {
        index[u] = indices[min(first + u, n_rows - 1)];
    }
#pragma unroll
    for (int u = 0; u < ROWS; u++) {
        value[u] = Piece<T, N>::load(table + (in_bounds(index[u], table_rows) ? index[u] : 0) * columns + column);
    }
#pragma unroll
    for (int u = 0; u < ROWS; u++) {
        if (first + u >= n_rows) {
            break;
        }
        const bool inside = in_bounds(index[u], table_rows);
#pragma unroll
        for (int j = 0; j < N; j++) {
            value[u].set(j, inside ? scale * value[u].get(j) : wide_t<T>(0));
        }
        value[u].store(output + static_cast<size_t>(first + u) * columns + column);
    }
}

/// sum[j] += rows row[0], row[1], .. (outside [0, n_rows): none) at `column`.
template <typename T, int N>
__device__ __forceinline__ void add_batch(
    wide_t<T> (&sum)[N], const T* __restrict__ rows, const int32_t (&row)[AHEAD], int32_t n_rows, size_t columns,
    int32_t column
) {
    Piece<T, N> value[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; u++) {
        value[u] = Piece<T, N>::load(rows + (in_bounds(row[u], n_rows) ? row[u] : 0) * columns + column);
    }
#pragma unroll
    for (int u = 0; u < AHEAD; u++) {
        if (in_bounds(row[u], n_rows)) {
#pragma unroll
            for (int j = 0; j < N; j++) {
                sum[j] += value[u].get(j);
            }
        }
    }
}

/// sum[j] += rows order[begin], order[begin + step], ... before `end`, at `column`. The lanes of a team read the order
/// side by side and hand it round, so that a row waits for its place once per `team` rows, not each time.
template <typename T, int N>
__device__ __forceinline__ void add_rows(
    wide_t<T> (&sum)[N], const T* __restrict__ rows, const int32_t* __restrict__ order, int32_t n_rows, int32_t begin,
    int32_t end, int32_t step, size_t columns, int32_t column, int32_t team
) {
    int32_t row[AHEAD];
    if (team < AHEAD) {
        for (int32_t p = begin; p < end; p += AHEAD * step) {
#pragma unroll
            for (int u = 0; u < AHEAD; u++) {
                row[u] = p + u * step < end ? order[p + u * step] : -1;
            }
            add_batch<T, N>(sum, rows, row, n_rows, columns, column);
        }
        return;
    }
    const int32_t width = min(team, WAVE), lane = threadIdx.x & (width - 1);
    for (int32_t p = begin; p < end; p += width * step) {
        const int32_t left = min((end - p + step - 1) / step, width); // rows of this round
        const int32_t mine = lane < left ? order[p + lane * step] : -1;
        for (int32_t first = 0; first < left; first += AHEAD) {
#pragma unroll
            for (int u = 0; u < AHEAD; u++) {
                row[u] = __shfl(mine, first + u, width); // (lanes behind the last place have none; AHEAD divides width)
            }
            add_batch<T, N>(sum, rows, row, n_rows, columns, column);
        }
    }
}

/// sum[j] of all teams, in the registers of team 0. All threads. (Teams of a wavefront in six steps, the wavefronts one
/// after the other: 4096 rows, 64 table rows, 8 columns of float16: 15 us, with all 256 teams one after the other 36.)
template <typename W, int N> __device__ __forceinline__ void join_teams(W (&sum)[N], W* joined, const Teams& teams) {
    if (teams.teams == 1) {
        return;
    }
    for (int32_t step = teams.team; step < WAVE; step *= 2) {
#pragma unroll
        for (int j = 0; j < N; j++) {
            sum[j] += __shfl_xor(sum[j], step);
        }
    }
#pragma unroll
    for (int j = 0; j < N; j++) {
        joined[j * THREADS + threadIdx.x] = sum[j];
    }
    __syncthreads();
    if (static_cast<int32_t>(threadIdx.x) < teams.team) {
        for (int32_t t = max(teams.team, WAVE); t < THREADS; t += max(teams.team, WAVE)) {
#pragma unroll
            for (int j = 0; j < N; j++) {
                sum[j] += joined[j * THREADS + t + threadIdx.x];
            }
        }
    }
    __syncthreads();
}

/// partial[chunk, :] := the sum over the places of a chunk that lies inside one row of the table. Bound by memory where
/// there are chunks to sum up (rows of grad_output, read once), else by two dependent loads per workgroup.
template <typename T, int N>
__global__ __launch_bounds__(THREADS) void chunk_kernel(
    wide_t<T>* __restrict__ partial, const T* __restrict__ grad_output, const int32_t* __restrict__ indices,
    const int32_t* __restrict__ order, int32_t n_rows, int32_t table_rows, Teams teams, int32_t chunk
) {
    __shared__ wide_t<T> joined[N * THREADS];
    const int32_t begin = blockIdx.x * chunk, end = begin + chunk;
    const int32_t first = order[begin], last = order[end - 1];
    const int32_t index = in_bounds(first, n_rows) ? indices[first] : -1;
    if (!in_bounds(index, table_rows) || !in_bounds(last, n_rows) || indices[last] != index) {
        return; // (uniform)
    }
    const int32_t piece = min(
        static_cast<int32_t>(blockIdx.y * teams.team + (threadIdx.x & (teams.team - 1))), teams.row.pieces - 1
    );
    const int32_t column = teams.row.start<N>(piece);
    wide_t<T> sum[N] = {};
    add_rows<T, N>(
        sum, grad_output, order, n_rows, begin + threadIdx.x / teams.team, end, teams.teams, teams.row.columns, column,
        teams.team
    );
    join_teams<wide_t<T>, N>(sum, joined, teams);
    if (static_cast<int32_t>(threadIdx.x) < teams.team) {
        wide_t<T>* to = partial + static_cast<size_t>(blockIdx.x) * teams.row.columns + column;
#pragma unroll
        for (int j = 0; j < N; j++) {
            to[j] = sum[j];
        }
    }
}

/// The gradient's rows, as a workgroup makes them.
template <typename T, int N> struct TableRows {
    typedef wide_t<T> W;
    T* grad_table;
    const T* grad_output;
    const W* partial; // (null: none)
    const int32_t* order;
    int32_t n_rows, chunk;
    const Teams& teams;
    W scale;
    bool holds;     // the lane has a piece of the row
    int32_t column, mine;

    __device__ __forceinline__ TableRows(
        T* grad_table, const T* grad_output, const W* partial, const int32_t* order, int32_t n_rows, int32_t chunk,
        const Teams& teams, W scale
    ) : grad_table(grad_table), grad_output(grad_output), partial(partial), order(order), n_rows(n_rows), chunk(chunk),
        teams(teams), scale(scale) {
        const int32_t piece = blockIdx.y * teams.team + (threadIdx.x & (teams.team - 1));
        holds = piece < teams.row.pieces;
        column = teams.row.start<N>(min(piece, teams.row.pieces - 1));
        mine = threadIdx.x / teams.team;
    }

    __device__ __forceinline__ void store(int32_t row, const W (&sum)[N]) const {
        Piece<T, N> value;
#pragma unroll
        for (int j = 0; j < N; j++) {
            value.set(j, scale * sum[j]);
        }
        value.stream_to(grad_table + static_cast<size_t>(row) * teams.row.columns + column);
    }
    /// Row `row`, which has these places, by the team alone.
    __device__ __forceinline__ void by_team(int32_t row, Range places) const {
        W sum[N] = {};
        add_rows<T, N>(sum, grad_output, order, n_rows, places.begin, places.end, 1, teams.row.columns, column, teams.team);
        if (holds) {
            store(row, sum);
        }
    }
    /// The same by all teams of the workgroup, with the sums of the chunks that lie inside.
    __device__ __forceinline__ void by_all(W* joined, int32_t row, Range places) const {
        W sum[N] = {};
        const Range inside = chunks_inside(places, chunk);
        const bool chunks = partial != nullptr && inside.begin < inside.end;
        add_rows<T, N>(
            sum, grad_output, order, n_rows, places.begin + mine, chunks ? inside.begin * chunk : places.end,
            teams.teams, teams.row.columns, column, teams.team
        );
        if (chunks) {
            for (int32_t c = inside.begin + mine; c < inside.end; c += AHEAD * teams.teams) {
                W value[AHEAD][N];
#pragma unroll
                for (int u = 0; u < AHEAD; u++) {
                    const size_t from = min(c + u * teams.teams, inside.end - 1);
#pragma unroll
                    for (int j = 0; j < N; j++) {
                        value[u][j] = partial[from * teams.row.columns + column + j];
                    }
                }
#pragma unroll
                for (int u = 0; u < AHEAD; u++) {
                    if (c + u * teams.teams < inside.end) {
#pragma unroll
                        for (int j = 0; j < N; j++) {
                            sum[j] += value[u][j];
                        }
                    }
                }
            }
            add_rows<T, N>(
                sum, grad_output, order, n_rows, inside.end * chunk + mine, places.end, teams.teams,
                teams.row.columns, column, teams.team
            );
        }
        join_teams<W, N>(sum, joined, teams);
        if (mine == 0 && holds) {
            store(row, sum);
        }
    }
};

/// The gradient, bound by memory: grad_output is read once (chunks apart) and grad_table stored once, past the caches
/// (32 768 tokens of 100 003, 2048 bfloat16, with a plan: 94 us, 5.8 TB/s; through them the whole call took 173 us
/// instead of 137). ONE_EACH: a workgroup per row of the table. Else workgroups that have `each` rows of it, a team per row, and in front of
/// them ceil(n_rows / ALONE) others for the rows of more than ALONE places: the places of such a row include a multiple of
/// ALONE, and the workgroup of the first one makes it. (The most frequent ones are often neighbours. 44 721 rows of
/// 33 749, 223 columns, float16: 26 us with a plan; 72 where the workgroup that has them makes them one after the other.)
template <typename T, int N, bool ONE_EACH>
__global__ __launch_bounds__(THREADS) void gradient_kernel(
    T* __restrict__ grad_table, const T* __restrict__ grad_output, const wide_t<T>* __restrict__ partial,
    const int32_t* __restrict__ indices, const int32_t* __restrict__ order, const int32_t* __restrict__ offsets,
    int32_t n_rows, int32_t table_rows, Teams teams, int32_t chunk, int32_t each, wide_t<T> scale
) {
    __shared__ wide_t<T> joined[N * THREADS];
    const TableRows<T, N> rows(grad_table, grad_output, partial, order, n_rows, chunk, teams, scale);
    auto places_of = [&](int32_t row) { return places_between(offsets[row], offsets[row + 1], n_rows); };
    if (ONE_EACH) {
        const int32_t row = blockIdx.x;
        rows.by_all(joined, row, places_of(row));
        return;
    }
    const int32_t others = (n_rows + ALONE - 1) / ALONE, block = static_cast<int32_t>(blockIdx.x);
    if (block < others) {
        const int32_t place = block * ALONE, listed = order[place];
        const int32_t row = in_bounds(listed, n_rows) ? indices[listed] : -1;
        if (in_bounds(row, table_rows)) { // (uniform, like the next one)
            const Range places = places_of(row);
            if (places.end - places.begin > ALONE && chunks_inside(places, ALONE).begin == block) {
                rows.by_all(joined, row, places);
            }
        }
        return;
    }
    const int32_t row0 = (block - others) * each, row_end = min(row0 + each, table_rows);
    for (int32_t row = row0 + rows.mine; row < row_end; row += teams.teams) {
        const Range places = places_of(row);
        if (places.end - places.begin <= ALONE) {
            rows.by_team(row, places);
        }
    }
}

/// The same for at most THREADS rows, without an order in memory: every workgroup looks at all indices and puts the rows
/// that name its part of the table in order in LDS. One launch instead of three or four (24 rows, 16 table rows: 4.4 us,
/// 7.1 with the sort).
template <typename T, int N>
__global__ __launch_bounds__(THREADS) void few_rows_kernel(
    T* __restrict__ grad_table, const T* __restrict__ grad_output, const int32_t* __restrict__ indices, int32_t n_rows,
    int32_t table_rows, Teams teams, int32_t each, bool one_each, wide_t<T> scale
) {
    constexpr int WAVES = THREADS / WAVE;
    __shared__ wide_t<T> joined[N * THREADS];
    __shared__ int32_t places[TABLE_ROWS + 1], key[THREADS], order[THREADS], of_wave[WAVES];
    const int32_t row0 = blockIdx.x * each, row_end = min(row0 + each, table_rows), tid = threadIdx.x;
    for (int32_t i = tid; i <= each; i += THREADS) {
        places[i] = 0;
    }
    const int32_t index = tid < n_rows ? indices[tid] : -1;
    const bool here = index >= row0 && index < row_end;
    key[tid] = here ? index - row0 : -1;
    __syncthreads();
    if (here) {
        atomicAdd(&places[index - row0], 1);
    }
    __syncthreads();
    const int32_t listed = scan_in_place<WAVES>(places, each, 0, of_wave);
    if (tid == 0) {
        places[each] = listed;
    }
    if (here) { // (among the rows of the same index, in ascending order)
        int32_t place = places[index - row0];
        for (int32_t earlier = 0; earlier < tid; earlier++) {
            place += key[earlier] == index - row0 ? 1 : 0;
        }
        order[place] = tid;
    }
    __syncthreads();
    const TableRows<T, N> rows(grad_table, grad_output, nullptr, order, n_rows, 1, teams, scale);
    if (one_each) { // (uniform)
        rows.by_all(joined, row0, Range{places[0], places[1]});
        return;
    }
    for (int32_t row = row0 + rows.mine; row < row_end; row += teams.teams) {
        rows.by_team(row, Range{places[row - row0], places[row - row0 + 1]});
    }
}

/// body(number of columns in a piece): 16 bytes, or single numbers for rows shorter than that.
template <typename T, typename Body> void by_width(int32_t columns, Body&& body) {
    if (columns >= PIECE<T>) {
        body(std::integral_constant<int, PIECE<T>>{});
    } else {
        body(std::integral_constant<int, 1>{});
    }
}

template <typename T>
void lookup(T* output, const T* table, const int32_t* indices, int32_t n_rows, int32_t table_rows, int32_t columns,
            double scale, hipStream_t stream) {
    by_width<T>(columns, [&](auto width) {
        constexpr int N = decltype(width)::value;
        const Teams teams = Teams::make<N>(columns);
        auto launch = [&](auto rows) {
            constexpr int ROWS = decltype(rows)::value;
            const size_t blocks = ceil_div(static_cast<size_t>(n_rows), static_cast<size_t>(teams.teams) * ROWS);
            lookup_kernel<T, N, ROWS><<<dim3(static_cast<unsigned>(blocks), teams.tiles), THREADS, 0, stream>>>(
                output, table, indices, n_rows, table_rows, teams, static_cast<wide_t<T>>(scale)
            );
        };
        // several rows per lane once there are enough of them for every compute unit (200 000 rows of 128 floats: 17.2 us,
        // with one 18.9)
        if (static_cast<size_t>(n_rows) * teams.row.pieces >= static_cast<size_t>(compute_units()) * THREADS * 16) {
            launch(std::integral_constant<int, 4>{});
        } else {
            launch(std::integral_constant<int, 1>{});
        }
    });
    MOPS_HIP_CHECK(hipGetLastError());
}

template <typename T>
void gradient(
    T* grad_table, const T* grad_output, const int32_t* indices, const int32_t* order, const int32_t* offsets,
    int32_t n_rows, int32_t table_rows, int32_t columns, double scale, hipStream_t stream
) {
    by_width<T>(columns, [&](auto width) {
        constexpr int N = decltype(width)::value;
        const size_t units = static_cast<size_t>(compute_units());
        // Rows of the table per workgroup: one where many rows name each on average (200 000 rows, 94 table rows, 128
        // floats: 32 us for the whole gradient, with a row per team 37; 4096 rows, 64 of 8 numbers: 15 and 19), else some per team if there are enough of them,
        // for workgroups that have nothing but zeros to store come and go faster than they are started.
        const bool many = static_cast<size_t>(n_rows) > static_cast<size_t>(table_rows) * FEW;
        const Teams teams = Teams::make<N>(columns);
        auto rows_each = [&](const Teams& t) {
            const size_t by_team = static_cast<size_t>(table_rows) * t.tiles / t.teams;
            return many ? size_t(1)
                        : std::min<size_t>(t.teams * std::clamp<size_t>(by_team / (8 * units), 1, ROWS_PER_TEAM), TABLE_ROWS);
        };
        // few workgroups: fewer columns in each of more
        Teams summing = teams;
        while (many && summing.team > 8 && static_cast<size_t>(table_rows) * summing.tiles < units) {
            summing = Teams::make<N>(columns, summing.team / 2);
        }
        const size_t each = rows_each(summing);
        const dim3 grid(static_cast<unsigned>(ceil_div(static_cast<size_t>(table_rows), each)), summing.tiles);
        if (n_rows <= THREADS) { // (also where the caller has a plan: reading it would take longer)
            few_rows_kernel<T, N><<<grid, THREADS, 0, stream>>>(
                grad_table, grad_output, indices, n_rows, table_rows, summing, static_cast<int32_t>(each), many,
                static_cast<wide_t<T>>(scale)
            );
            return;
        }
        const int32_t chunk = std::min<int32_t>(
            PLACES_EACH * teams.teams,
            static_cast<int32_t>(ceil_div(static_cast<size_t>(n_rows), CHUNKS * CHUNK_PLACES)) * CHUNK_PLACES
        );
        const int32_t chunks = n_rows / std::max(chunk, 1);
        const size_t partial_bytes =
            n_rows > ALONE ? align256(static_cast<size_t>(chunks) * columns * sizeof(wide_t<T>)) : 0;
        const size_t order_bytes = order == nullptr ? align256(static_cast<size_t>(n_rows) * 4) : 0;
        const size_t offsets_bytes = order == nullptr ? align256((static_cast<size_t>(table_rows) + 1) * 4) : 0;
        const size_t sort_bytes = order == nullptr ? order_all_by_group_bytes(table_rows, n_rows) : 0;
        char* workspace = nullptr;
        if (partial_bytes + order_bytes + offsets_bytes + sort_bytes > 0) {
            workspace = static_cast<char*>(scratch(partial_bytes + order_bytes + offsets_bytes + sort_bytes));
        }
        wide_t<T>* partial = partial_bytes > 0 ? reinterpret_cast<wide_t<T>*>(workspace) : nullptr;
        if (order == nullptr) {
            int32_t* places = reinterpret_cast<int32_t*>(workspace + partial_bytes);
            int32_t* begins = reinterpret_cast<int32_t*>(workspace + partial_bytes + order_bytes);
            order_all_by_group(
                places, begins, indices, n_rows, table_rows, workspace + partial_bytes + order_bytes + offsets_bytes,
                stream
            );
            order = places;
            offsets = begins;
        }
        if (partial != nullptr) {
            chunk_kernel<T, N><<<dim3(static_cast<unsigned>(chunks), teams.tiles), THREADS, 0, stream>>>(
                partial, grad_output, indices, order, n_rows, table_rows, teams, chunk
            );
        }
        auto launch = [&](auto one_each, dim3 workgroups) {
            gradient_kernel<T, N, decltype(one_each)::value><<<workgroups, THREADS, 0, stream>>>(
                grad_table, grad_output, partial, indices, order, offsets, n_rows, table_rows, summing, chunk,
                static_cast<int32_t>(each), static_cast<wide_t<T>>(scale)
            );
        };
        if (many) {
            launch(std::true_type{}, grid);
        } else {
            launch(std::false_type{}, dim3(grid.x + static_cast<unsigned>(ceil_div(n_rows, ALONE)), grid.y));
        }
    });
    MOPS_HIP_CHECK(hipGetLastError());
}

} // namespace
} // namespace embedding
} // namespace mops::amd

namespace mops::cuda {

using namespace mops::amd;

void order_by_group(Tensor<int32_t, 1> order, Tensor<int32_t, 1> offsets, Tensor<int32_t, 1> indices) {
    const checks::Validator check("order_by_group");
    check.same_extent(checks::axis_of(order, "order", 0), checks::axis_of(indices, "indices", 0));
    if (offsets.shape[0] < 1) {
        throw std::runtime_error("offsets must have at least one element in order_by_group");
    }
    const int32_t n_rows = count_i32(indices.shape[0], "number of rows");
    const int32_t groups = count_i32(offsets.shape[0], "number of groups + 1") - 1;
    const size_t bytes = n_rows > 0 ? order_all_by_group_bytes(groups, n_rows) : 0;
    void* workspace = bytes > 0 ? scratch(bytes) : nullptr;
    order_all_by_group(order.data, offsets.data, indices.data, n_rows, groups, workspace, current_stream());
    finish_call("order_by_group");
}

template <typename scalar_t>
void scaled_embedding(
    Tensor<scalar_t, 2> output, Tensor<scalar_t, 2> table, Tensor<int32_t, 1> indices, double scale
) {
    const checks::Validator check("scaled_embedding");
    check.same_extent(checks::axis_of(output, "output", 0), checks::axis_of(indices, "indices", 0));
    check.same_extent(checks::axis_of(output, "output", 1), checks::axis_of(table, "table", 1));
    const int32_t n_rows = count_i32(indices.shape[0], "number of rows");
    const int32_t table_rows = count_i32(table.shape[0], "number of table rows");
    const int32_t columns = count_i32(table.shape[1], "number of columns");
    if (n_rows > 0 && columns > 0) {
        typedef device_t<scalar_t> T;
        T* to = data_of(output);
        if (table_rows > 0) {
            embedding::lookup<T>(
                to, data_of(table), indices.data, n_rows, table_rows, columns, scale,
                current_stream()
            );
        } else { // (no row to look anything up in: every index is outside; `to` is never read as a table)
            embedding::lookup<T>(to, to, indices.data, n_rows, 0, columns, scale, current_stream());
        }
    }
    finish_call("scaled_embedding");
}

template <typename scalar_t>
void scaled_embedding_vjp(
    Tensor<scalar_t, 2> grad_table, Tensor<scalar_t, 2> grad_output, Tensor<int32_t, 1> indices,
    Tensor<int32_t, 1> order, Tensor<int32_t, 1> offsets, double scale
) {
    if (grad_table.data == nullptr) {
        return;
    }
    const checks::Validator check("scaled_embedding_vjp");
    check.same_extent(checks::axis_of(grad_output, "grad_output", 0), checks::axis_of(indices, "indices", 0));
    check.same_extent(checks::axis_of(grad_output, "grad_output", 1), checks::axis_of(grad_table, "grad_table", 1));
    const int32_t n_rows = count_i32(indices.shape[0], "number of rows");
    const int32_t table_rows = count_i32(grad_table.shape[0], "number of table rows");
    const int32_t columns = count_i32(grad_table.shape[1], "number of columns");
    if ((order.data == nullptr) != (offsets.data == nullptr) && n_rows > 0) {
        throw std::runtime_error("order and offsets must be given together in scaled_embedding_vjp");
    }
    if (order.data != nullptr) {
        check.same_extent(checks::axis_of(order, "order", 0), checks::axis_of(indices, "indices", 0));
        if (offsets.shape[0] != grad_table.shape[0] + 1) {
            throw std::runtime_error(
                "offsets must have " + std::to_string(grad_table.shape[0] + 1) + " elements (the rows of the table "
                "and one more) in scaled_embedding_vjp, got " + std::to_string(offsets.shape[0])
            );
        }
    }
    if (table_rows > 0 && columns > 0) {
        typedef device_t<scalar_t> T;
        embedding::gradient<T>(
            data_of(grad_table), data_of(grad_output), indices.data,
            order.data, offsets.data, n_rows, table_rows, columns, scale, current_stream()
        );
    }
    finish_call("scaled_embedding_vjp");
}

#define MOPS_EMBEDDING_INSTANTIATE(T)                                                              \
    template void scaled_embedding<T>(Tensor<T, 2>, Tensor<T, 2>, Tensor<int32_t, 1>, double);     \
    template void scaled_embedding_vjp<T>(                                                         \
        Tensor<T, 2>, Tensor<T, 2>, Tensor<int32_t, 1>, Tensor<int32_t, 1>, Tensor<int32_t, 1>, double \
    );
MOPS_EMBEDDING_INSTANTIATE(float)
MOPS_EMBEDDING_INSTANTIATE(double)
MOPS_EMBEDDING_INSTANTIATE(bfloat16)
MOPS_EMBEDDING_INSTANTIATE(float16)

} // namespace mops::cuda
