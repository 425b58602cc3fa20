// Tiles of products over groups of rows, on the matrix cores: the kernel behind
// grouped_product.hip, for all element types.
//
// A workgroup makes BM x BN numbers of a result, sum_k q(m, k) p(n, k): the "q"
// side is what the result's rows come from, the "p" side what its columns come
// from. It is computed as (p q^T), so that a lane holds consecutive COLUMNS of a
// row of the result and stores them as one piece.
//
//   form      result                     q(m, k)             p(n, k)
//   FORWARD   output[r, :], k over K     A[r, k]             W[g, k, n]
//   GRAD_ROWS grad_A[r, :], k over L     grad_output[r, k]   W[g, n, k]
//   GRAD_SUMS grad_W[g, m, :], k over    A[row k, m]         grad_output[row k, n]
//             the rows of the group
//
// A side goes through LDS in steps of 128 bytes of k (64 numbers of 16 bits, 32
// of 32, 16 of 64), double-buffered: while a step is multiplied, the next one is
// on its way to registers, and goes to the other buffer when it has arrived; one
// barrier per step. A side whose k is contiguous in memory ("straight") lies in
// LDS as it is read by the matrix instructions, [outer][k], in pieces of 16
// bytes that are permuted within a row so that the rows of a block fall into
// different banks. A side whose k is the row of memory ("turned") lies in LDS as
// [k][outer]; 16-bit numbers are turned by the LDS's transposing reads, wider
// ones are read one by one. Pieces of memory are loaded at any alignment; what
// lies outside a side in the direction of k is zero in LDS (never a value from
// somewhere else: 0 x infinity is not 0), what lies outside in the other
// direction is not stored.
#ifndef MOPS_AMD_GROUPED_TILES_HPP
#define MOPS_AMD_GROUPED_TILES_HPP

#include <cstdint>
#include <type_traits>

#include <hip/hip_runtime.h>

#include "device_common.hpp"
#include "group_units.hpp"
#include "numbers.hpp"

namespace mops::amd::grouped_product {

enum class Form { FORWARD, GRAD_ROWS, GRAD_SUMS };

/// The operands of a launch. FORWARD and GRAD_ROWS: q is [rows][k_size], p the matrices of all groups; GRAD_SUMS: q is
/// [rows][m_size], p is [rows][n_size].
template <typename T> struct Product {
    T* out;
    wide_t<T>* partial; // GRAD_SUMS: [unit][m_size][n_size], for groups of more than one unit
    const T *q, *p;
    RowGroups groups;
    int32_t m_size, n_size, k_size;
    int32_t step;            // places per unit
    int32_t most_units;      // that the grid and `partial` have room for (offsets that are none could give more)
    int32_t m_tiles, n_tiles; // tiles of a unit (m_tiles: GRAD_SUMS)
};

/// The matrix instructions of a type: blocks of BLOCK x BLOCK, and a piece of 16 bytes of k per lane and side: lane l
/// has row l % BLOCK of the block, numbers (l / BLOCK) * COUNT + (0 .. COUNT - 1) of the k of one multiplication.
/// Lane l, number i of the result: column l % BLOCK (of q's side), row row_of(l, i) (of p's side).
template <typename T> struct Matrix;

template <> struct Matrix<__bf16> {
    static constexpr int BLOCK = 32, COUNT = 8, HELD = 16;
    typedef __bf16 Numbers __attribute__((ext_vector_type(8)));
    typedef float Sums __attribute__((ext_vector_type(16)));
    static __device__ __forceinline__ Sums multiply(Numbers p, Numbers q, Sums sums) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(p, q, sums, 0, 0, 0);
    }
    static __device__ __forceinline__ int row_of(int lane, int i) { return 8 * (i / 4) + 4 * (lane / 32) + i % 4; }
    static constexpr int RUN = 4; // numbers i, i + 1, .. that are consecutive rows
};
template <> struct Matrix<_Float16> {
    static constexpr int BLOCK = 32, COUNT = 8, HELD = 16;
    typedef _Float16 Numbers __attribute__((ext_vector_type(8)));
    typedef float Sums __attribute__((ext_vector_type(16)));
    static __device__ __forceinline__ Sums multiply(Numbers p, Numbers q, Sums sums) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(p, q, sums, 0, 0, 0);
    }
    static __device__ __forceinline__ int row_of(int lane, int i) { return 8 * (i / 4) + 4 * (lane / 32) + i % 4; }
    static constexpr int RUN = 4;
};
template <> struct Matrix<float> {
    static constexpr int BLOCK = 32, COUNT = 4, HELD = 16;
    typedef float Numbers __attribute__((ext_vector_type(4)));
    typedef float Sums __attribute__((ext_vector_type(16)));
    static __device__ __forceinline__ Sums multiply(Numbers p, Numbers q, Sums sums) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            sums = __builtin_amdgcn_mfma_f32_32x32x2f32(p[i], q[i], sums, 0, 0, 0);
        }
        return sums;
    }
    static __device__ __forceinline__ int row_of(int lane, int i) { return 8 * (i / 4) + 4 * (lane / 32) + i % 4; }
    static constexpr int RUN = 4;
};
template <> struct Matrix<double> {
    static constexpr int BLOCK = 16, COUNT = 2, HELD = 4;
    typedef double Numbers __attribute__((ext_vector_type(2)));
    typedef double Sums __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ Sums multiply(Numbers p, Numbers q, Sums sums) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            sums = __builtin_amdgcn_mfma_f64_16x16x4f64(p[i], q[i], sums, 0, 0, 0);
        }
        return sums;
    }
    static __device__ __forceinline__ int row_of(int lane, int i) { return 4 * i + lane / 16; }
    static constexpr int RUN = 1;
};

constexpr int PIECES_OF_STEP = 8; // pieces of 16 bytes of k in LDS

template <typename T> using Numbers = typename Matrix<T>::Numbers;

/// The first `count` of a piece's numbers, zeros behind them (count may be negative, or beyond the piece).
template <typename T> __device__ __forceinline__ Numbers<T> load_numbers(const T* from, int32_t count) {
    constexpr int COUNT = Matrix<T>::COUNT;
    Numbers<T> v;
    if (count >= COUNT) {
        typedef T Anywhere __attribute__((ext_vector_type(COUNT), aligned(sizeof(T))));
        const Anywhere a = *reinterpret_cast<const Anywhere*>(from);
#pragma unroll
        for (int i = 0; i < COUNT; i++) {
            v[i] = a[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < COUNT; i++) {
            v[i] = i < count ? from[i] : static_cast<T>(0.f);
        }
    }
    return v;
}

/// LDS of a straight side of OUTER rows: [OUTER][8 pieces].
template <typename T, int OUTER> struct Straight {
    static __device__ __forceinline__ int place(int row, int piece) {
        return (row * PIECES_OF_STEP + (piece ^ (row >> 1 & 7))) * 16;
    }
    /// Numbers `step` of the k of a block that begins at row `outer0`.
    static __device__ __forceinline__ Numbers<T> read(const char* lds, int outer0, int step, int lane) {
        constexpr int BLOCK = Matrix<T>::BLOCK;
        const int row = outer0 + lane % BLOCK, piece = step * (WAVE / BLOCK) + lane / BLOCK;
        return *reinterpret_cast<const Numbers<T>*>(lds + place(row, piece));
    }
};

/// LDS of a turned side: [k][OUTER numbers], 16-byte pieces of a row permuted so that the four rows that the lanes of
/// a transposing read look at fall into different banks.
template <typename T, int OUTER> struct Turned {
    static constexpr int PIECES = OUTER / Matrix<T>::COUNT; // of a row of k
    static __device__ __forceinline__ int place(int k, int piece) {
        int at = piece;
        if constexpr (sizeof(T) == 2 && PIECES >= 16) {
            at = piece ^ (k & 3) << 2;
        } else if constexpr (sizeof(T) == 2 && PIECES == 8) {
            at = piece ^ (k >> 1 & 1) << 2;
        }
        return (k * PIECES + at) * 16;
    }
    static __device__ __forceinline__ Numbers<T> read(const char* lds, int outer0, int step, int lane) {
        constexpr int BLOCK = Matrix<T>::BLOCK, COUNT = Matrix<T>::COUNT;
        const int k0 = (step * (WAVE / BLOCK) + lane / BLOCK) * COUNT;
        Numbers<T> v;
        if constexpr (sizeof(T) == 2) {
            // 16 lanes name four rows of four times four numbers; lane i gets column i of the sixteen
            typedef short Turning __attribute__((ext_vector_type(4)));
            const int in16 = lane % 16, outer = outer0 + (lane / 16 % 2) * 16 + in16 % 4 * 4, k = k0 + in16 / 4;
            const int half = outer / 4 % 2 * 8;
            union {
                Turning turned[2];
                Numbers<T> numbers;
            } both;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                both.turned[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) Turning*)(lds + place(k + 4 * i, outer / 8) + half)
                );
            }
            v = both.numbers;
        } else {
            const int outer = outer0 + lane % BLOCK;
#pragma unroll
            for (int i = 0; i < COUNT; i++) {
                v[i] = reinterpret_cast<const T*>(lds + place(k0 + i, outer / COUNT))[outer % COUNT];
            }
        }
        return v;
    }
};

/// A straight side on its way to LDS: THREADS threads, OUTER rows.
template <typename T, int OUTER, int THREADS> struct StraightLoader {
    typedef Straight<T, OUTER> Layout;
    static constexpr int EACH = OUTER * PIECES_OF_STEP / THREADS, COUNT = Matrix<T>::COUNT;
    const T* from[EACH];
    Numbers<T> piece[EACH];
    int32_t k_size;

    static __device__ __forceinline__ int row(int j) { return (threadIdx.x + j * THREADS) / PIECES_OF_STEP; }
    static __device__ __forceinline__ int of_row(int j) { return (threadIdx.x + j * THREADS) % PIECES_OF_STEP; }

    /// row_at(i): pointer to the row of memory behind row i of the side
    template <typename RowAt> __device__ __forceinline__ void begin(int32_t k, RowAt&& row_at) {
        k_size = k;
#pragma unroll
        for (int j = 0; j < EACH; j++) {
            from[j] = row_at(row(j)) + of_row(j) * COUNT;
        }
    }
    __device__ __forceinline__ void load(int32_t k0) {
#pragma unroll
        for (int j = 0; j < EACH; j++) {
            piece[j] = load_numbers<T>(from[j] + k0, k_size - k0 - of_row(j) * COUNT);
        }
    }
    __device__ __forceinline__ void store(char* lds) const {
#pragma unroll
        for (int j = 0; j < EACH; j++) {
            *reinterpret_cast<Numbers<T>*>(lds + Layout::place(row(j), of_row(j))) = piece[j];
        }
    }
};

/// A turned side: rows of `width` numbers, of which those from outer0 on are used.
template <typename T, int OUTER, int THREADS> struct TurnedLoader {
    typedef Turned<T, OUTER> Layout;
    static constexpr int EACH = OUTER * PIECES_OF_STEP / THREADS, COUNT = Matrix<T>::COUNT;
    Numbers<T> piece[EACH];
    const T* from;
    int32_t width, outer0;

    static __device__ __forceinline__ int k(int j) { return (threadIdx.x + j * THREADS) / Layout::PIECES; }
    static __device__ __forceinline__ int of_row(int j) { return (threadIdx.x + j * THREADS) % Layout::PIECES; }

    __device__ __forceinline__ void begin(const T* memory, int32_t row_width, int32_t first) {
        from = memory;
        width = row_width;
        outer0 = first;
    }
    /// row_at(k): the row of memory, negative: none
    template <typename RowAt> __device__ __forceinline__ void load(RowAt&& row_at) {
#pragma unroll
        for (int j = 0; j < EACH; j++) {
            const int32_t row = row_at(k(j));
            const int32_t outer = outer0 + of_row(j) * COUNT;
            const size_t at = static_cast<size_t>(max(row, 0)) * width + outer;
            piece[j] = load_numbers<T>(from + at, row < 0 ? 0 : width - outer);
        }
    }
    __device__ __forceinline__ void store(char* lds) const {
#pragma unroll
        for (int j = 0; j < EACH; j++) {
            *reinterpret_cast<Numbers<T>*>(lds + Layout::place(k(j), of_row(j))) = piece[j];
        }
    }
};

/// WM x WN wavefronts; every one of them makes BM / WM x BN / WN numbers.
template <typename T, Form FORM, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM* WN* WAVE) void tiles_kernel(Product<T> g) {
    typedef Matrix<T> M;
    constexpr int THREADS = WM * WN * WAVE, COUNT = M::COUNT, BLOCK = M::BLOCK;
    constexpr int STEP = PIECES_OF_STEP * COUNT, STEPS = PIECES_OF_STEP * BLOCK / WAVE;
    constexpr int MB = BM / WM / BLOCK, NB = BN / WN / BLOCK; // blocks of a wavefront
    constexpr bool SUMS = FORM == Form::GRAD_SUMS, Q_TURNED = SUMS, P_TURNED = FORM != Form::GRAD_ROWS;
    constexpr Units UNITS = SUMS ? Units::OF_GROUPS : Units::OF_ROWS;
    using QLoader = std::conditional_t<Q_TURNED, TurnedLoader<T, BM, THREADS>, StraightLoader<T, BM, THREADS>>;
    using PLoader = std::conditional_t<P_TURNED, TurnedLoader<T, BN, THREADS>, StraightLoader<T, BN, THREADS>>;
    constexpr int BYTES = (BM + BN) * PIECES_OF_STEP * 16;
    __shared__ __attribute__((aligned(16))) char lds[2 * BYTES];
    __shared__ int32_t rows[SUMS ? 1 : BM];

    // Workgroups b, b + 8, .. run on the same XCD: each XCD gets consecutive tiles, so that its L2 holds what they share.
    const int32_t tiles_of_unit = (SUMS ? g.m_tiles : 1) * g.n_tiles;
    const int32_t units = min(count_units<UNITS>(g.groups, g.step), g.most_units);
    const int64_t tiles = static_cast<int64_t>(units) * tiles_of_unit;
    const int32_t per_xcd = static_cast<int32_t>((tiles + 7) / 8);
    const int64_t tile = static_cast<int64_t>(blockIdx.x % 8) * per_xcd + blockIdx.x / 8;
    if (static_cast<int32_t>(blockIdx.x / 8) >= per_xcd || tile >= tiles) {
        return; // (uniform)
    }
    int32_t unit_index, m0, n0;
    if (SUMS) {
        unit_index = static_cast<int32_t>(tile / tiles_of_unit);
        const int32_t of_unit = static_cast<int32_t>(tile % tiles_of_unit);
        m0 = of_unit / g.n_tiles * BM;
        n0 = of_unit % g.n_tiles * BN;
    } else {
        // bands of four units: their rows and a tile's columns of the matrix are read together
        const int32_t band = static_cast<int32_t>(tile / (4 * g.n_tiles)), in_band = static_cast<int32_t>(tile % (4 * g.n_tiles));
        const int32_t height = min(4, units - 4 * band);
        unit_index = 4 * band + in_band % height;
        m0 = 0;
        n0 = in_band / height * BN;
    }
    const GroupUnit unit = find_unit<UNITS>(g.groups, g.step, unit_index);
    if (unit.group < 0) {
        return; // (uniform; offsets that are none)
    }
    const bool rest = !SUMS && unit.group == g.groups.n_groups;
    if constexpr (!SUMS) {
        for (int i = threadIdx.x; i < BM; i += THREADS) {
            const int32_t at = min(i, unit.count - 1);
            rows[i] = g.groups.row_at(rest ? place_of_rest(g.groups, unit.begin + at) : unit.begin + at);
        }
        __syncthreads();
    }

    const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
    const int wave_m = wave / WN * (BM / WM), wave_n = wave % WN * (BN / WN);
    typename M::Sums sums[MB][NB];
#pragma unroll
    for (int i = 0; i < MB; i++) {
#pragma unroll
        for (int j = 0; j < NB; j++) {
#pragma unroll
            for (int e = 0; e < M::HELD; e++) {
                sums[i][j][e] = 0;
            }
        }
    }

    const int32_t k_size = rest ? 0 : SUMS ? unit.count : g.k_size;
    if (k_size > 0) {
        QLoader q;
        PLoader p;
        if constexpr (Q_TURNED) {
            q.begin(g.q, g.m_size, m0);
        } else {
            q.begin(k_size, [&](int i) { return g.q + static_cast<size_t>(rows[i]) * g.k_size; });
        }
        const size_t of_group = static_cast<size_t>(unit.group) * g.k_size * g.n_size;
        if constexpr (SUMS) {
            p.begin(g.p, g.n_size, n0);
        } else if constexpr (P_TURNED) {
            p.begin(g.p + of_group, g.n_size, n0);
        } else {
            p.begin(k_size, [&](int i) { return g.p + of_group + static_cast<size_t>(min(n0 + i, g.n_size - 1)) * g.k_size; });
        }
        auto load = [&](int32_t k0) {
            if constexpr (SUMS) {
                auto row_at = [&](int k) { return k0 + k < k_size ? g.groups.row_at(unit.begin + k0 + k) : -1; };
                q.load(row_at);
                p.load(row_at);
            } else {
                q.load(k0);
                if constexpr (P_TURNED) {
                    p.load([&](int k) { return k0 + k < k_size ? k0 + k : -1; });
                } else {
                    p.load(k0);
                }
            }
        };
        load(0);
        char* buffer = lds;
        q.store(buffer);
        p.store(buffer + BM * PIECES_OF_STEP * 16);
        __syncthreads();
        for (int32_t k0 = 0; k0 < k_size; k0 += STEP) {
            const bool more = k0 + STEP < k_size; // (uniform)
            if (more) {
                load(k0 + STEP);
            }
#pragma unroll
            for (int step = 0; step < STEPS; step++) {
                Numbers<T> of_q[MB], of_p[NB];
#pragma unroll
                for (int i = 0; i < MB; i++) {
                    of_q[i] = QLoader::Layout::read(buffer, wave_m + i * BLOCK, step, lane);
                }
#pragma unroll
                for (int j = 0; j < NB; j++) {
                    of_p[j] = PLoader::Layout::read(buffer + BM * PIECES_OF_STEP * 16, wave_n + j * BLOCK, step, lane);
                }
#pragma unroll
                for (int i = 0; i < MB; i++) {
#pragma unroll
                    for (int j = 0; j < NB; j++) {
                        sums[i][j] = M::multiply(of_p[j], of_q[i], sums[i][j]);
                    }
                }
            }
            if (more) {
                buffer = lds + (buffer == lds ? BYTES : 0);
                q.store(buffer);
                p.store(buffer + BM * PIECES_OF_STEP * 16);
                __syncthreads();
            }
        }
    }

    // lane l has column wave_m + i * BLOCK + l % BLOCK of the tile's transpose, RUN consecutive numbers at a time
    constexpr int RUN = M::RUN;
    auto store = [&](auto* row, int j, int i, auto zero) {
        typedef decltype(zero) To;
        typedef To Run __attribute__((ext_vector_type(RUN), aligned(sizeof(To))));
#pragma unroll
        for (int e = 0; e < M::HELD; e += RUN) {
            const int32_t n = n0 + wave_n + j * BLOCK + M::row_of(lane, e);
            if (n + RUN <= g.n_size) {
                Run run;
#pragma unroll
                for (int r = 0; r < RUN; r++) {
                    run[r] = static_cast<To>(sums[i][j][e + r]);
                }
                *reinterpret_cast<Run*>(row + n) = run;
            } else {
#pragma unroll
                for (int r = 0; r < RUN; r++) {
                    if (n + r < g.n_size) {
                        row[n + r] = static_cast<To>(sums[i][j][e + r]);
                    }
                }
            }
        }
    };
#pragma unroll
    for (int i = 0; i < MB; i++) {
        const int32_t m = wave_m + i * BLOCK + lane % BLOCK;
        if constexpr (SUMS) {
            if (m0 + m < g.m_size) {
                const size_t of_unit = static_cast<size_t>(m0 + m) * g.n_size;
                const size_t size = static_cast<size_t>(g.m_size) * g.n_size;
#pragma unroll
                for (int j = 0; j < NB; j++) {
                    if (unit.of_group > 1) {
                        store(g.partial + unit_index * size + of_unit, j, i, wide_t<T>());
                    } else {
                        store(g.out + unit.group * size + of_unit, j, i, T());
                    }
                }
            }
        } else if (m < unit.count) {
#pragma unroll
            for (int j = 0; j < NB; j++) {
                store(g.out + static_cast<size_t>(rows[m]) * g.n_size, j, i, T());
            }
        }
    }
}

/// out[g, :] := the sum of its units' partial results, for groups of more than one unit.
constexpr int JOIN_THREADS = 256;
template <typename T> __global__ __launch_bounds__(JOIN_THREADS) void join_units_kernel(Product<T> g) {
    const int32_t first = static_cast<int32_t>(blockIdx.x);
    const GroupUnit unit = find_unit<Units::OF_GROUPS>(g.groups, g.step, first);
    if (unit.group < 0 || unit.of_group < 2 || unit.index != 0) {
        return; // (uniform)
    }
    const int32_t parts = min(unit.of_group, g.most_units - first);
    const size_t size = static_cast<size_t>(g.m_size) * g.n_size;
    const wide_t<T>* from = g.partial + first * size;
    for (size_t i = blockIdx.y * static_cast<size_t>(JOIN_THREADS) + threadIdx.x; i < size;
         i += static_cast<size_t>(gridDim.y) * JOIN_THREADS) {
        wide_t<T> sum = 0;
#pragma unroll 8
        for (int32_t u = 0; u < parts; u++) {
            sum += from[u * size + i];
        }
        g.out[unit.group * size + i] = static_cast<T>(sum);
    }
}

} // namespace mops::amd::grouped_product

#endif
