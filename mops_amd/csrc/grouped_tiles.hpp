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
// of 32, 16 of 64), double-buffered. A side whose k is contiguous in memory
// ("straight") lies in LDS as it is read by the matrix instructions,
// [outer][k], in pieces of 16 bytes that are permuted within a row so that the
// rows of a block fall into different banks. A side whose k is the row of memory
// ("turned") lies in LDS as [k][outer]; 16-bit numbers are turned by the LDS's
// transposing reads, wider ones are read one by one. Either way piece i of a
// buffer is the business of thread i (i + THREADS, ..), so that a piece can go
// from memory to LDS without a register (ALIGNED: rows that begin on 16-byte
// boundaries, in which a piece is inside a row or outside as a whole), or
// through registers (rows of any length, pieces at any alignment). What lies
// outside a side in the direction of k is zero in LDS (never a value from
// somewhere else: 0 x infinity is not 0); what lies outside in the other
// direction is not stored.
//
// The numbers of a multiplication are read from LDS while the one before runs.
// In front of the last multiplication of a step, whose numbers are in registers
// by then, the workgroup meets: the step's buffer is free for the step after
// the next, the next step's has arrived. So there is one barrier per step, and
// nothing waits for LDS or memory behind it.
//
// Large products are bound by the matrix units (and, in 16 bits, by the clock
// that the power of random numbers leaves): one group of 8192 rows, K = L =
// 8192: bfloat16 1040 to 1170 TFLOP/s, float 130, double 65; K = L = 2048 1080
// (float16), at odd addresses, with the copy, 750. Tiles of 128 read memory and
// LDS twice as often for the same work: 890 there. Few rows are bound by the
// matrices' bytes: 24 rows, 16 experts of 2048 x 1408 bfloat16, 15.8 us, 5.8 TB/s.
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

/// Rows in memory: `stride` numbers from one to the next, their width or as much as whole pieces take.
template <typename T> struct Operand {
    const T* data;
    int32_t stride;
};

/// The operands of a launch. FORWARD and GRAD_ROWS: q is [rows][k_size], p the matrices of all groups; GRAD_SUMS: q is
/// [rows][m_size], p is [rows][n_size].
template <typename T> struct Product {
    T* out;
    // GRAD_SUMS: [slot][partial_size(m_size, n_size)], for the units of groups of more than one; else [split][row][n_size], where
    // there are several
    wide_t<T>* partial;
    Operand<T> q, p;
    bool in_place; // all rows begin on 16-byte boundaries and have whole pieces, with zeros behind their numbers
    RowGroups groups;
    int32_t m_size, n_size, k_size;
    int32_t step;            // places per unit
    int32_t most_units;      // that the grid has room for (offsets that are none could give more)
    int32_t most_slots;      // GRAD_SUMS: that `partial` has room for (likewise)
    int32_t m_tiles, n_tiles; // tiles of a unit (m_tiles: GRAD_SUMS)
    int32_t splits, k_each;   // FORWARD, GRAD_ROWS: shares of k, and how long they are (whole steps)
};

/// Numbers from one unit's partial result to the next: whole pieces of four.
__host__ __device__ __forceinline__ size_t partial_size(int32_t m_size, int32_t n_size) {
    return (static_cast<size_t>(m_size) * n_size + 3) / 4 * 4;
}

/// The matrix instructions of a type: blocks of BLOCK x BLOCK, and a piece of 16 bytes of k per lane and side: lane l
/// has row l % BLOCK of the block, numbers (l / BLOCK) * COUNT + (0 .. COUNT - 1) of the k of one multiplication.
/// PARTS instructions make up the multiplication. Lane l, number i of the result: column l % BLOCK (of q's side), row row_of(l, i) (of p's side).
template <typename T> struct Matrix;

template <> struct Matrix<__bf16> {
    static constexpr int BLOCK = 32, COUNT = 8, HELD = 16;
    typedef __bf16 Numbers __attribute__((ext_vector_type(8)));
    typedef float Sums __attribute__((ext_vector_type(16)));
    static constexpr int PARTS = 1;
    static __device__ __forceinline__ Sums multiply(int, Numbers p, Numbers q, Sums sums) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(p, q, sums, 0, 0, 0);
    }
    static __device__ __forceinline__ int row_of(int lane, int i) { return 8 * (i / 4) + 4 * (lane / 32) + i % 4; }
    static constexpr int RUN = 4; // numbers i, i + 1, .. that are consecutive rows
};
template <> struct Matrix<_Float16> {
    static constexpr int BLOCK = 32, COUNT = 8, HELD = 16;
    typedef _Float16 Numbers __attribute__((ext_vector_type(8)));
    typedef float Sums __attribute__((ext_vector_type(16)));
    static constexpr int PARTS = 1;
    static __device__ __forceinline__ Sums multiply(int, Numbers p, Numbers q, Sums sums) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(p, q, sums, 0, 0, 0);
    }
    static __device__ __forceinline__ int row_of(int lane, int i) { return 8 * (i / 4) + 4 * (lane / 32) + i % 4; }
    static constexpr int RUN = 4;
};
template <> struct Matrix<float> {
    static constexpr int BLOCK = 32, COUNT = 4, HELD = 16;
    typedef float Numbers __attribute__((ext_vector_type(4)));
    typedef float Sums __attribute__((ext_vector_type(16)));
    static constexpr int PARTS = 4;
    static __device__ __forceinline__ Sums multiply(int part, Numbers p, Numbers q, Sums sums) {
        return __builtin_amdgcn_mfma_f32_32x32x2f32(p[part], q[part], sums, 0, 0, 0);
    }
    static __device__ __forceinline__ int row_of(int lane, int i) { return 8 * (i / 4) + 4 * (lane / 32) + i % 4; }
    static constexpr int RUN = 4;
};
template <> struct Matrix<double> {
    static constexpr int BLOCK = 16, COUNT = 2, HELD = 4;
    typedef double Numbers __attribute__((ext_vector_type(2)));
    typedef double Sums __attribute__((ext_vector_type(4)));
    static constexpr int PARTS = 2;
    static __device__ __forceinline__ Sums multiply(int part, Numbers p, Numbers q, Sums sums) {
        return __builtin_amdgcn_mfma_f64_16x16x4f64(p[part], q[part], sums, 0, 0, 0);
    }
    static __device__ __forceinline__ int row_of(int lane, int i) { return 4 * i + lane / 16; }
    static constexpr int RUN = 1;
};

template <typename T> using Numbers = typename Matrix<T>::Numbers;

/// A piece at any alignment.
template <typename T> __device__ __forceinline__ Numbers<T> load_numbers(const T* from) {
    constexpr int COUNT = Matrix<T>::COUNT;
    typedef T Anywhere __attribute__((ext_vector_type(COUNT), aligned(sizeof(T))));
    const Anywhere a = *reinterpret_cast<const Anywhere*>(from);
    Numbers<T> v;
#pragma unroll
    for (int i = 0; i < COUNT; i++) {
        v[i] = a[i];
    }
    return v;
}
/// The first `count` numbers (at least one), zeros behind them.
template <typename T> __device__ __forceinline__ Numbers<T> load_some_numbers(const T* from, int32_t count) {
    Numbers<T> v;
#pragma unroll
    for (int i = 0; i < Matrix<T>::COUNT; i++) {
        const T number = from[min(i, count - 1)];
        v[i] = i < count ? number : static_cast<T>(0.f);
    }
    return v;
}
/// Numbers `missing` .. of a piece, and as many zeros behind them (missing = all: zeros).
template <typename T> __device__ __forceinline__ Numbers<T> without_first(Numbers<T> v, int32_t missing) {
    union {
        Numbers<T> numbers;
        uint64_t half[2];
    } both;
    both.numbers = v;
    const int bits = missing * static_cast<int>(8 * sizeof(T));
    const uint64_t low = both.half[0], high = both.half[1];
    both.half[0] = bits >= 128 ? 0 : bits >= 64 ? high >> (bits - 64) : bits > 0 ? low >> bits | high << (64 - bits) : low;
    both.half[1] = bits >= 64 ? 0 : high >> bits;
    return both.numbers;
}

/// LDS of a straight side of OUTER rows: [OUTER][DEEP pieces], permuted so that 16 lanes that read the same piece of 16
/// rows reach all banks.
template <typename T, int OUTER, int DEEP> struct Straight {
    static_assert(DEEP == 8, "pieces of 128 bytes");
    static __device__ __forceinline__ int permuted(int row, int piece) { return piece ^ (row >> 1 & 7); }
    static __device__ __forceinline__ int place(int row, int piece) { return (row * DEEP + permuted(row, piece)) * 16; }
    /// which piece of its row lies at place i
    static __device__ __forceinline__ int piece(int i) { return permuted(i / DEEP, i % DEEP); }
    /// Numbers `step` of the k of a block that begins at row `outer0`.
    static __device__ __forceinline__ Numbers<T> read(const char* lds, int outer0, int step, int lane) {
        constexpr int BLOCK = Matrix<T>::BLOCK;
        const int row = outer0 + lane % BLOCK, piece = step * (WAVE / BLOCK) + lane / BLOCK;
        return *reinterpret_cast<const Numbers<T>*>(lds + place(row, piece));
    }
};

/// LDS of a turned side: [k][OUTER numbers], 16-byte pieces of a row permuted so that the four rows that the lanes of
/// a transposing read look at fall into different banks.
template <typename T, int OUTER, int DEEP> struct Turned {
    static constexpr int PIECES = OUTER / Matrix<T>::COUNT; // of a row of k
    static __device__ __forceinline__ int permuted(int k, int piece) {
        if constexpr (sizeof(T) == 2 && PIECES >= 16) {
            return piece ^ (k & 3) << 2;
        } else if constexpr (sizeof(T) == 2 && PIECES == 8) {
            return piece ^ (k >> 1 & 1) << 2;
        } else {
            return piece;
        }
    }
    static __device__ __forceinline__ int place(int k, int piece) { return (k * PIECES + permuted(k, piece)) * 16; }
    /// which piece of its row lies at place i
    static __device__ __forceinline__ int piece(int i) { return permuted(i / PIECES, i % PIECES); }
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

__device__ __constant__ const uint4 zeros_in_memory = {0, 0, 0, 0};

/// 16 bytes from memory to LDS, at `lds` (the same for all lanes) + 16 * lane, without a register. Arrived when the
/// wavefront's vmcnt says so, which `meet` waits for. (Not the builtin: behind it the compiler waits for vmcnt at the
/// next read of LDS, of whichever buffer. There is no register here that it could lose track of.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm" // (m0 as a clobber: reserved, and written here)
__device__ __forceinline__ void fetch(const void* from, char* lds) {
    const uint32_t at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)lds));
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(at), "v"(from) : "m0");
}
#pragma clang diagnostic pop

/// How the pieces of a step are loaded to registers. WHOLE: all of them lie inside of their rows, or do not matter. ALL: those
/// outside as well, from somewhere. SOME: not those.
enum class Take { WHOLE, ALL, SOME };

/// A side of the product on its way to LDS: piece i = threadIdx.x + j * THREADS, j < EACH. Through registers: SETS steps
/// are on their way at once, each in a set of registers.
template <typename T, int OUTER, int DEEP, int THREADS, int SETS> struct Pieces {
    static constexpr int EACH = OUTER * DEEP / THREADS, COUNT = Matrix<T>::COUNT;
    static constexpr bool ALIGNED = SETS == 0;
    Numbers<T> piece[ALIGNED ? 1 : SETS][ALIGNED ? 1 : EACH];

    /// piece j of a step: numbers `from` .. of a row, of which `left` are in the row (at most 0: none). Through registers,
    /// the last piece of a row is the row's last COUNT numbers (`short_rows`: there are fewer), of which it drops those of
    /// the piece before when it is stored.
    template <Take HOW>
    __device__ __forceinline__ void take(int set, int j, const T* from, int32_t left, bool short_rows, char* lds, int wave) {
        const void* const nowhere = &zeros_in_memory;
        const int32_t missing = max(COUNT - left, 0);
        if constexpr (ALIGNED) {
            fetch(left > 0 ? static_cast<const void*>(from) : nowhere, lds + (wave * WAVE + j * THREADS) * 16);
        } else if constexpr (HOW == Take::WHOLE) {
            piece[set][j] = load_numbers<T>(from);
        } else if constexpr (HOW == Take::ALL) {
            const T* const any = static_cast<const T*>(nowhere);
            piece[set][j] = short_rows ? load_some_numbers<T>(left > 0 ? from : any, left > 0 ? left : COUNT)
                                       : load_numbers<T>(missing < COUNT ? from - missing : any);
        } else if (short_rows) { // (uniform)
            piece[set][j] = left > 0 ? load_some_numbers<T>(from, left) : Numbers<T>{};
        } else if (missing < COUNT) {
            piece[set][j] = load_numbers<T>(from - missing);
        }
    }
    /// a piece that came through registers
    __device__ __forceinline__ void put(int set, int j, int32_t left, bool complete, char* lds) const {
        if constexpr (!ALIGNED) {
            *reinterpret_cast<Numbers<T>*>(lds + (threadIdx.x + j * THREADS) * 16) =
                complete ? piece[set][j] : without_first<T>(piece[set][j], min(max(COUNT - left, 0), COUNT));
        }
    }
};

template <typename T, int OUTER, int DEEP, int THREADS, int SETS>
struct StraightLoader : public Pieces<T, OUTER, DEEP, THREADS, SETS> {
    typedef Pieces<T, OUTER, DEEP, THREADS, SETS> Base;
    typedef Straight<T, OUTER, DEEP> Layout;
    using Base::COUNT;
    using Base::EACH;
    const T* from[EACH];
    int32_t k_size;

    static __device__ __forceinline__ int row(int j) { return (threadIdx.x + j * THREADS) / DEEP; }
    static __device__ __forceinline__ int of_row(int j) { return Layout::piece((threadIdx.x + j * THREADS)); }

    /// row_at(i): pointer to the row of memory behind row i of the side (any one for a row that does not matter)
    template <typename RowAt> __device__ __forceinline__ void begin(int32_t k, RowAt&& row_at) {
        k_size = k;
#pragma unroll
        for (int j = 0; j < EACH; j++) {
            from[j] = row_at(row(j)) + of_row(j) * COUNT;
        }
    }
    /// Piece j of the next step, which begins at k0 (steps are asked for in order).
    template <Take HOW> __device__ __forceinline__ void load(int set, int j, int32_t k0, char* lds, int wave) {
        this->template take<HOW>(set, j, from[j], k_size - k0 - of_row(j) * COUNT, k_size < COUNT, lds, wave);
        from[j] += DEEP * COUNT;
    }
    /// The pieces of a step that came through registers (`whole`: as WHOLE).
    __device__ __forceinline__ void store(int set, int32_t k0, bool whole, char* lds) const {
#pragma unroll
        for (int j = 0; j < EACH; j++) {
            this->put(set, j, k_size - k0 - of_row(j) * COUNT, whole || k_size < COUNT, lds);
        }
    }
};

/// Rows of `width` numbers, of which those from outer0 on are used.
template <typename T, int OUTER, int DEEP, int THREADS, int SETS>
struct TurnedLoader : public Pieces<T, OUTER, DEEP, THREADS, SETS> {
    typedef Pieces<T, OUTER, DEEP, THREADS, SETS> Base;
    typedef Turned<T, OUTER, DEEP> Layout;
    using Base::ALIGNED;
    using Base::COUNT;
    using Base::EACH;
    static constexpr int K_EACH = THREADS / Layout::PIECES; // rows of k between a thread's pieces
    const T* from; // the thread's column of row 0 of the matrix; of the next step's first piece (load)
    size_t next;   // numbers from a step to the next
    size_t between; // numbers between a thread's pieces
    int32_t left;   // numbers in the row from the thread's column on
    bool short_rows;

    static __device__ __forceinline__ int k(int j) { return threadIdx.x / Layout::PIECES + j * K_EACH; }
    /// (the same for all pieces of a thread: their rows differ by multiples of four)
    static __device__ __forceinline__ int of_row() { return Layout::piece(threadIdx.x); }

    __device__ __forceinline__ void begin(const T* memory, int32_t row_width, int32_t first) {
        static_assert(K_EACH % 4 == 0 && EACH * THREADS == OUTER * DEEP, "");
        const int32_t outer = first + of_row() * COUNT;
        left = row_width - outer;
        short_rows = row_width < COUNT;
        // (a piece that is outside of the rows: any piece that is not)
        from = memory + (left > 0 ? outer : 0);
        next = static_cast<size_t>(DEEP * COUNT) * row_width;
        between = static_cast<size_t>(K_EACH) * row_width;
    }
    /// Every piece of the step inside of its row, or outside as a whole.
    __device__ __forceinline__ bool whole() const { return ALIGNED || left >= COUNT || left <= 0; }

    /// Piece j of the next step of consecutive rows (after begin_rows), of which the matrix has rows_left.
    __device__ __forceinline__ void begin_rows() { from += static_cast<size_t>(k(0)) * (between / K_EACH); }
    template <Take HOW> __device__ __forceinline__ void load(int set, int j, int32_t rows_left, char* lds, int wave) {
        this->template take<HOW>(set, j, from + j * between, k(j) < rows_left ? left : 0, short_rows, lds, wave);
        from += j == EACH - 1 ? next : 0;
    }
    /// Piece j of a step whose row is `row` there (negative: none; not with WHOLE).
    template <Take HOW> __device__ __forceinline__ void load_row(int set, int j, int32_t row, char* lds, int wave) {
        const size_t at = static_cast<size_t>(HOW == Take::WHOLE ? row : max(row, 0)) * (between / K_EACH);
        this->template take<HOW>(set, j, from + at, row >= 0 ? left : 0, short_rows, lds, wave);
    }
    /// The pieces of a step that came through registers, of a side that has rows_left more rows.
    __device__ __forceinline__ void store(int set, int32_t rows_left, bool whole, char* lds) const {
#pragma unroll
        for (int j = 0; j < EACH; j++) {
            this->put(set, j, k(j) < rows_left ? left : 0, whole || short_rows, lds);
        }
    }
};

/// Everything this wavefront has asked of LDS has arrived, and of what it has asked of memory for LDS all but the last
/// LATER pieces (negative: nothing goes that way); then the workgroup meets.
template <int LATER> __device__ __forceinline__ void meet() {
    if constexpr (LATER < 0) {
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    } else {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LATER) : "memory");
    }
}

/// WM x WN wavefronts; every one of them makes BM / WM x BN / WN numbers, in steps of DEEP pieces of k of which STAGES
/// are in LDS or on their way there.
template <int BM, int BN, int DEEP, int STAGES> struct TileLds {
    char stages[STAGES * (BM + BN) * DEEP * 16] __attribute__((aligned(16)));
    int32_t rows[BM];
};
template <typename T, Form FORM, int BM, int BN, int WM, int WN, int DEEP, int STAGES, bool ALIGNED>
__device__ __forceinline__ void make_tile(
    const Product<T>& g, const uint32_t block, TileLds<BM, BN, DEEP, STAGES>& lds
) {
    typedef Matrix<T> M;
    constexpr int THREADS = WM * WN * WAVE, COUNT = M::COUNT, BLOCK = M::BLOCK;
    constexpr int STEP = DEEP * COUNT, STEPS = DEEP * BLOCK / WAVE;
    constexpr int MB = BM / WM / BLOCK, NB = BN / WN / BLOCK; // blocks of a wavefront
    constexpr bool SUMS = FORM == Form::GRAD_SUMS, Q_TURNED = SUMS, P_TURNED = FORM != Form::GRAD_ROWS;
    constexpr Units UNITS = SUMS ? Units::OF_GROUPS : Units::OF_ROWS;
    constexpr int SETS = ALIGNED ? 0 : 2; // (what there is room for in registers)
    using QLoader = std::conditional_t<
        Q_TURNED, TurnedLoader<T, BM, DEEP, THREADS, SETS>, StraightLoader<T, BM, DEEP, THREADS, SETS>>;
    using PLoader = std::conditional_t<
        P_TURNED, TurnedLoader<T, BN, DEEP, THREADS, SETS>, StraightLoader<T, BN, DEEP, THREADS, SETS>>;
    constexpr int P_AT = BM * DEEP * 16, BYTES = P_AT + BN * DEEP * 16;
    static_assert(ALIGNED || STAGES == 2, "through registers: one step in LDS beside the present one");
    char* const stages = lds.stages;
    int32_t* const rows = lds.rows;

    // Workgroups b, b + 8, .. run on the same XCD. Tiles of rows take the same time each: an XCD gets consecutive ones, so
    // that its L2 holds what they share. A unit of GRAD_SUMS takes as long as it has rows: its tiles go to all XCDs (24
    // uneven groups, 1280 x 1000, in consecutive tiles: 122 us instead of 115).
    constexpr bool MAY_SPLIT = !SUMS && BM == 64;
    const int32_t splits = MAY_SPLIT ? g.splits : 1;
    const int32_t tiles_of_unit = (SUMS ? g.m_tiles : splits) * g.n_tiles;
    UnitsOfGroups<UNITS> of_groups(g.groups, g.step);
    const int32_t units = min(of_groups.total(), g.most_units);
    const int64_t tiles = static_cast<int64_t>(units) * tiles_of_unit;
    const int32_t per_xcd = static_cast<int32_t>((tiles + 7) / 8);
    const int64_t tile = SUMS ? block : static_cast<int64_t>(block % 8) * per_xcd + block / 8;
    if (static_cast<int32_t>(block / 8) >= per_xcd || tile >= tiles) {
        return; // (uniform)
    }
    int32_t unit_index, m0, n0, split = 0;
    if (SUMS) {
        unit_index = static_cast<int32_t>(tile / tiles_of_unit);
        const int32_t of_unit = static_cast<int32_t>(tile % tiles_of_unit);
        m0 = of_unit / g.n_tiles * BM;
        n0 = of_unit % g.n_tiles * BN;
    } else {
        // bands of four units: their rows and a tile's columns of the matrix are read together (of two or eight: the same
        // time)
        const int32_t of_band = 4 * tiles_of_unit;
        const int32_t band = static_cast<int32_t>(tile / of_band), in_band = static_cast<int32_t>(tile % of_band);
        const int32_t height = min(4, units - 4 * band);
        unit_index = 4 * band + in_band % height;
        m0 = 0;
        n0 = in_band / height / splits * BN;
        split = in_band / height % splits;
    }
    const GroupUnit unit = of_groups.find(unit_index);
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

    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
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

    const int32_t k_begin = MAY_SPLIT ? split * g.k_each : 0;
    const int32_t k_size = __builtin_amdgcn_readfirstlane(
        rest ? 0 : SUMS ? unit.count : splits > 1 ? min(g.k_size - k_begin, g.k_each) : g.k_size
    );
    if (k_size > 0) {
        QLoader q;
        PLoader p;
        if constexpr (Q_TURNED) {
            q.begin(g.q.data, g.q.stride, m0);
        } else {
            q.begin(k_size, [&](int i) { return g.q.data + static_cast<size_t>(rows[i]) * g.q.stride + k_begin; });
        }
        const size_t of_group = static_cast<size_t>(unit.group) * (P_TURNED ? g.k_size : g.n_size) * g.p.stride;
        if constexpr (SUMS) {
            p.begin(g.p.data, g.p.stride, n0);
        } else if constexpr (P_TURNED) {
            p.begin(g.p.data + of_group + static_cast<size_t>(k_begin) * g.p.stride, g.p.stride, n0);
            p.begin_rows();
        } else {
            p.begin(k_size, [&](int i) {
                return g.p.data + of_group + static_cast<size_t>(min(n0 + i, g.n_size - 1)) * g.p.stride + k_begin;
            });
        }
        constexpr int Q_EACH = QLoader::EACH, P_EACH = PLoader::EACH, EACH = Q_EACH + P_EACH;
        // GRAD_SUMS: the rows behind the pieces of a step, found SETS steps before its pieces are asked for (what waits for
        // them then waits for no pieces that were asked for later)
        constexpr int ROW_SETS = ALIGNED ? 1 : SETS;
        [[maybe_unused]] int32_t row_of_piece[ROW_SETS][SUMS ? EACH : 1];
        auto find_rows = [&](int set, int32_t k0) {
            if constexpr (SUMS) {
                auto row_at = [&](int k) { return k0 + k < k_size ? g.groups.row_at(unit.begin + k0 + k) : -1; };
#pragma unroll
                for (int j = 0; j < EACH; j++) {
                    row_of_piece[set][j] = j >= Q_EACH && QLoader::K_EACH == PLoader::K_EACH
                                               ? row_of_piece[set][j - Q_EACH]
                                               : row_at(j < Q_EACH ? QLoader::k(j) : PLoader::k(j - Q_EACH));
                }
            }
        };
        // Piece `piece` of the step that begins at k0 (find_rows of it before).
        auto load_piece = [&](auto take, int set, int piece, int32_t k0, char* buffer) {
            constexpr Take HOW = decltype(take)::value;
            if constexpr (SUMS) {
                if (piece < Q_EACH) {
                    q.template load_row<HOW>(set, piece, row_of_piece[set][piece], buffer, wave);
                } else {
                    p.template load_row<HOW>(set, piece - Q_EACH, row_of_piece[set][piece], buffer + P_AT, wave);
                }
            } else if (piece < Q_EACH) {
                q.template load<HOW>(set, piece, k0, buffer, wave);
            } else {
                p.template load<HOW>(set, piece - Q_EACH, P_TURNED ? k_size - k0 : k0, buffer + P_AT, wave);
            }
        };
        typedef std::integral_constant<Take, Take::WHOLE> Whole;
        typedef std::integral_constant<Take, Take::ALL> All;
        typedef std::integral_constant<Take, Take::SOME> Some;
        // through registers, no step but the last one needs to look where the matrices end
        bool whole = true;
        if constexpr (!ALIGNED) {
            if constexpr (Q_TURNED) {
                whole = whole && q.whole();
            }
            if constexpr (P_TURNED) {
                whole = whole && p.whole();
            }
            whole = __all(whole);
        }
        auto load_some = [&](int from, int upto, int32_t k0, char* buffer) {
#pragma unroll
            for (int piece = 0; piece < EACH; piece++) {
                if (piece >= from && piece < upto) {
                    load_piece(Some(), 0, piece, k0, buffer);
                }
            }
        };
        // through registers: a step from memory to a set of them, and from there to LDS
        auto is_whole = [&](int32_t k0) { return whole && k0 + STEP <= k_size; }; // (uniform)
        auto load = [&](auto otherwise, int set, int32_t k0) {
            if (is_whole(k0)) {
#pragma unroll
                for (int piece = 0; piece < EACH; piece++) {
                    load_piece(Whole(), set, piece, k0, nullptr);
                }
            } else {
#pragma unroll
                for (int piece = 0; piece < EACH; piece++) {
                    load_piece(otherwise, set, piece, k0, nullptr);
                }
            }
        };
        auto store = [&](int set, int32_t k0, char* buffer) {
            q.store(set, Q_TURNED ? k_size - k0 : k0, is_whole(k0), buffer);
            p.store(set, P_TURNED ? k_size - k0 : k0, is_whole(k0), buffer + P_AT);
        };
        Numbers<T> of_q[2][MB], of_p[2][NB];
        // what a multiplication needs, in the order in which it needs it: q 0, p 0 .. NB - 1, q 1 .. MB - 1
        auto read = [&](const char* buffer, int step, int which) {
            if (which == 0 || which > NB) {
                const int i = which == 0 ? 0 : which - NB;
                of_q[step % 2][i] = QLoader::Layout::read(buffer, wave_m + i * BLOCK, step, lane);
            } else {
                const int j = which - 1;
                of_p[step % 2][j] = PLoader::Layout::read(buffer + P_AT, wave_n + j * BLOCK, step, lane);
            }
        };
        // wavefronts whose rows are all behind the unit's only carry pieces (a unit's last tile)
        const bool works = SUMS || wave_m < unit.count;
        // One multiplication of a step, and between its matrix instructions, in this order: the reads of the next one, and
        // pieces [first, last) of another step, asked for by between(from, upto). (Left to itself the compiler puts all
        // reads in front, where they are waited for, and a wavefront that asks for eight pieces in a row waits until the
        // memory pipeline has taken them.)
        constexpr int SLOTS = MB * NB * M::PARTS, READS = MB + NB, OF_SLOT = (READS + SLOTS - 1) / SLOTS;
        auto multiply = [&](int step, const char* next_buffer, int next_step, int first, int last, auto&& between) {
            if (!works) {
                between(first, last);
                return;
            }
            int asked = first;
#pragma unroll
            for (int slot = 0; slot < SLOTS; slot++) {
#pragma unroll
                for (int r = slot * OF_SLOT; r < (slot + 1) * OF_SLOT; r++) {
                    if (r < READS) {
                        read(next_buffer, next_step, r);
                    }
                }
                const int upto = first + (slot + 1) * (last - first) / SLOTS;
                between(asked, upto);
                asked = upto;
                const int i = slot / (NB * M::PARTS), j = slot % NB;
                sums[i][j] = M::multiply(slot / NB % M::PARTS, of_p[step % 2][j], of_q[step % 2][i], sums[i][j]);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        auto nothing = [](int, int) {};
        static_assert(STEPS % 2 == 0, "the numbers of step 0 come to the place of the last step but one");
        // Step t is multiplied from stage t % STAGES. Where the workgroup meets in it, step t + 1 has arrived, and the
        // stage is free for step t + STAGES: EARLY of its pieces are asked for right then, the others in the next step's
        // first multiplication. (Steps behind the last one are asked for like all others: zeros.) Through registers: in
        // front of the meeting step t + 1 is put into its stage, from a set that step t + 1 + SETS comes to. (32768 rows of
        // 32 groups, K = 2048, L = 4096, bfloat16: 585 us with half of the pieces early, 600 with a quarter.)
        constexpr int EARLY = EACH / 2;
        char *before = stages + (STAGES - 1) * BYTES, *buffer = stages;
        auto read_first = [&] {
            if (works) {
#pragma unroll
                for (int r = 0; r < READS; r++) {
                    read(buffer, 0, r);
                }
            }
        };
        if constexpr (ALIGNED) {
#pragma unroll
            for (int t = 0; t < STAGES; t++) {
                find_rows(0, t * STEP);
                load_some(0, t == STAGES - 1 ? EARLY : EACH, t * STEP, stages + t * BYTES);
            }
            meet<(STAGES - 2) * EACH + EARLY>();
            read_first();
            for (int32_t k0 = 0; k0 < k_size; k0 += STEP) {
#pragma unroll
                for (int step = 0; step < STEPS - 1; step++) {
                    if (step == 0) {
                        multiply(step, buffer, step + 1, EARLY, EACH, [&](int from, int upto) {
                            load_some(from, upto, k0 + (STAGES - 1) * STEP, before);
                        });
                        find_rows(0, k0 + STAGES * STEP);
                    } else {
                        multiply(step, buffer, step + 1, 0, 0, nothing);
                    }
                }
                char* const following = buffer + BYTES < stages + STAGES * BYTES ? buffer + BYTES : stages;
                meet<(STAGES - 2) * EACH>();
                multiply(STEPS - 1, following, 0, 0, EARLY, [&](int from, int upto) {
                    load_some(from, upto, k0 + STAGES * STEP, buffer);
                });
                before = buffer;
                buffer = following;
            }
        } else {
            // Long sums have a loop in which every step loads all of its pieces: the compiler counts what is on its way, and
            // behind a load that may not have been issued it can only wait for everything (4402 rows of 24 groups,
            // K = 1797, L = 269, float16: 37 us instead of 61). Their last steps, and sums that have no more, load what
            // there is (53740 rows, K = 9, L = 2389: 124 us instead of 145).
            constexpr int LOOKS = (SUMS ? 2 * SETS : SETS) + 1; // steps behind the present one that a step has to do with
            auto begin_with = [&](auto take) {
                constexpr bool ALL = decltype(take)::value == Take::ALL;
                // (SOME: the first step is not to wait for the others)
                constexpr int FIRST = ALL ? SETS : 1;
#pragma unroll
                for (int t = 0; t < FIRST; t++) {
                    find_rows(t, t * STEP);
                    load(take, t, t * STEP);
                }
                if (!ALL) {
                    store(0, 0, stages);
                }
#pragma unroll
                for (int t = FIRST; t < SETS; t++) {
                    find_rows(t, t * STEP);
                    if (t * STEP < k_size) { // (uniform)
                        load(take, t, t * STEP);
                    }
                }
#pragma unroll
                for (int t = 0; t < SETS; t++) {
                    find_rows(t, (SETS + t) * STEP);
                }
                if (ALL) {
                    store(0, 0, stages);
                }
                if (ALL || SETS * STEP < k_size) { // (uniform)
                    load(take, 0, SETS * STEP);
                }
                find_rows(0, 2 * SETS * STEP);
                meet<-1>();
                read_first();
            };
            auto step_at = [&](auto take, int set, int32_t k0) {
#pragma unroll
                for (int step = 0; step < STEPS - 1; step++) {
                    multiply(step, buffer, step + 1, 0, 0, nothing);
                }
                char* const following = buffer == stages ? stages + BYTES : stages;
                store(set, k0 + STEP, following);
                meet<-1>();
                if (decltype(take)::value == Take::ALL || k0 + (SETS + 1) * STEP < k_size) { // (uniform)
                    load(take, set, k0 + (SETS + 1) * STEP);
                    find_rows(set, k0 + (2 * SETS + 1) * STEP);
                }
                multiply(STEPS - 1, following, 0, 0, 0, nothing);
                buffer = following;
            };
            int32_t k0 = 0;
            if (k_size >= (LOOKS + SETS) * STEP) {
                begin_with(All());
                for (; k0 + (LOOKS + SETS) * STEP <= k_size; k0 += SETS * STEP) {
#pragma unroll
                    for (int u = 0; u < SETS; u++) {
                        step_at(All(), (u + 1) % SETS, k0 + u * STEP);
                    }
                }
            } else {
                begin_with(Some());
            }
            for (; k0 < k_size; k0 += SETS * STEP) {
#pragma unroll
                for (int u = 0; u < SETS; u++) {
                    if (k0 + u * STEP < k_size) { // (uniform)
                        step_at(Some(), (u + 1) % SETS, k0 + u * STEP);
                    }
                }
            }
        }
        meet<0>(); // (nothing is on its way to LDS any more)
    }

    // Every wavefront turns its blocks over in LDS of its own, to store whole pieces of rows side by side (straight from
    // the registers, 8 bytes of 32 rows per store: 32768 rows, K = 2048, L = 4096, bfloat16: 657 us instead of 613).
    __syncthreads();
    auto put = [&](auto zero, auto is_partial, auto&& row_at) {
        typedef decltype(zero) To;
        constexpr int COLUMNS = BN / WN, OF_PIECE = 16 / sizeof(To), RUN = M::RUN, PIECES = COLUMNS / OF_PIECE;
        constexpr int ROWS_ABREAST = PIECES >= 16 ? 1 : 16 / PIECES; // rows in 256 bytes, all banks
        static_assert(BLOCK * COLUMNS * sizeof(To) * WM * WN <= sizeof(lds.stages), "");
        typedef To Run __attribute__((ext_vector_type(RUN)));
        typedef To Piece __attribute__((ext_vector_type(OF_PIECE), aligned(sizeof(To))));
        char* const mine = stages + wave * (BLOCK * COLUMNS * sizeof(To));
        auto place = [](int row, int piece) {
            return (row * PIECES + (piece ^ (row / ROWS_ABREAST & (PIECES - 1)))) * 16;
        };
#pragma unroll
        for (int i = 0; i < MB; i++) {
#pragma unroll
            for (int j = 0; j < NB; j++) {
#pragma unroll
                for (int e = 0; e < M::HELD; e += RUN) {
                    const int column = j * BLOCK + M::row_of(lane, e);
                    Run run;
#pragma unroll
                    for (int r = 0; r < RUN; r++) {
                        run[r] = static_cast<To>(sums[i][j][e + r]);
                    }
                    *reinterpret_cast<Run*>(
                        mine + place(lane % BLOCK, column / OF_PIECE) + column % OF_PIECE * sizeof(To)
                    ) = run;
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
            for (int at = 0; at < BLOCK * PIECES; at += WAVE) {
                const int row = (at + lane) / PIECES, piece = (at + lane) % PIECES;
                const int32_t n = n0 + wave_n + piece * OF_PIECE;
                To* const to = row_at(wave_m + i * BLOCK + row); // (null: no such row)
                if (to != nullptr && n < g.n_size) {
                    const Piece numbers = *reinterpret_cast<const Piece*>(mine + place(row, piece));
                    if (n + OF_PIECE <= g.n_size) {
                        // (a result streams past the caches: 20011 rows, K = 1280, L = 1000, gradients: 182 us instead of
                        // 191; partial results are read again at once)
                        if constexpr (decltype(is_partial)::value) {
                            *reinterpret_cast<Piece*>(to + n) = numbers;
                        } else {
                            __builtin_nontemporal_store(numbers, reinterpret_cast<Piece*>(to + n));
                        }
                    } else {
#pragma unroll
                        for (int r = 0; r < OF_PIECE; r++) {
                            if (n + r < g.n_size) {
                                to[n + r] = numbers[r];
                            }
                        }
                    }
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        }
    };
    if constexpr (SUMS) {
        const size_t size = static_cast<size_t>(g.m_size) * g.n_size;
        auto row_of = [&](auto* result) {
            return [=, &g](int m) {
                return m0 + m < g.m_size ? result + static_cast<size_t>(m0 + m) * g.n_size : nullptr;
            };
        };
        if (unit.of_group > 1) { // (uniform)
            if (unit.slot < g.most_slots) {
                put(wide_t<T>(), std::true_type(), row_of(g.partial + unit.slot * partial_size(g.m_size, g.n_size)));
            }
        } else {
            put(T(), std::false_type(), row_of(g.out + unit.group * size));
        }
    } else {
        auto row_of = [&](auto* result) {
            return [=, &g](int m) { return m < unit.count ? result + static_cast<size_t>(rows[m]) * g.n_size : nullptr; };
        };
        if (MAY_SPLIT && splits > 1) { // (uniform)
            if constexpr (MAY_SPLIT) {
                put(wide_t<T>(), std::true_type(), row_of(g.partial + static_cast<size_t>(split) * g.groups.n_rows * g.n_size));
            }
        } else {
            put(T(), std::false_type(), row_of(g.out));
        }
    }
}

/// The rows of a matrix, each continued with zeros to whole pieces. A workgroup copies COPY_ROWS of them.
constexpr int COPY_ROWS = 8, COPY_THREADS = 256;
template <typename T>
__global__ __launch_bounds__(COPY_THREADS) void copy_rows_kernel(
    T* __restrict__ to, const T* __restrict__ from, size_t n_rows, int32_t width, int32_t pieces
) {
    constexpr int32_t COUNT = Matrix<T>::COUNT;
    const size_t row0 = static_cast<size_t>(blockIdx.x) * COPY_ROWS;
    const uint32_t count = static_cast<uint32_t>(min(n_rows - row0, static_cast<size_t>(COPY_ROWS))) * pieces;
#pragma unroll 4
    for (uint32_t i = threadIdx.x; i < count; i += COPY_THREADS) {
        const uint32_t row = i / pieces;
        const int32_t first = static_cast<int32_t>(i % pieces) * COUNT;
        const T* at = from + (row0 + row) * width + first;
        const Numbers<T> numbers =
            first + COUNT <= width ? load_numbers<T>(at) : load_some_numbers<T>(at, width - first);
        *reinterpret_cast<Numbers<T>*>(to + ((row0 + row) * pieces + i % pieces) * COUNT) = numbers;
    }
}

/// out := the sum of the shares of k.
constexpr int JOIN_THREADS = 256;
template <typename T> __global__ __launch_bounds__(JOIN_THREADS) void join_splits_kernel(Product<T> g) {
    const size_t size = static_cast<size_t>(g.groups.n_rows) * g.n_size;
    const size_t i = blockIdx.x * static_cast<size_t>(JOIN_THREADS) + threadIdx.x;
    if (i < size) {
        wide_t<T> sum = 0;
#pragma unroll 8
        for (int32_t s = 0; s < g.splits; s++) {
            sum += g.partial[s * size + i];
        }
        g.out[i] = static_cast<T>(sum);
    }
}

/// Wavefronts per SIMD: small tiles through registers wait for memory most of the time and have room for four (60094 rows,
/// K = 107, L = 31, float16: 9.4 us, with three and more pieces on their way in each 12.0).
template <typename T, int BM, bool ALIGNED> constexpr int ABREAST = BM == 64 && !ALIGNED && sizeof(T) < 8 ? 4 : 2;

template <typename T, Form FORM, int BM, int BN, int WM, int WN, int DEEP, int STAGES, bool ALIGNED>
__global__ __launch_bounds__(WM* WN* WAVE, (ABREAST<T, BM, ALIGNED>)) void tiles_kernel(Product<T> g) {
    __shared__ TileLds<BM, BN, DEEP, STAGES> lds;
    make_tile<T, FORM, BM, BN, WM, WN, DEEP, STAGES, ALIGNED>(g, blockIdx.x, lds);
}

/// Both gradients in one launch, the sums' tiles (of which there are `of_sums` workgroups, a multiple of 8) in front: they
/// take longer, and the rows' tiles fill in behind them.
template <typename T, int BM, int BN, int WM, int WN, int DEEP, int STAGES, bool ALIGNED>
__global__ __launch_bounds__(WM* WN* WAVE, 2) void gradients_kernel(Product<T> sums, Product<T> rows, uint32_t of_sums) {
    __shared__ TileLds<BM, BN, DEEP, STAGES> lds;
    if (blockIdx.x < of_sums) {
        make_tile<T, Form::GRAD_SUMS, BM, BN, WM, WN, DEEP, STAGES, ALIGNED>(sums, blockIdx.x, lds);
    } else {
        make_tile<T, Form::GRAD_ROWS, BM, BN, WM, WN, DEEP, STAGES, ALIGNED>(rows, blockIdx.x - of_sums, lds);
    }
}

/// out[g, :] := the sum of its units' partial results, for groups of more than one unit, each shared out over all
/// workgroups. A lane has four numbers; of many partial results, a wavefront has every fourth.
constexpr int JOIN_WAVES = 4, JOINED = 4;
template <typename T> __global__ __launch_bounds__(JOIN_WAVES* WAVE) void join_units_kernel(Product<T> g) {
    typedef wide_t<T> Wide __attribute__((ext_vector_type(JOINED)));
    typedef T Narrow __attribute__((ext_vector_type(JOINED), aligned(sizeof(T))));
    __shared__ Wide shared[JOIN_WAVES][WAVE];
    const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
    const size_t size = static_cast<size_t>(g.m_size) * g.n_size, pieces = partial_size(g.m_size, g.n_size) / JOINED;
    UnitsOfGroups<Units::OF_GROUPS> of_groups(g.groups, g.step);
    int32_t turn = static_cast<int32_t>(blockIdx.x); // (another workgroup begins with each group)
    of_groups.for_split_groups([&](const GroupUnit& unit) {
        const int32_t parts = min(unit.of_group, g.most_slots - unit.slot);
        const int32_t sharing = parts >= 4 * JOIN_WAVES ? JOIN_WAVES : 1;
        const size_t at_once = JOIN_WAVES / sharing * WAVE;
        const Wide* from = reinterpret_cast<const Wide*>(g.partial) + unit.slot * pieces;
        T* const to = g.out + unit.group * size;
        size_t first = turn * at_once;
        for (; first < pieces; first += gridDim.x * at_once) {
            const size_t i = first + (sharing > 1 ? lane : threadIdx.x);
            Wide sum{};
            if (i < pieces) {
#pragma unroll 8
                for (int32_t u = sharing > 1 ? wave : 0; u < parts; u += sharing) {
                    sum += from[u * pieces + i];
                }
            }
            if (sharing > 1) { // (uniform)
                __syncthreads();
                shared[wave][lane] = sum;
                __syncthreads();
                if (wave == 0) {
#pragma unroll
                    for (int w = 1; w < JOIN_WAVES; w++) {
                        sum += shared[w][lane];
                    }
                }
            }
            if (i < pieces && (sharing == 1 || wave == 0)) {
                Narrow narrow;
#pragma unroll
                for (int j = 0; j < JOINED; j++) {
                    narrow[j] = static_cast<T>(sum[j]);
                }
                if ((i + 1) * JOINED <= size) {
                    *reinterpret_cast<Narrow*>(to + i * JOINED) = narrow;
                } else {
#pragma unroll
                    for (int j = 0; j < JOINED; j++) {
                        if (i * JOINED + j < size) {
                            to[i * JOINED + j] = narrow[j];
                        }
                    }
                }
            }
        }
        turn = static_cast<int32_t>((first - pieces) / at_once % gridDim.x);
    });
}

} // namespace mops::amd::grouped_product

#endif
