// Element types of the layers' operators (mops/layers.h): what a number is
// computed in, wide loads and stores, and the rounding to 16 bits.
#ifndef MOPS_AMD_NUMBERS_HPP
#define MOPS_AMD_NUMBERS_HPP

#include <cstdint>
#include <type_traits>

#include <hip/hip_runtime.h>

#include "mops/layers.hpp"

#include "runtime.hpp"

namespace mops::amd {

/// The device's own type behind an element type of the interface (same bits).
template <typename T> struct DeviceNumber {
    typedef T type;
};
template <> struct DeviceNumber<bfloat16> {
    typedef __bf16 type;
};
template <> struct DeviceNumber<float16> {
    typedef _Float16 type;
};
template <typename T> using device_t = typename DeviceNumber<T>::type;

/// What sums of T are held in: 32 bits for the 16-bit types, else T.
template <typename T> using wide_t = std::conditional_t<std::is_same_v<T, double>, double, float>;

/// N numbers of a row, loaded and stored as one piece of memory. Aligned to the numbers only: rows of
/// odd length start anywhere, and the hardware's wide loads and stores take any address.
template <typename T, int N> struct Piece {
    typedef T Vector __attribute__((ext_vector_type(N), aligned(sizeof(T))));
    Vector v;

    static __device__ __forceinline__ Piece load(const T* p) {
        return Piece{*reinterpret_cast<const Vector*>(p)};
    }
    __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<Vector*>(p) = v; }
    /// The same for memory that is passed over once: caches do not keep it.
    static __device__ __forceinline__ Piece stream(const T* p) {
        return Piece{__builtin_nontemporal_load(reinterpret_cast<const Vector*>(p))};
    }
    __device__ __forceinline__ void stream_to(T* p) const {
        __builtin_nontemporal_store(v, reinterpret_cast<Vector*>(p));
    }
    __device__ __forceinline__ wide_t<T> get(int i) const { return static_cast<wide_t<T>>(v[i]); }
    /// (to nearest, ties to even: the one rounding of a result)
    __device__ __forceinline__ void set(int i, wide_t<T> x) { v[i] = static_cast<T>(x); }
};
template <typename T> struct Piece<T, 1> {
    T v;

    static __device__ __forceinline__ Piece load(const T* p) { return Piece{*p}; }
    __device__ __forceinline__ void store(T* p) const { *p = v; }
    static __device__ __forceinline__ Piece stream(const T* p) { return Piece{*p}; }
    __device__ __forceinline__ void stream_to(T* p) const { *p = v; }
    __device__ __forceinline__ wide_t<T> get(int) const { return static_cast<wide_t<T>>(v); }
    __device__ __forceinline__ void set(int, wide_t<T> x) { v = static_cast<T>(x); }
};

/// Numbers of T in 16 bytes.
template <typename T> constexpr int PIECE = 16 / static_cast<int>(sizeof(T));

/// Columns of a row in pieces of N: piece i begins at column start(i). The last one is moved to the
/// left so that it ends with the row (it then repeats columns of the one before; both hold the same
/// values), so that no row needs a loop over single columns. For rows of at least N columns.
struct PiecesOfRow {
    int32_t columns, pieces;

    template <int N> static __host__ __device__ __forceinline__ PiecesOfRow make(int32_t columns) {
        return PiecesOfRow{columns, (columns + N - 1) / N};
    }
    template <int N> __device__ __forceinline__ int32_t start(int32_t piece) const {
        return min(piece * N, columns - N);
    }
};

/// An extent as the kernels count it: 32 bits, with room for the rows that a workgroup counts past the end.
inline int32_t count_i32(size_t value, const char* what) {
    constexpr size_t ROOM = 65536;
    return narrow_i32(value + ROOM, what) - static_cast<int32_t>(ROOM);
}

/// A piece of memory in the element type of the interface, as the device has it.
template <typename T, size_t N> device_t<T>* data_of(const Tensor<T, N>& tensor) {
    return reinterpret_cast<device_t<T>*>(tensor.data);
}

} // namespace mops::amd

#endif
