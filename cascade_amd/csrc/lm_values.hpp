// Rows of 16-bit or 32-bit floating point, which may begin anywhere and have any length from eight on, in pieces of V values: sixteen bytes, or eight where a
// 16-bit row goes with one of 32. What begins at no multiple of its size is one access all the same; a row's last piece, where it is not whole, is moved back over the piece
// before it. What two pieces hold both is computed and stored twice, with the same result, and left out of sums once.
#pragma once
#include "lm_common.hpp"

namespace lm {

constexpr int LEAST_DIM = 8;

template <class T>
constexpr int PIECE = 16 / sizeof(T);

struct Piece {
    int d;     // its first value
    int skip;  // how many of its values the piece before it holds, too; all of them where the row has no such piece
    bool mine; // the row has such a piece
};

// The piece that begins at `first`, a multiple of V, of a row of dim values. It is always there to be read.
template <int V>
__device__ inline Piece piece_at(int first, int dim)
{
    const int d = first < dim - V ? first : dim - V;
    return {d, first < dim ? first - d : V, first < dim};
}

template <class T, int V>
struct __attribute__((packed, aligned(sizeof(T)))) Several {
    T x[V];
};

// V values as they lie in memory.
template <class T, int V>
using Raw = uint32_t __attribute__((ext_vector_type(sizeof(T) * V / 4)));

template <class T, int V>
__device__ inline Raw<T, V> load_raw(const T* p)
{
    return __builtin_bit_cast(Raw<T, V>, *reinterpret_cast<const Several<T, V>*>(p));
}

template <class T, int V>
__device__ inline void unpack(Raw<T, V> raw, float (&x)[V])
{
    const Several<T, V> y = __builtin_bit_cast(Several<T, V>, raw);
#pragma unroll
    for (int k = 0; k < V; ++k)
        x[k] = static_cast<float>(y.x[k]);
}

template <class T, int V>
__device__ inline void load(const T* p, float (&x)[V])
{
    unpack<T, V>(load_raw<T, V>(p), x);
}

// PAST: past the caches, for results that are larger than those.
template <bool PAST = false, class T, int V>
__device__ inline void store(T* p, const float (&x)[V])
{
    Several<T, V> raw;
#pragma unroll
    for (int k = 0; k < V; ++k)
        raw.x[k] = static_cast<T>(x[k]);
    if constexpr (PAST) {
        typedef uint32_t anywhere __attribute__((ext_vector_type(sizeof(T) * V / 4), aligned(sizeof(T))));
        __builtin_nontemporal_store(__builtin_bit_cast(anywhere, raw), reinterpret_cast<anywhere*>(p));
    } else {
        *reinterpret_cast<Several<T, V>*>(p) = raw;
    }
}

} // namespace lm
