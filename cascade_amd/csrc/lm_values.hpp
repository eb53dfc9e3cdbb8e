// Eight values at a time of rows of 16-bit or 32-bit floating point that may begin anywhere and have any length from eight on. Sixteen bytes that begin at no
// multiple of sixteen are one access all the same; a row's last piece, where it is not whole, is moved back over the piece before it. What two pieces
// hold both is computed and stored twice, with the same result, and left out of sums once.
#pragma once
#include "lm_common.hpp"

namespace lm {

constexpr int PIECE = 8;

struct Piece {
    int d;     // its first value
    int skip;  // how many of its values the piece before it holds, too; all of them where the row has no such piece
    bool mine; // the row has such a piece
};

// The piece that begins at `first`, a multiple of eight, of a row of dim >= 8 values. It is always there to be read.
__device__ inline Piece piece_at(int first, int dim)
{
    const int d = first < dim - PIECE ? first : dim - PIECE;
    return {d, first < dim ? first - d : PIECE, first < dim};
}

template <class T>
struct __attribute__((packed, aligned(sizeof(T)))) Eight {
    T x[PIECE];
};

template <class T>
__device__ inline void load8(const T* p, float (&x)[PIECE])
{
    const Eight<T> raw = *reinterpret_cast<const Eight<T>*>(p);
#pragma unroll
    for (int k = 0; k < PIECE; ++k)
        x[k] = static_cast<float>(raw.x[k]);
}

template <class T>
__device__ inline void store8(T* p, const float (&x)[PIECE])
{
    Eight<T> raw;
#pragma unroll
    for (int k = 0; k < PIECE; ++k)
        raw.x[k] = static_cast<T>(x[k]);
    *reinterpret_cast<Eight<T>*>(p) = raw;
}

} // namespace lm
