// The spans of a text's documents: for position i, lo = the last separator at or before it (0 if there is none), hi = i + 1, and the
// target text[i + 1], or -1 at the end and in front of a separator.
//
// 2 bytes in and 12 out a position: bound by memory. A running maximum of separator positions: up to 4096 tiles, each of a whole
// number of 4096-token turns; the first kernel leaves every tile's last separator (skipped where there is one tile), the second looks back over
// those of the tiles before its own, at most 16 loads a lane, and walks its tile with a scan of the workgroup a turn.
#pragma once
#include "lm_common.hpp"

namespace lm {

constexpr int SPAN_ITEMS = 16, SPAN_TURN = 256 * SPAN_ITEMS, SPAN_TILES = 4096;

__device__ inline void load_tokens(const uint16_t* text, int64_t n, int64_t at, bool wide, uint16_t (&t)[SPAN_ITEMS])
{
    if (wide && at + SPAN_ITEMS <= n) {
        *reinterpret_cast<u32x4*>(t) = *reinterpret_cast<const u32x4*>(text + at);
        *reinterpret_cast<u32x4*>(t + 8) = *reinterpret_cast<const u32x4*>(text + at + 8);
    } else {
        for (int i = 0; i < SPAN_ITEMS; ++i)
            t[i] = at + i < n ? text[at + i] : 0;
    }
}

__device__ inline int wave_max(int x)
{
    for (int d = 32; d; d /= 2) {
        const int y = __shfl_xor(x, d);
        x = y > x ? y : x;
    }
    return x;
}

__global__ __launch_bounds__(256) void last_separators_kernel(const uint16_t* text, int64_t n, uint16_t separator, int64_t tile, bool wide, int32_t* last)
{
    __shared__ int tops[4];
    int top = -1;
    const int64_t begin = blockIdx.x * tile, end = begin + tile < n ? begin + tile : n;
    for (int64_t at = begin + threadIdx.x * SPAN_ITEMS; at < end; at += SPAN_TURN) {
        alignas(16) uint16_t t[SPAN_ITEMS];
        load_tokens(text, n, at, wide, t);
        for (int i = 0; i < SPAN_ITEMS; ++i)
            if (t[i] == separator && at + i < n)
                top = static_cast<int>(at + i);
    }
    top = wave_max(top);
    if (threadIdx.x % 64 == 0)
        tops[threadIdx.x / 64] = top;
    __syncthreads();
    if (threadIdx.x == 0)
        last[blockIdx.x] = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
}

__global__ __launch_bounds__(256) void spans_kernel(const uint16_t* text, int64_t n, uint16_t separator, int64_t tile, bool wide, const int32_t* last, int32_t* lo,
                                                    int32_t* hi, int32_t* target)
{
    __shared__ int tops[2][4];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    int before = -1; // the last separator in front of the turn
    for (uint32_t t = threadIdx.x; t < blockIdx.x; t += 256)
        before = max(before, last[t]);
    before = wave_max(before);
    if (lane == 0)
        tops[1][wave] = before;
    __syncthreads();
    before = max(max(tops[1][0], tops[1][1]), max(tops[1][2], tops[1][3]));

    const int64_t begin = blockIdx.x * tile, end = begin + tile < n ? begin + tile : n;
    int turn = 0;
    for (int64_t first = begin; first < end; first += SPAN_TURN, turn ^= 1) {
        const int64_t at = first + threadIdx.x * SPAN_ITEMS;
        alignas(16) uint16_t t[SPAN_ITEMS + 1];
        uint16_t(&mine)[SPAN_ITEMS] = *reinterpret_cast<uint16_t(*)[SPAN_ITEMS]>(t);
        load_tokens(text, n, at, wide, mine);
        t[SPAN_ITEMS] = at + SPAN_ITEMS < n ? text[at + SPAN_ITEMS] : separator;
        int top = -1;
        for (int i = 0; i < SPAN_ITEMS; ++i)
            if (t[i] == separator && at + i < n)
                top = static_cast<int>(at + i);
        for (int d = 1; d < 64; d *= 2) {
            const int y = __shfl_up(top, d);
            if (lane >= d)
                top = max(top, y);
        }
        __syncthreads(); // the turn before last has been read
        if (lane == 63)
            tops[turn][wave] = top;
        __syncthreads();
        int own = __shfl_up(top, 1);
        own = lane ? max(own, before) : before;
        for (int w = 0; w < 4; ++w) {
            if (w < wave)
                own = max(own, tops[turn][w]);
            before = max(before, tops[turn][w]);
        }
        int32_t los[SPAN_ITEMS], his[SPAN_ITEMS], targets[SPAN_ITEMS];
        for (int i = 0; i < SPAN_ITEMS; ++i) {
            if (t[i] == separator)
                own = static_cast<int>(at + i);
            los[i] = max(own, 0);
            his[i] = static_cast<int32_t>(at + i + 1);
            targets[i] = at + i + 1 < n && t[i + 1] != separator ? t[i + 1] : -1;
        }
        if (wide && at + SPAN_ITEMS <= n) {
            for (int i = 0; i < SPAN_ITEMS; i += 4) {
                *reinterpret_cast<int4*>(lo + at + i) = *reinterpret_cast<int4*>(los + i);
                *reinterpret_cast<int4*>(hi + at + i) = *reinterpret_cast<int4*>(his + i);
                *reinterpret_cast<int4*>(target + at + i) = *reinterpret_cast<int4*>(targets + i);
            }
        } else {
            for (int i = 0; i < SPAN_ITEMS; ++i)
                if (at + i < n) {
                    lo[at + i] = los[i];
                    hi[at + i] = his[i];
                    target[at + i] = targets[i];
                }
        }
    }
}

} // namespace lm
