// The spans of a text's documents: for position i, lo = the last separator at or before it (0 if there is none), hi = i + 1, and the
// target text[i + 1], or -1 at the end and in front of a separator.
//
// 2 bytes in and 12 out a position: bound by memory. A running maximum of separator positions: up to 4096 tiles, each of a whole
// number of 4096-token turns; the first kernel leaves every tile's last separator (skipped where there is one tile), the second looks back over
// those of the tiles before its own, at most 16 loads a lane, and walks its tile with a scan of the workgroup a turn. Lanes hold four neighbouring
// tokens of every 1024, so that a wave's stores are whole lines.
// 16777213 tokens: 9 + 40 us, 4.5 TB/s of those 14 bytes (a large copy does 4.8).
#pragma once
#include "lm_common.hpp"

namespace lm {

constexpr int SPAN_GROUPS = 4, SPAN_TURN = 256 * 4 * SPAN_GROUPS, SPAN_TILES = 4096; // a lane has four tokens of every 1024

__device__ inline void load_tokens(const uint16_t* text, int64_t n, int64_t at, bool wide, uint16_t (&t)[4])
{
    if (wide && at + 4 <= n) {
        const uint64_t x = *reinterpret_cast<const uint64_t*>(text + at);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            t[i] = static_cast<uint16_t>(x >> 16 * i);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            t[i] = at + i < n ? text[at + i] : 0;
    }
}

// The last separator among a lane's four tokens, -1 if there is none.
__device__ inline int last_of(const uint16_t (&t)[4], int64_t at, int64_t n, uint16_t separator)
{
    int last = -1;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        last = t[i] == separator && at + i < n ? static_cast<int>(at + i) : last;
    return last;
}

__device__ inline int largest(int x)
{
    for (int d = 32; d; d /= 2)
        x = max(x, __shfl_xor(x, d));
    return x;
}

__global__ __launch_bounds__(256) void last_separators_kernel(const uint16_t* text, int64_t n, uint16_t separator, int64_t tile, bool wide, int32_t* last)
{
    __shared__ int tops[4];
    int top = -1;
    const int64_t begin = blockIdx.x * tile, end = begin + tile < n ? begin + tile : n;
    for (int64_t first = begin; first < end; first += SPAN_TURN) {
        uint16_t t[SPAN_GROUPS][4];
#pragma unroll
        for (int g = 0; g < SPAN_GROUPS; ++g)
            load_tokens(text, n, first + g * 1024 + threadIdx.x * 4, wide, t[g]);
#pragma unroll
        for (int g = 0; g < SPAN_GROUPS; ++g)
            top = max(top, last_of(t[g], first + g * 1024 + threadIdx.x * 4, n, separator));
    }
    top = largest(top);
    if (threadIdx.x % 64 == 0)
        tops[threadIdx.x / 64] = top;
    __syncthreads();
    if (threadIdx.x == 0)
        last[blockIdx.x] = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
}

__global__ __launch_bounds__(256) void spans_kernel(const uint16_t* text, int64_t n, uint16_t separator, int64_t tile, bool wide, const int32_t* last, int32_t* lo,
                                                    int32_t* hi, int32_t* target)
{
    __shared__ int tops[2][SPAN_GROUPS][4];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    int before = -1; // the last separator in front of the turn
    for (uint32_t t = threadIdx.x; t < blockIdx.x; t += 256)
        before = max(before, last[t]);
    before = largest(before);
    if (lane == 0)
        tops[1][0][wave] = before;
    __syncthreads();
    before = max(max(tops[1][0][0], tops[1][0][1]), max(tops[1][0][2], tops[1][0][3]));

    const int64_t begin = blockIdx.x * tile, end = begin + tile < n ? begin + tile : n;
    int turn = 0;
    for (int64_t first = begin; first < end; first += SPAN_TURN, turn ^= 1) {
        uint16_t t[SPAN_GROUPS][4];
        uint16_t next[SPAN_GROUPS]; // the token behind a lane's four
        int top[SPAN_GROUPS], own[SPAN_GROUPS];
#pragma unroll
        for (int g = 0; g < SPAN_GROUPS; ++g) {
            const int64_t at = first + g * 1024 + threadIdx.x * 4;
            load_tokens(text, n, at, wide, t[g]);
            next[g] = at + 4 < n ? text[at + 4] : separator;
        }
#pragma unroll
        for (int g = 0; g < SPAN_GROUPS; ++g) {
            top[g] = last_of(t[g], first + g * 1024 + threadIdx.x * 4, n, separator);
            for (int d = 1; d < 64; d *= 2) {
                const int y = __shfl_up(top[g], d);
                top[g] = lane >= d ? max(top[g], y) : top[g];
            }
        }
        __syncthreads(); // what the turn before last left has been read
        if (lane == 63)
#pragma unroll
            for (int g = 0; g < SPAN_GROUPS; ++g)
                tops[turn][g][wave] = top[g];
        __syncthreads();
#pragma unroll
        for (int g = 0; g < SPAN_GROUPS; ++g) {
            own[g] = __shfl_up(top[g], 1);
            own[g] = lane ? max(own[g], before) : before;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const int x = tops[turn][g][w];
                own[g] = w < wave ? max(own[g], x) : own[g];
                before = max(before, x);
            }
        }
#pragma unroll
        for (int g = 0; g < SPAN_GROUPS; ++g) {
            const int64_t at = first + g * 1024 + threadIdx.x * 4;
            int los[4], his[4], targets[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                own[g] = t[g][i] == separator ? static_cast<int>(at + i) : own[g];
                const uint16_t follows = i < 3 ? t[g][i + 1] : next[g];
                los[i] = max(own[g], 0);
                his[i] = static_cast<int>(at + i + 1);
                targets[i] = at + i + 1 < n && follows != separator ? follows : -1;
            }
            if (wide && at + 4 <= n) {
                *reinterpret_cast<int4*>(lo + at) = make_int4(los[0], los[1], los[2], los[3]);
                *reinterpret_cast<int4*>(hi + at) = make_int4(his[0], his[1], his[2], his[3]);
                *reinterpret_cast<int4*>(target + at) = make_int4(targets[0], targets[1], targets[2], targets[3]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (at + i < n) {
                        lo[at + i] = los[i];
                        hi[at + i] = his[i];
                        target[at + i] = targets[i];
                    }
            }
        }
    }
}

} // namespace lm
