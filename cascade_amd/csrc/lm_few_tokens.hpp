// The two products behind the logits' gradients P where there are at most 64 tokens: d_weight = P^T H and d_hidden = P W. Both are bound by memory, the one by writing a
// vocabulary's rows, the other by reading them, and take no barriers on the way: a wave walks words on its own, its next ones on their way while it multiplies.
//
// P comes in both orders: along the words (tokens x words, zeros behind the last word up to a multiple of 64) and along the tokens (words x 32 or 64, zeros for tokens that there are
// not). It is the sum of two numbers of 16 bits, what the rounding leaves being the second one, in rows of its own and behind the first ones of a word. With one number its rounding and the
// results' own add up to 1.4 times the latter where entries are many, but a short text's errors are those of a few entries, its tokens' likeliest words, and spread about that: up to 1.6 times.
// For up to 32 tokens the second number takes the places of tokens that are not there, and no time. For 33 to 64 it is read and multiplied where it matters, in blocks of 64 words that
// hold an entry above an eighth of its token's weight: errors of 1.00 to 1.18 times, where those entries make most of the sums, for 7 % of the time (61 tokens of 512 values trained 80 -> 85 us,
// 40 of 2560 260 -> 265); in all blocks it would be 12 and 9 %. An entry is held against its own token's weight, since a row of d_hidden is as large as that: 64 tokens of 512 values whose weights differ
// by up to 2^10 take 86 us, 83 if only entries above an eighth of the largest weight counted, which left the rows of the others with errors of about twice the rounding.
// d_weight of 61 tokens of 512 values and 50257 words takes 16 us, of 40 of 2560 58 us, of 3 of 4096 73 us, 5.6 TB/s (by the tiles of lm_product.hpp, with one number, 21, 77 and 118: one
// workgroup a compute unit, which waits for its loads, multiplies and stores one after the other). d_hidden reads the weight behind what has just been written: 18 and 86 us, by tiles the
// same, but 6 us instead of 34 over 3000 words, whose tiles are too few.
#pragma once
#include "lm_cross_entropy.hpp"

namespace lm {

constexpr int FEW_TOKENS = 64; // at most
constexpr int FEW_DIMS = 128;                     // of a wave

// All of the wave's loads and LDS accesses are done; the compiler moves none across.
__device__ inline void settle()
{
    asm volatile("" ::: "memory");
    wait_for_all();
    asm volatile("" ::: "memory");
}

// d_weight: a wave has FEW_DIMS values of all tokens in registers and walks `words_each` words, 32 at a time: products of values and words, which it turns in LDS
// and stores as lines of a word.
template <class Type, int TOKENS>
__global__ __launch_bounds__(256, 2) void few_weight_gradients_kernel(Operand hidden, const short* p_words, const uint32_t* __restrict__ heavy, int tokens, int64_t words, int64_t words_each, uint32_t parts, uint32_t chunks,
                                                                   const float* scale, short* out, int64_t stride, bool wide)
{
    typedef Loader<FEW_DIMS, true, 1> Values;
    constexpr int TILES = FEW_DIMS / 32, STEPS = TOKENS / 8, KINDS = TOKENS / 16, PIECES = FEW_DIMS / 8;
    __shared__ __attribute__((aligned(16))) short all[4][FEW_DIMS * SLICE];
    const int lane = threadIdx.x % 64, half = lane / 32, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    // lines of memory that two waves share are written by one XCD (61 tokens of 968 values 155 -> 151 us trained; where there are none it takes 1 % more of 4096 values)
    const uint32_t id = (stride % 64 ? by_xcd(blockIdx.x, gridDim.x) : blockIdx.x) * 4 + wave;
    if (id >= parts * chunks) // whole waves, which meet nobody
        return;
    short* mine = all[wave];
    const int64_t d0 = static_cast<int64_t>(id % parts) * FEW_DIMS, begin = static_cast<int64_t>(id / parts) * words_each, end = begin + words_each < words ? begin + words_each : words;
    s16x8 values[KINDS][TILES]; // with two numbers of P the tokens come twice
    {
        Values load;
        load.begin(hidden, d0, 0, tokens, 0, lane);
        load.load(mine, 0, 0);
        Reader<FEW_DIMS, true, TILES> read;
        read.begin(0, lane);
        settle();
#pragma unroll
        for (int s = 0; s < KINDS; ++s)
#pragma unroll
            for (int t = 0; t < TILES; ++t)
                values[s][t] = read.read(mine, t, s);
        wait_for_lds();
    }
    auto load_words = [&](s16x8 (&p)[STEPS], int64_t first, uint32_t twice) { // 32 words: those behind the last one are the last one again, not used
        const int64_t word = first + lane % 32 < words ? first + lane % 32 : words - 1;
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
            if (s < KINDS || twice)
                p[s] = read16(p_words + word * (2 * TOKENS) + s * 16 + half * 8);
    };
    auto load_heavy = [&](int64_t first) -> uint32_t { return TOKENS == FEW_TOKENS ? heavy[(first < words ? first : words - 1) / SLICE] : 1; };
    const float back = scale[1];
    const int piece = lane % PIECES;
    const int64_t d = d0 + piece * 8;
    s16x8 now[STEPS], next[STEPS];
    uint32_t twice = load_heavy(begin), after = load_heavy(begin + 32);
    load_words(now, begin, twice);
    for (int64_t first = begin; first < end; first += 32) {
        const uint32_t next_twice = after;
        load_words(next, first + 32, next_twice);
        after = load_heavy(first + 64);
        f32x16 sums[TILES] = {};
#pragma unroll
        for (int s = 0; s < KINDS; ++s)
#pragma unroll
            for (int t = 0; t < TILES; ++t)
                sums[t] = Type::mfma32(values[s][t], now[s], sums[t]);
        if (twice)
#pragma unroll
            for (int s = 0; s < KINDS; ++s)
#pragma unroll
                for (int t = 0; t < TILES; ++t)
                    sums[t] = Type::mfma32(values[s][t], now[KINDS + s], sums[t]);
        twice = next_twice;
        const int column = lane % 32; // a line holds a word's values; its pieces stand at places piece ^ word
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                s16x4 y;
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    y[r] = to16<Type>(sums[t][4 * g + r] * back);
                *reinterpret_cast<s16x4*>(mine + column * FEW_DIMS + ((4 * t + g) ^ column % PIECES) * 8 + 4 * half) = y;
            }
        wait_for_lds();
#pragma unroll
        for (int c = 0; c < 32; c += 64 / PIECES) {
            const int word = c + lane / PIECES;
            const s16x8 y = read16(mine + word * FEW_DIMS + (piece ^ word % PIECES) * 8);
            if (first + word >= end || d >= hidden.rows)
                continue;
            short* to = out + (first + word) * stride + d;
            if (wide && d + 8 <= hidden.rows) {
                *reinterpret_cast<s16x8*>(to) = y;
            } else {
                for (int r = 0; r < 8; ++r)
                    if (d + r < hidden.rows)
                        to[r] = y[r];
            }
        }
        wait_for_lds();
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
            now[s] = next[s];
    }
}

// One share of d_hidden: FEW_DIMS values of 32 ROWS tokens, over words_each words; the four waves take 64 words in turn (a line of P), and add up what they have at the end. A wave loads
// words as they lie, four neighbouring values a lane, 16 words at a time and DEPTH times as many on their way, and turns blocks of eight words by four
// values in its registers: the k-th product of a step has the k-th of every lane's values.
template <class Type, int ROWS>
__global__ __launch_bounds__(256, 1) void few_hidden_gradients_kernel(const short* p, const short* p_low, const uint32_t* heavy, int64_t p_stride, Operand weight, int tokens, int64_t words, int64_t words_each, uint32_t parts,
                                                                      float* out, int64_t stride)
{
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    constexpr int DEPTH = 4, STEP = 16, VALUES = 4;
    __shared__ f32x4 all[4][ROWS * 16 * 64];
    const int lane = threadIdx.x % 64, half = lane / 32, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t id = by_xcd(blockIdx.x, gridDim.x), share = id / parts; // the parts that read the same of P: by way of one L2 (61 tokens of 512 values trained 82 -> 80 us, of 1000 138 -> 126)
    const int64_t d0 = static_cast<int64_t>(id % parts) * FEW_DIMS, begin = share * words_each, end = begin + words_each < words ? begin + words_each : words;
    const int64_t line = weight.stride * 2;
    const int64_t d = d0 + VALUES * (lane % 32);
    const bool there = d < stride; // of the row's values, up to a multiple of eight
    const uint32_t offset = there ? static_cast<uint32_t>(8 * half * line + VALUES * (lane % 32) * 2) : OUTSIDE;
    f32x16 sums[ROWS][VALUES] = {};
    struct Step {
        u32x2 w[8];
        s16x8 p[2][ROWS]; // both numbers of 32 tokens each
    } steps[DEPTH];
    auto load = [&](Step& s, int64_t k0, bool twice) { // behind the end: zeros, by an empty window, and any P
        const int64_t left = end - k0, bytes = (left < STEP ? left : STEP) * line - d0 * 2;
        const buffer_t rows = window(static_cast<const char*>(weight.data) + k0 * line + d0 * 2, left > 0 ? static_cast<uint32_t>(bytes) : 0);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            s.w[i] = __builtin_amdgcn_raw_buffer_load_b64(rows, static_cast<int>(offset + (there ? i * static_cast<uint32_t>(line) : 0)), 0, 0);
        const int64_t k = left > 0 ? k0 : begin;
        int64_t at[ROWS];
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const int token = 32 * i + lane % 32;
            at[i] = (token < tokens ? token : tokens - 1) * p_stride + k + 8 * half; // rows of tokens that there are not are not stored
            s.p[0][i] = read16(p + at[i]);
        }
        if (twice)
#pragma unroll
            for (int i = 0; i < ROWS; ++i)
                s.p[1][i] = read16(p_low + at[i]);
    };
    auto multiply_by = [&](const Step& s, const s16x8 (&p)[ROWS]) {
#pragma unroll
        for (int k = 0; k < VALUES; ++k) {
            u32x4 turned;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                turned[i] = __builtin_amdgcn_perm(s.w[2 * i + 1][k / 2], s.w[2 * i][k / 2], k % 2 ? 0x07060302 : 0x05040100);
#pragma unroll
            for (int i = 0; i < ROWS; ++i)
                sums[i][k] = Type::mfma32(p[i], __builtin_bit_cast(s16x8, turned), sums[i][k]);
        }
    };
    auto multiply = [&](const Step& s, bool twice) {
        multiply_by(s, s.p[0]);
        if (twice)
            multiply_by(s, s.p[1]);
    };
    static_assert(DEPTH * STEP == SLICE, "a turn's words of a wave");
    const int64_t first = begin + wave * SLICE;
    auto load_heavy = [&](int64_t k0) -> uint32_t { return ROWS == 2 ? heavy[(k0 < words ? k0 : words - 1) / SLICE] : 1; };
    uint32_t after = load_heavy(first + 4 * SLICE);
    bool twice = __builtin_amdgcn_readfirstlane(load_heavy(first));
#pragma unroll
    for (int s = 0; s < DEPTH; ++s)
        load(steps[s], first + s * STEP, twice);
    for (int64_t k0 = first; k0 < end; k0 += 4 * SLICE) {
        const bool next_twice = __builtin_amdgcn_readfirstlane(after);
        after = load_heavy(k0 + 8 * SLICE);
#pragma unroll
        for (int s = 0; s < DEPTH; ++s) {
            if (k0 + s * STEP < end)
                multiply(steps[s], twice);
            load(steps[s], k0 + 4 * SLICE + s * STEP, next_twice);
        }
        twice = next_twice;
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r)
            all[wave][(i * 16 + r) * 64 + lane] = f32x4{sums[i][0][r], sums[i][1][r], sums[i][2][r], sums[i][3][r]};
    __syncthreads();
    for (int k = 0; k < ROWS * 4; ++k) { // a quarter of the rows a wave
        const int row = wave * ROWS * 4 + k, i = row / 16, r = row % 16, token = 32 * i + 8 * (r / 4) + 4 * half + r % 4, at = row * 64 + lane;
        if (token < tokens && there)
            *reinterpret_cast<f32x4*>(out + (static_cast<int64_t>(share) * tokens + token) * stride + d) = (all[0][at] + all[1][at]) + (all[2][at] + all[3][at]);
    }
}

} // namespace lm
