// The two products behind the logits' gradients P where there are at most 64 tokens: d_weight = P^T H and d_hidden = P W. Both are bound by memory, the one by writing a
// vocabulary's rows, the other by reading them, and take no barriers on the way: a wave walks words on its own, its next ones on their way while it multiplies.
//
// P comes in both orders: along the words (tokens x words, zeros behind the last word up to a multiple of 64) and along the tokens (words x 64, zeros for tokens that there are not).
// 61 tokens of 512 values, 50257 words: d_weight 13 us and d_hidden 15 (by the tiles of lm_product.hpp: 21 and 18, and twice as many shares to add up).
#pragma once
#include "lm_cross_entropy.hpp"

namespace lm {

constexpr int FEW_TOKENS = 64, FEW_DIMS = 128; // of a wave

// All of the wave's loads and LDS accesses are done; the compiler moves none across.
__device__ inline void settle()
{
    asm volatile("" ::: "memory");
    wait_for_all();
    asm volatile("" ::: "memory");
}

// d_weight: a wave has FEW_DIMS values of all tokens in registers and walks `words_each` words, 32 at a time: products of values and words, which it turns in LDS
// and stores as lines of a word.
template <class Type>
__global__ __launch_bounds__(256, 2) void few_weight_gradients_kernel(Operand hidden, const short* p_words, int tokens, int64_t words, int64_t words_each, uint32_t parts, uint32_t chunks,
                                                                   const float* scale, short* out, int64_t stride, bool wide)
{
    typedef Loader<FEW_DIMS, true, 1> Values;
    constexpr int TILES = FEW_DIMS / 32, STEPS = FEW_TOKENS / 16, PIECES = FEW_DIMS / 8;
    __shared__ __attribute__((aligned(16))) short all[4][FEW_DIMS * SLICE];
    const int lane = threadIdx.x % 64, half = lane / 32, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t id = blockIdx.x * 4 + wave;
    if (id >= parts * chunks) // whole waves, which meet nobody
        return;
    short* mine = all[wave];
    const int64_t d0 = static_cast<int64_t>(id % parts) * FEW_DIMS, begin = static_cast<int64_t>(id / parts) * words_each, end = begin + words_each < words ? begin + words_each : words;
    s16x8 values[STEPS][TILES];
    {
        Values load;
        load.begin(hidden, d0, 0, tokens, 0, lane);
        load.load(mine, 0, 0);
        Reader<FEW_DIMS, true, TILES> read;
        read.begin(0, lane);
        settle();
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
#pragma unroll
            for (int t = 0; t < TILES; ++t)
                values[s][t] = read.read(mine, t, s);
        wait_for_lds();
    }
    auto load_words = [&](s16x8 (&p)[STEPS], int64_t first) { // 32 words: those behind the last one are the last one again, not used
        const int64_t word = first + lane % 32 < words ? first + lane % 32 : words - 1;
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
            p[s] = read16(p_words + word * FEW_TOKENS + s * 16 + half * 8);
    };
    const float back = scale[1];
    const int piece = lane % PIECES;
    const int64_t d = d0 + piece * 8;
    s16x8 now[STEPS], next[STEPS];
    load_words(now, begin);
    for (int64_t first = begin; first < end; first += 32) {
        load_words(next, first + 32);
        f32x16 sums[TILES] = {};
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
            if (s * 16 < tokens)
#pragma unroll
                for (int t = 0; t < TILES; ++t)
                    sums[t] = Type::mfma32(values[s][t], now[s], sums[t]);
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

// One share of d_hidden: FEW_DIMS values of all tokens, over the words [share, share + words_each); the four waves take slices of 64 words in turn, and add up what they
// have at the end.
template <class Type>
__global__ __launch_bounds__(256) void few_hidden_gradients_kernel(const short* p, int64_t p_stride, Operand weight, int tokens, int64_t words, int64_t words_each, uint32_t parts,
                                                                   float* out, int64_t stride)
{
    typedef Loader<FEW_DIMS, true, 1> Words;
    constexpr int TILES = FEW_DIMS / 32, STEPS = SLICE / 16, ROWS = FEW_TOKENS / 32;
    __shared__ __attribute__((aligned(16))) short b0[4][FEW_DIMS * SLICE], b1[4][FEW_DIMS * SLICE];
    const int lane = threadIdx.x % 64, half = lane / 32, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t share = blockIdx.x / parts;
    const int64_t d0 = static_cast<int64_t>(blockIdx.x % parts) * FEW_DIMS, begin = share * words_each, end = begin + words_each < words ? begin + words_each : words;
    Reader<FEW_DIMS, true, TILES> read;
    read.begin(0, lane);
    f32x16 sums[ROWS][TILES] = {};
    struct Entries {
        s16x8 x[STEPS][ROWS];
    } now, next;
    // a slice of the weight on its way to LDS, and of P to registers
    auto load = [&](short* buffer, Entries& e, int64_t k0) {
        if (k0 >= end)
            return;
        Words w;
        w.begin(weight, d0, k0, end, 0, lane);
        w.load(buffer, k0, 0);
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
#pragma unroll
            for (int i = 0; i < ROWS; ++i) {
                const int token = 32 * i + lane % 32;
                e.x[s][i] = read16(p + (token < tokens ? token : tokens - 1) * p_stride + k0 + s * 16 + half * 8); // rows of tokens that there are not are not stored
            }
    };
    auto multiply = [&](const short* buffer, const Entries& e, int64_t k0) {
        if (k0 >= end)
            return;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            s16x8 w[TILES];
#pragma unroll
            for (int t = 0; t < TILES; ++t)
                w[t] = read.read(buffer, t, s);
#pragma unroll
            for (int i = 0; i < ROWS; ++i)
#pragma unroll
                for (int t = 0; t < TILES; ++t)
                    sums[i][t] = Type::mfma32(e.x[s][i], w[t], sums[i][t]);
        }
    };
    constexpr int64_t TURN = 4 * SLICE; // of all waves
    const int64_t first = begin + wave * SLICE;
    load(b0[wave], now, first);
    settle();
    for (int64_t k0 = first; k0 < end; k0 += 2 * TURN) { // two slices a turn, one from each buffer
        load(b1[wave], next, k0 + TURN);
        multiply(b0[wave], now, k0);
        settle();
        load(b0[wave], now, k0 + 2 * TURN);
        multiply(b1[wave], next, k0 + TURN);
        settle();
    }
    __syncthreads(); // no load is in flight
    // all sums in LDS, a wave's 32 KB after the other; then two tiles a wave
    constexpr int EACH = ROWS * TILES * 16 * 64;
    float* lines[4] = {reinterpret_cast<float*>(b0), reinterpret_cast<float*>(b0) + EACH, reinterpret_cast<float*>(b1), reinterpret_cast<float*>(b1) + EACH};
    static_assert(2 * EACH * sizeof(float) <= sizeof(b0), "two waves' sums fit a buffer");
    float* own = wave < 2 ? lines[0] + wave * EACH : lines[2] + (wave - 2) * EACH;
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                own[((i * TILES + t) * 16 + r) * 64 + lane] = sums[i][t][r];
    __syncthreads();
    constexpr int TILES_EACH = ROWS * TILES / 4;
    for (int k = 0; k < TILES_EACH; ++k) {
        const int tile = wave * TILES_EACH + k, i = tile / TILES, t = tile % TILES;
        const int64_t d = d0 + 32 * t + lane % 32;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int at = (tile * 16 + r) * 64 + lane, token = 32 * i + 8 * (r / 4) + 4 * half + r % 4;
            const float sum = (lines[0][at] + lines[1][at]) + (lines[2][at] + lines[3][at]);
            if (token < tokens && d < weight.rows)
                out[(static_cast<int64_t>(share) * tokens + token) * stride + d] = sum;
        }
    }
}

} // namespace lm
