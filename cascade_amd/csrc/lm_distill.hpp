// Distillation from the logits that a teacher kept of every token: with z = hidden weight^T / T over the vocabulary and q the teacher's softmax
// over its own logits / T, wherever it has some,
//   loss = sum over the kept words of q (ln q - z) + ln sum exp z,   d_z = d_loss / T (softmax(z) - q).
//
// The cross entropy's path (lm_cross_entropy.hpp) with many targets a token instead of one: the same tile products, without logits that are kept. A first kernel makes q,
// sorts every token's words and notes where each block of words (those that a wave's part of a tile holds) begins among them. A
// tile that is done lays its logits, or their exponentials, into LDS in 32 bits, a line of words for each token, and the token's lanes pick theirs there, or take q off
// before anything is rounded: p - q, which a student that has learnt leaves small, keeps all its bits.
#pragma once
#include "lm_few_tokens.hpp"

namespace lm {

constexpr uint32_t MOST_KEPT = 1024; // logits of a token

// Entries of a token in the order of their words; those of block b stand at first[b] to first[b + 1].
struct Teacher {
    const int32_t* ids;    // tokens x kept
    const float* q;        // tokens x kept
    const uint16_t* first; // tokens x (blocks + 1)
    int64_t kept, blocks;
};

// WAVES a token, ITEMS entries a lane. words_each: of a block. Entries are ranked by comparing all with all (one token of 256: 12 us with four
// waves, 31 with one; 2999 of 100: 23 us with four waves, 17 with one, whose lanes have two each).
template <int WAVES, int ITEMS>
__global__ __launch_bounds__(256) void teacher_kernel(const int32_t* ids, const float* logits, int64_t tokens, int kept, int64_t vocab, float rate, int words_each, int64_t blocks,
                                                      int32_t* sorted_ids, float* sorted_q, uint16_t* first, int32_t* counts, float* entropy)
{
    constexpr int LANES = WAVES * 64, TOKENS = 4 / WAVES;
    constexpr uint32_t NONE = 0xffffffffu; // behind all words
    __shared__ __attribute__((aligned(16))) uint32_t all_words[TOKENS][ITEMS * LANES];
    __shared__ uint32_t all_sorted[TOKENS][ITEMS * LANES];
    __shared__ float all_q[TOKENS][ITEMS * LANES];
    __shared__ float joined[4][WAVES];
    const int lane = threadIdx.x % LANES, which = threadIdx.x / LANES;
    const int64_t n = static_cast<int64_t>(blockIdx.x) * TOKENS + which;
    if (n >= tokens) // whole waves, which meet nobody
        return;
    uint32_t *words = all_words[which], *sorted = all_sorted[which];
    float* qs = all_q[which];
    int turn = 0;
    // one value of all lanes from one of each: the waves' by way of LDS, where there are more than one
    auto over_lanes = [&](float x, auto join) {
        for (int d = 32; d; d /= 2)
            x = join(x, __shfl_xor(x, d));
        if (WAVES > 1) {
            if (threadIdx.x % 64 == 0)
                joined[turn][threadIdx.x / 64] = x;
            __syncthreads();
            x = joined[turn][0];
            for (int w = 1; w < WAVES; ++w)
                x = join(x, joined[turn][w]);
            ++turn;
        }
        return x;
    };
    auto larger = [](float x, float y) { return fmaxf(x, y); };
    auto sum_of = [](float x, float y) { return x + y; };
    uint32_t word[ITEMS], rank[ITEMS];
    float told[ITEMS], top = -INFINITY, here = 0;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const int k = i * LANES + lane;
        const int32_t id = k < kept ? ids[n * kept + k] : -1;
        told[i] = id >= 0 && id < vocab ? logits[n * kept + k] : -INFINITY;
        word[i] = told[i] == -INFINITY ? NONE : static_cast<uint32_t>(id); // nothing is told: no entry
        here += word[i] != NONE;
        top = fmaxf(top, told[i]);
        rank[i] = 0;
        words[k] = word[i];
    }
    top = over_lanes(top, larger);
    const int there = static_cast<int>(over_lanes(here, sum_of));
    float sum = 0, part = 0;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        told[i] = (told[i] - top) * rate; // in this order nothing finite becomes infinite but what has no weight
        sum += word[i] != NONE ? expf(told[i]) : 0.f;
    }
    sum = over_lanes(sum, sum_of);
    const float all = logf(sum);
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const float q = expf(told[i]) / sum;
        part += word[i] != NONE && told[i] != -INFINITY ? q * (told[i] - all) : 0.f;
        told[i] = q;
    }
    part = over_lanes(part, sum_of);
    if (lane == 0) {
        counts[n] = there ? 0 : -1;
        entropy[n] = part;
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll 4
    for (int j = 0; j < kept; j += 4) { // entries of one word stay in their order
        const u32x4 others = *reinterpret_cast<const u32x4*>(words + j);
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int i = 0; i < ITEMS; ++i)
                rank[i] += others[k] < word[i] || (others[k] == word[i] && j + k < i * LANES + lane);
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
        if (word[i] != NONE) {
            sorted[rank[i]] = word[i];
            qs[rank[i]] = told[i];
        }
    if (WAVES > 1)
        __syncthreads();
    __builtin_amdgcn_wave_barrier();
    for (int k = lane; k < there; k += LANES) {
        sorted_ids[n * kept + k] = static_cast<int32_t>(sorted[k]);
        sorted_q[n * kept + k] = qs[k];
    }
    for (int64_t b = lane; b <= blocks; b += LANES) {
        int lo = 0, hi = there; // the first entry whose word is of block b or behind it
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (sorted[mid] < b * words_each)
                lo = mid + 1;
            else
                hi = mid;
        }
        first[n * (blocks + 1) + b] = static_cast<uint16_t>(lo);
    }
}

// What a wave's part of a tile is to the teacher: 32 tokens at a time, a line of LINE words in 32 bits for each, in pieces of four that stand at
// places piece ^ token, so that lanes of different tokens reach different banks.
template <class P>
struct Lines {
    static constexpr int LINE = P::BM / P::WM, PIECES = LINE / 4, SIZE = LINE * 32;
    static_assert((PIECES & (PIECES - 1)) == 0, "places are a permutation");

    // A wave's region, from the buffers of the operands.
    static __device__ float* region(short* a0, short* a1, short* b0, short* b1)
    {
        constexpr int IN_A = P::BM * SLICE / 2 / SIZE, IN_B = P::BN * SLICE / 2 / SIZE;
        static_assert(2 * IN_A + 2 * IN_B >= P::WAVES, "the lines fit the buffers");
        const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
        short* base = w < IN_A ? a0 : w < 2 * IN_A ? a1 : w < 2 * IN_A + IN_B ? b0 : b1;
        const int in = w < IN_A ? w : w < 2 * IN_A ? w - IN_A : w < 2 * IN_A + IN_B ? w - 2 * IN_A : w - 2 * IN_A - IN_B;
        return reinterpret_cast<float*>(base) + in * SIZE;
    }
    static __device__ float* piece(float* lines, int token, int k) { return lines + token * LINE + (k ^ (token & (PIECES - 1))) * 4; }
    static __device__ float& word(float* lines, int token, int w) { return piece(lines, token, w / 4)[w % 4]; }

    // value(word, x) of tile column j
    template <class F>
    static __device__ void put(float* lines, const typename P::Sums& sums, int j, F value)
    {
        const int lane = threadIdx.x % 64, half = lane / 32;
#pragma unroll
        for (int i = 0; i < P::TM; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                f32x4 y;
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    y[r] = value(sums[i][j][4 * g + r]);
                *reinterpret_cast<f32x4*>(piece(lines, lane % 32, 8 * i + 2 * g + half)) = y;
            }
    }
};

struct Listed { // a token's entries in a wave's words
    int begin, end;
};

__device__ inline Listed listed(const Teacher& t, int64_t n, bool there, int64_t block)
{
    if (!there || block >= t.blocks)
        return {0, 0};
    const uint16_t* first = t.first + n * (t.blocks + 1) + block;
    return {first[0], first[1]};
}

template <class P>
__global__ __launch_bounds__(P::THREADS) void distill_sums_kernel(Logits l, Teacher teacher, float rate, float2* part, float* dots)
{
    LM_TILE_BUFFERS(P);
    typedef Lines<P> Words;
    uint32_t mi, ni;
    tile_of(blockIdx.x, l.mt, l.nt, mi, ni);
    typename P::Sums sums;
    const int64_t m0 = static_cast<int64_t>(mi) * P::BM, n0 = static_cast<int64_t>(ni) * P::BN;
    P::run(l.weight, l.hidden, m0, n0, 0, l.dim, a0, a1, b0, b1, sums);
    const int lane = threadIdx.x % 64, half = lane / 32;
    const int64_t tokens = l.hidden.rows, mw = m0 + P::wave_m(), rows = l.weight.rows - mw, block = mw / Words::LINE;
    const int left = static_cast<int>(rows < Words::LINE ? rows : Words::LINE) - 4 * half; // this lane's words there are: row < left
    float* lines = Words::region(a0, a1, b0, b1);
    meet(); // everybody has read the last slice
#pragma unroll
    for (int j = 0; j < P::TN; ++j) {
        const int64_t n = n0 + P::wave_n() + 32 * j + lane % 32;
        const bool there = n < tokens;
        const Listed mine = listed(teacher, n, there, block);
        float dot = 0;
        if (__any(mine.end > mine.begin)) {
            Words::put(lines, sums, j, [](float x) { return x; });
            wait_for_lds();
            for (int e = mine.begin + half; e < mine.end; e += 2)
                dot += teacher.q[n * teacher.kept + e] * Words::word(lines, lane % 32, static_cast<int>(teacher.ids[n * teacher.kept + e] - mw));
            dot += other_half(dot);
        }
        if (rows < Words::LINE) // words past the end, in a few tiles only
#pragma unroll
            for (int i = 0; i < P::TM; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (32 * i + 8 * (r / 4) + r % 4 >= left)
                        sums[i][j][r] = -INFINITY;
        float top = -3.0e38f;
#pragma unroll
        for (int i = 0; i < P::TM; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                top = fmaxf(top, sums[i][j][r]);
        const float steps = rate * LOG2E;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < P::TM; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                sum += __builtin_amdgcn_exp2f((sums[i][j][r] - top) * steps);
        const float top2 = other_half(top), sum2 = other_half(sum), high = fmaxf(top, top2);
        sum = sum * __builtin_amdgcn_exp2f((top - high) * steps) + sum2 * __builtin_amdgcn_exp2f((top2 - high) * steps);
        if (there && half == 0) {
            const int64_t at = (static_cast<int64_t>(mi) * P::WM + P::wave_m() / Words::LINE) * tokens + n;
            part[at] = make_float2(high * rate, sum);
            dots[at] = dot * rate;
        }
    }
}

// lse and loss from the waves' maxima, sums and products with q: TOKENS tokens by 256 / TOKENS runs of them a workgroup.
template <int TOKENS>
__global__ __launch_bounds__(256) void join_distill_kernel(const float2* part, const float* dots, int64_t parts, const int32_t* counts, const float* entropy, int64_t tokens,
                                                           float* loss, float* lse)
{
    constexpr int RUNS = 256 / TOKENS;
    __shared__ float2 got[RUNS][TOKENS + 1];
    __shared__ float got_dots[RUNS][TOKENS + 1];
    const int x = threadIdx.x % TOKENS, y = threadIdx.x / TOKENS;
    const int64_t n = static_cast<int64_t>(blockIdx.x) * TOKENS + x;
    const float2 none = make_float2(-3.0e38f, 0.f);
    float2 sum = none;
    float dot = 0;
    if (n < tokens)
        for (int64_t p = y; p < parts; p += 8 * RUNS) {
            float2 v[8];
            float d[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const bool there = p + k * RUNS < parts;
                v[k] = there ? part[(p + k * RUNS) * tokens + n] : none;
                d[k] = there ? dots[(p + k * RUNS) * tokens + n] : 0.f;
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                add_exponentials(sum, v[k]);
                dot += d[k];
            }
        }
    got[y][x] = sum;
    got_dots[y][x] = dot;
    for (int far = RUNS / 2; far; far /= 2) {
        __syncthreads();
        if (y < far) {
            add_exponentials(sum, got[y + far][x]);
            dot += got_dots[y + far][x];
            got[y][x] = sum;
            got_dots[y][x] = dot;
        }
    }
    if (y == 0 && n < tokens) {
        const float all = sum.x + logf(sum.y);
        lse[n] = all;
        loss[n] = counts[n] >= 0 ? entropy[n] - dot + all : 0.f;
    }
}

// What few tokens take beside P (lm_few_tokens.hpp).
struct FewGradients {
    short *by_words, *low; // P and what its rounding leaves in the other order, in rows of `width` tokens each, or null; what the rounding leaves in P's order
    int width;
    uint16_t* heavy; // two a block of 64 words, for 32 tokens each: whether an entry there is larger than an eighth of its token's weight
};

// P[n][v] = d_loss[n] (exp(z - lse[n]) - q) relative to the largest |d_loss|, as logit_gradients_kernel leaves it; 1 / T is in what the products are scaled back with.
// FEW: of few tokens.
template <class P, class Type, bool FEW>
__global__ __launch_bounds__(P::THREADS) void distill_gradients_kernel(Logits l, Teacher teacher, float rate, const float* lse, const float* d_loss, const float* scale,
                                                                       short* out, int64_t stride, FewGradients few)
{
    LM_TILE_BUFFERS(P);
    typedef Lines<P> Words;
    uint32_t mi, ni;
    tile_of(blockIdx.x, l.mt, l.nt, mi, ni);
    typename P::Sums sums;
    const int64_t m0 = static_cast<int64_t>(mi) * P::BM, n0 = static_cast<int64_t>(ni) * P::BN;
    P::run(l.weight, l.hidden, m0, n0, 0, l.dim, a0, a1, b0, b1, sums);
    const int lane = threadIdx.x % 64;
    const int64_t tokens = l.hidden.rows, mw = m0 + P::wave_m(), word0 = l.first_word + mw;
    float* lines = Words::region(a0, a1, b0, b1);
    meet(); // everybody has read the last slice
    constexpr int EIGHTS = Words::LINE / 8;
    const int eight = lane % EIGHTS;
    const int64_t m = mw + eight * 8;
    static_assert(!FEW || Words::LINE == SLICE, "a line of P is a wave's");
#pragma unroll
    for (int j = 0; j < P::TN; ++j) {
        const int64_t first = n0 + P::wave_n() + 32 * j, n = first + lane % 32;
        const bool counts = n < tokens && l.target[n] >= 0;
        const float factor = counts ? d_loss[n] * scale[0] : 0.f, shift = counts ? lse[n] : 0.f;
        const Listed mine = listed(teacher, n, counts, word0 / Words::LINE);
        Words::put(lines, sums, j, [&](float x) { return counts ? __builtin_amdgcn_exp2f(fmaf(x, rate, -shift) * LOG2E) * factor : 0.f; }); // tokens left out: zeros, whatever their logits are
        if (__any(mine.end > mine.begin)) {
            wait_for_lds();
            if (lane < 32) // one lane a token: a word may be listed twice
                for (int e = mine.begin; e < mine.end; ++e)
                    Words::word(lines, lane, static_cast<int>(teacher.ids[n * teacher.kept + e] - word0)) -= teacher.q[n * teacher.kept + e] * factor;
        }
        wait_for_lds();
        if (FEW && few.by_words && n < few.width)
            for (int k = 0; k < Words::PIECES; k += 2) { // four words a lane
                const int piece = k + lane / 32;
                const f32x4 y = *reinterpret_cast<const f32x4*>(Words::piece(lines, lane % 32, piece));
                for (int r = 0; r < 4; ++r)
                    if (mw + 4 * piece + r < l.weight.rows) {
                        short* to = few.by_words + (mw + 4 * piece + r) * (2 * few.width) + n;
                        const short rounded = to16<Type>(y[r]);
                        to[0] = rounded;
                        to[few.width] = to16<Type>(y[r] - to32<Type>(rounded));
                    }
            }
        bool heavy = false;
#pragma unroll
        for (int c = 0; c < 32; c += 64 / EIGHTS) {
            const int token = c + lane / EIGHTS;
            const float least = FEW ? fabsf(__shfl(factor, token)) * 0.125f : 0.f;
            const f32x4 front = *reinterpret_cast<const f32x4*>(Words::piece(lines, token, 2 * eight)), back = *reinterpret_cast<const f32x4*>(Words::piece(lines, token, 2 * eight + 1));
            s16x8 y, rest = {};
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                const float x = r < 4 ? front[r] : back[r - 4];
                y[r] = to16<Type>(x);
                if (FEW) {
                    rest[r] = to16<Type>(x - to32<Type>(y[r]));
                    heavy |= fabsf(x) > least; // never of infinite weights, which change nothing for other tokens
                }
            }
            if (first + token >= tokens || m >= l.weight.rows)
                continue;
            const int64_t to = (first + token) * stride + m;
            if (m + 8 <= l.weight.rows) {
                *reinterpret_cast<s16x8*>(out + to) = y;
                if (FEW)
                    *reinterpret_cast<s16x8*>(few.low + to) = rest;
            } else {
                for (int r = 0; r < 8; ++r)
                    if (m + r < l.weight.rows) {
                        out[to + r] = y[r];
                        if (FEW)
                            few.low[to + r] = rest[r];
                    }
            }
        }
        if (FEW) {
            const bool some = __any(heavy);
            if (lane == 0 && mw < l.weight.rows)
                few.heavy[mw / SLICE * 2 + first / 32] = some;
        }
        wait_for_lds();
    }
    // k of the products to come runs along these rows, to a multiple of 8, or of 64
    if (mi == l.mt - 1)
        for (int64_t tail = l.weight.rows + threadIdx.x % 8; tail < stride; tail += 8)
            for (int64_t n = n0 + threadIdx.x / 8; n < n0 + P::BN && n < tokens; n += P::THREADS / 8) {
                out[n * stride + tail] = 0;
                if (FEW)
                    few.low[n * stride + tail] = 0;
            }
}

} // namespace lm
