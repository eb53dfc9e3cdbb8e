// Distillation from the logits that a teacher kept of every token: with z = hidden weight^T / T over the vocabulary and q the teacher's softmax
// over its own logits / T, wherever it has some,
//   loss = sum over the kept words of q (ln q - z) + ln sum exp z,   d_z = d_loss / T (softmax(z) - q).
//
// The cross entropy's path (lm_cross_entropy.hpp) with many targets a token instead of one: the same tile products, without logits that are kept. A first kernel makes q,
// sorts every token's words and notes where each block of words (those that a wave's part of a tile holds) begins among them. A
// tile that is done lays its logits, or their exponentials, into LDS in 32 bits, a line of words for each token, and the token's lanes pick theirs there, or take q off
// before anything is rounded: p - q, which a student that has learnt leaves small, keeps all its bits.
#pragma once
#include "lm_cross_entropy.hpp"

namespace lm {

constexpr uint32_t MOST_KEPT = 1024; // logits of a token

// Entries of a token in the order of their words; those of block b stand at first[b] to first[b + 1].
struct Teacher {
    const int32_t* ids;    // tokens x kept
    const float* q;        // tokens x kept
    const uint16_t* first; // tokens x (blocks + 1)
    int64_t kept, blocks;
};

// A wave a token. words_each: of a block.
template <int ITEMS>
__global__ __launch_bounds__(256) void teacher_kernel(const int32_t* ids, const float* logits, int64_t tokens, int kept, int64_t vocab, float rate, int words_each, int64_t blocks,
                                                      int32_t* sorted_ids, float* sorted_q, uint16_t* first, int32_t* counts, float* entropy)
{
    __shared__ uint32_t all_words[4][ITEMS * 64];
    __shared__ float all_q[4][ITEMS * 64];
    const int lane = threadIdx.x % 64;
    const int64_t n = static_cast<int64_t>(blockIdx.x) * 4 + threadIdx.x / 64;
    if (n >= tokens)
        return;
    uint32_t* words = all_words[threadIdx.x / 64]; // a wave's own: no barriers
    float* qs = all_q[threadIdx.x / 64];
    uint32_t word[ITEMS], rank[ITEMS];
    float told[ITEMS], top = -INFINITY;
    int there = 0;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const int k = i * 64 + lane;
        const int32_t id = k < kept ? ids[n * kept + k] : -1;
        told[i] = id >= 0 && id < vocab ? logits[n * kept + k] * rate : -INFINITY;
        word[i] = told[i] == -INFINITY ? 0xffffffffu : static_cast<uint32_t>(id); // nothing is told: no entry
        there += word[i] != 0xffffffffu;
        top = fmaxf(top, told[i]);
        rank[i] = 0;
        words[k] = word[i];
    }
    for (int d = 32; d; d /= 2) {
        top = fmaxf(top, __shfl_xor(top, d));
        there += __shfl_xor(there, d);
    }
    float sum = 0, part = 0;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        told[i] -= top;
        sum += word[i] != 0xffffffffu ? expf(told[i]) : 0.f;
    }
    sum = wave_sum(sum);
    const float all = logf(sum);
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const float q = expf(told[i]) / sum;
        part += word[i] != 0xffffffffu ? q * (told[i] - all) : 0.f;
        told[i] = q;
    }
    part = wave_sum(part);
    if (lane == 0) {
        counts[n] = there ? 0 : -1;
        entropy[n] = part;
    }
    __builtin_amdgcn_wave_barrier();
    for (int j = 0; j < kept; ++j) { // entries of one word stay in their order
        const uint32_t other = words[j];
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
            rank[i] += other < word[i] || (other == word[i] && j < i * 64 + lane);
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
        if (i * 64 + lane < kept) {
            words[rank[i]] = word[i];
            qs[rank[i]] = told[i];
        }
    __builtin_amdgcn_wave_barrier();
    for (int k = lane; k < there; k += 64) {
        sorted_ids[n * kept + k] = static_cast<int32_t>(words[k]);
        sorted_q[n * kept + k] = qs[k];
    }
    for (int64_t b = lane; b <= blocks; b += 64) {
        int lo = 0, hi = there; // the first entry whose word is of block b or behind it
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (words[mid] < b * words_each)
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

// P[n][v] = d_loss[n] (exp(z - lse[n]) - q) relative to the largest |d_loss|, as logit_gradients_kernel leaves it; 1 / T is in what the products are scaled back with.
template <class P, class Type>
__global__ __launch_bounds__(P::THREADS) void distill_gradients_kernel(Logits l, Teacher teacher, float rate, const float* lse, const float* d_loss, const float* scale,
                                                                       short* out, int64_t stride)
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
#pragma unroll
        for (int c = 0; c < 32; c += 64 / EIGHTS) {
            const int token = c + lane / EIGHTS;
            const f32x4 low = *reinterpret_cast<const f32x4*>(Words::piece(lines, token, 2 * eight)), high = *reinterpret_cast<const f32x4*>(Words::piece(lines, token, 2 * eight + 1));
            s16x8 y;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                y[r] = to16<Type>(low[r]);
                y[4 + r] = to16<Type>(high[r]);
            }
            if (first + token >= tokens || m >= l.weight.rows)
                continue;
            short* to = out + (first + token) * stride + m;
            if (m + 8 <= l.weight.rows) {
                *reinterpret_cast<s16x8*>(to) = y;
            } else {
                for (int r = 0; r < 8; ++r)
                    if (m + r < l.weight.rows)
                        to[r] = y[r];
            }
        }
        wait_for_lds();
    }
    // k of the products to come runs along these rows, to a multiple of 8
    const int64_t tail = l.weight.rows + threadIdx.x % 8;
    if (mi == l.mt - 1 && tail < stride)
        for (int64_t n = n0 + threadIdx.x / 8; n < n0 + P::BN && n < tokens; n += P::THREADS / 8)
            out[n * stride + tail] = 0;
}

} // namespace lm
