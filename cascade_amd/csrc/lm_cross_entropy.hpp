// Softmax cross entropy of logits that are never kept: loss[n] = ln sum_v exp(h_n . w_v) - h_n . w_target[n].
//
// Forward: tiles of the product W H^T (vocabulary down, tokens across) end in the largest logit and the sum of exponentials
// of every token over the 128 (or 64) words of a wave, 8 bytes where the logits would have been 512; a second kernel joins
// them. Vocabulary runs along a lane's registers, so that a token's maximum and sum are taken without leaving the lane but once.
// Backward: the vocabulary in pieces, each piece's logits computed again and turned into
//   P[n][v] = d_loss[n] (exp(logit - lse[n]) - (v == target[n])),
// rounded to 16 bits as the operand of the two products that follow, d_weight = P^T H and d_hidden = P W. The rounding is the
// matrix unit's price, of the size of the gradients' own last rounding. P of a piece is all that is kept.
// P is held relative to the largest |d_loss|, and the products are scaled back in 32 bits. The entries that weigh most are those of the targets, nearly
// -d_loss[n] each, and a mean over tokens gives all tokens one d_loss: rounded as it is, its error (up to 2^-9) would be the same in all of
// them and stay in every sum; relative to itself it is 1, which rounds to itself. In half precision that 1 is 2^14, since probabilities of 1e-9 would
// otherwise vanish.
//
// Measured on 8192 tokens of 4096 values and 50257 words (bfloat16): forward 2.7 ms, 1250 TFLOP/s; backward 8.2 ms for three products of that size, 1230.
// Bound by the product (lm_product.hpp); the gradients' stores as whole lines took 0.7 ms off. 61 tokens of 512 values, forward: 11.6 us for 51 MB of weights, 4.4 TB/s.
#pragma once
#include "lm_product.hpp"

namespace lm {

// Workgroup id % 8 tells the XCD that it runs on: the order in which each of these has a run of its own.
__device__ inline uint32_t by_xcd(uint32_t id, uint32_t total)
{
    const uint32_t xcd = id % 8, per = total / 8, more = total % 8;
    return xcd * per + (xcd < more ? xcd : more) + id / 8;
}

// The order of tiles: bands of 8 row tiles that are walked column by column, so that the 32 workgroups of an XCD that run together share operands in its L2 (bands of 4 take the
// same time, of 16 5 % more, of 32 13 % more).
__device__ inline void in_bands(uint32_t id, uint32_t mt, uint32_t nt, uint32_t& m, uint32_t& n)
{
    constexpr uint32_t BAND = 8;
    const uint32_t band = id / (BAND * nt), first = band * BAND, high = mt - first < BAND ? mt - first : BAND, in = id - first * nt;
    m = first + in % high;
    n = in / high;
}

__device__ inline void tile_of(uint32_t id, uint32_t mt, uint32_t nt, uint32_t& m, uint32_t& n) { in_bands(by_xcd(id, mt * nt), mt, nt, m, n); }

struct Logits {
    Operand weight, hidden; // vocabulary rows of this piece, tokens
    int64_t dim;
    uint32_t mt, nt;
    const int32_t* target;
    int64_t first_word; // of this piece in the vocabulary
};

#define LM_TILE_BUFFERS(P) \
    __shared__ __attribute__((aligned(16))) short a0[P::BM * SLICE], a1[P::BM * SLICE], b0[P::BN * SLICE], b1[P::BN * SLICE]

template <class P>
__global__ __launch_bounds__(P::THREADS) void logit_sums_kernel(Logits l, float2* part, float* target_logit)
{
    LM_TILE_BUFFERS(P);
    uint32_t mi, ni;
    tile_of(blockIdx.x, l.mt, l.nt, mi, ni);
    typename P::Sums sums;
    const int64_t m0 = static_cast<int64_t>(mi) * P::BM, n0 = static_cast<int64_t>(ni) * P::BN;
    P::run(l.weight, l.hidden, m0, n0, 0, l.dim, a0, a1, b0, b1, sums);
    const int lane = threadIdx.x % 64, half = lane / 32;
    const int64_t tokens = l.hidden.rows, mw = m0 + P::wave_m();
    const int64_t rows = l.weight.rows - mw;
    const int left = static_cast<int>(rows < P::BM / P::WM ? rows : P::BM / P::WM) - 4 * half; // this lane's words there are: row < left
#pragma unroll
    for (int j = 0; j < P::TN; ++j) {
        const int64_t n = n0 + P::wave_n() + 32 * j + lane % 32;
        const bool there = n < tokens;
        const int64_t t = (there ? l.target[n] : -1) - (l.first_word + mw) - 4 * half;
        const int word = t >= 0 && t < left ? static_cast<int>(t) : -1;
        float top = -3.0e38f, picked = 0.f;
#pragma unroll
        for (int i = 0; i < P::TM; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int row = 32 * i + 8 * (r / 4) + r % 4;
                picked = word == row ? sums[i][j][r] : picked;
                if (row >= left) // words past the end
                    sums[i][j][r] = -INFINITY;
                top = fmaxf(top, sums[i][j][r]);
            }
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < P::TM; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                sum += __builtin_amdgcn_exp2f((sums[i][j][r] - top) * LOG2E);
        if (word >= 0 && !(word & 4)) // row % 8 < 4 always: a word whose rest is 4 or more is the other half's
            target_logit[n] = picked;
        const float top2 = other_half(top), sum2 = other_half(sum), high = fmaxf(top, top2);
        sum = sum * __builtin_amdgcn_exp2f((top - high) * LOG2E) + sum2 * __builtin_amdgcn_exp2f((top2 - high) * LOG2E);
        if (there && half == 0)
            part[(static_cast<int64_t>(mi) * P::WM + P::wave_m() / (P::BM / P::WM)) * tokens + n] = make_float2(high, sum);
    }
}

// (maximum, sum of exponentials over it)
__device__ inline void add_exponentials(float2& sum, float2 v)
{
    const float high = fmaxf(sum.x, v.x);
    sum.y = sum.y * __builtin_amdgcn_exp2f((sum.x - high) * LOG2E) + v.y * __builtin_amdgcn_exp2f((v.x - high) * LOG2E);
    sum.x = high;
}

// lse and loss from the waves' maxima and sums: TOKENS tokens by 256 / TOKENS runs of them a workgroup.
template <int TOKENS>
__global__ __launch_bounds__(256) void join_sums_kernel(const float2* part, int64_t parts, const float* target_logit, const int32_t* target,
                                                        int64_t tokens, int64_t vocab, float* loss, float* lse)
{
    constexpr int RUNS = 256 / TOKENS;
    __shared__ float2 got[RUNS][TOKENS + 1];
    const int x = threadIdx.x % TOKENS, y = threadIdx.x / TOKENS;
    const int64_t n = static_cast<int64_t>(blockIdx.x) * TOKENS + x;
    const float2 none = make_float2(-3.0e38f, 0.f);
    float2 sum = none;
    if (n < tokens)
        for (int64_t p = y; p < parts; p += 8 * RUNS) {
            float2 v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k)
                v[k] = p + k * RUNS < parts ? part[(p + k * RUNS) * tokens + n] : none;
#pragma unroll
            for (int k = 0; k < 8; ++k)
                add_exponentials(sum, v[k]);
        }
    got[y][x] = sum;
    for (int far = RUNS / 2; far; far /= 2) {
        __syncthreads();
        if (y < far) {
            add_exponentials(sum, got[y + far][x]);
            got[y][x] = sum;
        }
    }
    if (y == 0 && n < tokens) {
        const float all = sum.x + logf(sum.y);
        const int32_t t = target[n];
        lse[n] = all;
        loss[n] = t >= 0 && t < vocab ? all - target_logit[n] : 0.f;
    }
}

template <class P, class Type>
__global__ __launch_bounds__(P::THREADS) void logit_gradients_kernel(Logits l, const float* lse, const float* d_loss, const float* scale, int64_t vocab,
                                                                     short* out, int64_t stride)
{
    LM_TILE_BUFFERS(P);
    uint32_t mi, ni;
    tile_of(blockIdx.x, l.mt, l.nt, mi, ni);
    typename P::Sums sums;
    const int64_t m0 = static_cast<int64_t>(mi) * P::BM, n0 = static_cast<int64_t>(ni) * P::BN;
    P::run(l.weight, l.hidden, m0, n0, 0, l.dim, a0, a1, b0, b1, sums);
    const int lane = threadIdx.x % 64;
    const int64_t tokens = l.hidden.rows, mw = m0 + P::wave_m();
    float factor[P::TN], shift[P::TN];
    int word[P::TN]; // the target's row of the wave's part, if it is one
#pragma unroll
    for (int j = 0; j < P::TN; ++j) {
        const int64_t n = n0 + P::wave_n() + 32 * j + lane % 32, goal = n < tokens ? l.target[n] : -1;
        const bool counts = goal >= 0 && goal < vocab;
        factor[j] = counts ? d_loss[n] * scale[0] : 0.f;
        shift[j] = counts ? lse[n] : INFINITY; // tokens left out: zeros, whatever their logits are
        const int64_t t = goal - (l.first_word + mw);
        word[j] = counts && t >= 0 && t < P::BM ? static_cast<int>(t) : -1;
    }
    meet(); // everybody has read the last slice
    P::template store_turned<Type>(
        sums, P::wave_region(a0, a1, b0, b1), m0, n0, l.weight.rows, tokens, out, stride, true,
        [&](int j, int row, float x) {
            const float p = __builtin_amdgcn_exp2f((x - shift[j]) * LOG2E) - (word[j] == row ? 1.f : 0.f);
            return shift[j] == INFINITY ? 0.f : p * factor[j];
        });
    // k of the products to come runs along these rows, to a multiple of 8
    const int64_t tail = l.weight.rows + threadIdx.x % 8;
    if (mi == l.mt - 1 && tail < stride)
        for (int64_t n = n0 + threadIdx.x / 8; n < n0 + P::BN && n < tokens; n += P::THREADS / 8)
            out[n * stride + tail] = 0;
}

// d_weight rows of a piece, turned: sum over tokens of h[n] P[n][v].
template <class P, class Type>
__global__ __launch_bounds__(P::THREADS) void weight_gradients_kernel(Operand hidden, Operand p, int64_t tokens, uint32_t mt, uint32_t nt, const float* scale,
                                                                      short* out, int64_t stride, bool wide)
{
    LM_TILE_BUFFERS(P);
    uint32_t mi, ni;
    tile_of(blockIdx.x, mt, nt, mi, ni);
    typename P::Sums sums;
    const int64_t m0 = static_cast<int64_t>(mi) * P::BM, n0 = static_cast<int64_t>(ni) * P::BN;
    P::run(hidden, p, m0, n0, 0, tokens, a0, a1, b0, b1, sums);
    const float back = scale[1];
    meet();
    P::template store_turned<Type>(sums, P::wave_region(a0, a1, b0, b1), m0, n0, hidden.rows, p.rows, out, stride, wide,
                                   [&](int, int, float x) { return x * back; });
}

// One share of d_hidden: the sum over words [k, k + share) of P[n][v] w[v], in 32 bits, added to what earlier pieces left.
template <class P>
__global__ __launch_bounds__(P::THREADS) void hidden_gradients_kernel(Operand p, Operand weight, int64_t words, int64_t share, uint32_t mt, uint32_t nt,
                                                                      float* out, int64_t stride, bool add)
{
    LM_TILE_BUFFERS(P);
    // an XCD's workgroups are of one share or of neighbouring ones (100 tokens of 512 values trained 109 -> 102 us, 1000 of 1024 525 -> 512, 2000 of 1024 916 -> 919)
    const uint32_t id = by_xcd(blockIdx.x, gridDim.x), which = id / (mt * nt);
    uint32_t mi, ni;
    in_bands(id % (mt * nt), mt, nt, mi, ni);
    typename P::Sums sums;
    const int64_t m0 = static_cast<int64_t>(mi) * P::BM, n0 = static_cast<int64_t>(ni) * P::BN;
    const int64_t k = which * share, end = k + share < words ? k + share : words;
    P::run(p, weight, m0, n0, k, end, a0, a1, b0, b1, sums);
    const int lane = threadIdx.x % 64, half = lane / 32;
    const int64_t mw = m0 + P::wave_m(), rows = p.rows - mw;
    const int left = static_cast<int>(rows < P::BM / P::WM ? rows : P::BM / P::WM) - 4 * half;
#pragma unroll
    for (int j = 0; j < P::TN; ++j) {
        const int64_t n = n0 + P::wave_n() + 32 * j + lane % 32;
        float* to = out + (which * p.rows + mw + 4 * half) * stride + n;
        if (n < weight.rows)
#pragma unroll
            for (int i = 0; i < P::TM; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int row = 32 * i + 8 * (r / 4) + r % 4;
                    if (row < left) {
                        float* at = to + static_cast<int64_t>(row) * stride;
                        *at = add ? *at + sums[i][j][r] : sums[i][j][r];
                    }
                }
    }
}

// d_hidden from its shares: LANES lanes for four values, each with every LANES-th share.
template <class Type, int LANES>
__global__ __launch_bounds__(256) void join_shares_kernel(const float* shares, uint32_t count, int64_t tokens, int64_t dim, int64_t stride, const float* scale,
                                                          short* out, int64_t out_stride)
{
    constexpr int HERE = 256 / LANES; // fours of values a workgroup: neighbouring lanes hold neighbouring ones
    __shared__ f32x4 got[LANES][HERE];
    const int x = threadIdx.x % HERE, y = threadIdx.x / HERE;
    const int64_t at = static_cast<int64_t>(blockIdx.x) * HERE + x, quads = stride / 4;
    const bool there = at < tokens * quads;
    const int64_t n = there ? at / quads : 0, d = there ? at % quads * 4 : 0;
    f32x4 sum = {};
    if (there)
#pragma unroll 4
        for (uint32_t c = y; c < count; c += LANES)
            sum += *reinterpret_cast<const f32x4*>(shares + (c * tokens + n) * stride + d);
    if (LANES > 1) {
        got[y][x] = sum;
        __syncthreads();
        if (y == 0)
            for (int k = 1; k < LANES; ++k)
                sum += got[k][x];
    }
    if (!there || y)
        return;
    const float back = scale[1];
    for (int i = 0; i < 4; ++i)
        if (d + i < dim)
            out[n * out_stride + d + i] = to16<Type>(sum[i] * back);
}

// A row's piece of eight in a layout that 16-byte loads can walk: padded to 8 values with zeros; with targets, rows without one are zeros (their
// values may be anything, and 0 times infinity is no 0).
__device__ inline void lay_out_piece(int64_t at, const short* in, int64_t in_stride, int64_t rows, int64_t dim, const int32_t* target, int64_t vocab, short* out, int64_t stride,
                                     bool whole)
{
    const int64_t pieces = stride / 8;
    if (at >= rows * pieces)
        return;
    const int64_t row = at / pieces, d = at % pieces * 8;
    const bool keep = !target || (target[row] >= 0 && target[row] < vocab);
    s16x8 v = {};
    if (keep && whole) {
        v = *reinterpret_cast<const s16x8*>(in + row * in_stride + d);
    } else if (keep) {
        for (int i = 0; i < 8; ++i)
            v[i] = d + i < dim ? in[row * in_stride + d + i] : static_cast<short>(0);
    }
    *reinterpret_cast<s16x8*>(out + row * stride + d) = v;
}

__global__ __launch_bounds__(256) void lay_out_rows_kernel(const short* in, int64_t in_stride, int64_t rows, int64_t dim, short* out, int64_t stride, bool whole)
{
    lay_out_piece(static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, in, in_stride, rows, dim, nullptr, 0, out, stride, whole);
}

// The factor of P, range / max |d_loss|, and what the products of P are scaled back with: its inverse times `rate`, the logits' own. What is not finite among them has no say: its token is lost whatever the factor is, and takes nothing from the others.
struct LossScale {
    const float* d_loss;
    float range, rate;
    float* scale; // two
};

// What the gradients begin with: the first workgroup finds the factor, the others lay out the rows of hidden.
__global__ __launch_bounds__(1024) void scale_and_lay_out_kernel(LossScale l, const short* in, int64_t in_stride, int64_t rows, int64_t dim, const int32_t* target, int64_t vocab,
                                                                short* out, int64_t stride, bool whole)
{
    if (blockIdx.x) {
        lay_out_piece(static_cast<int64_t>(blockIdx.x - 1) * 1024 + threadIdx.x, in, in_stride, rows, dim, target, vocab, out, stride, whole);
        return;
    }
    __shared__ float tops[16];
    float top = 0.f;
    for (int64_t n0 = threadIdx.x; n0 < rows; n0 += 8 * 1024) { // eight loads on their way at a time
        int32_t goal[8];
        float x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int64_t n = n0 + k * 1024 < rows ? n0 + k * 1024 : n0;
            goal[k] = target[n];
            x[k] = fabsf(l.d_loss[n]);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (goal[k] >= 0 && goal[k] < vocab && x[k] < INFINITY)
                top = fmaxf(top, x[k]);
    }
    for (int d = 32; d; d /= 2)
        top = fmaxf(top, __shfl_xor(top, d));
    if (threadIdx.x % 64 == 0)
        tops[threadIdx.x / 64] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 16; ++w)
            top = fmaxf(top, tops[w]);
        const bool fine = top > 1e-30f && top < 1e30f; // both factors are ordinary numbers
        l.scale[0] = fine ? l.range / top : 1.f;
        l.scale[1] = (fine ? top / l.range : 1.f) * l.rate;
    }
}

__global__ __launch_bounds__(256) void zero_rows_kernel(short* out, int64_t stride, int64_t rows, int64_t dim)
{
    for (int i = 0; i < 4; ++i) {
        const int64_t at = static_cast<int64_t>(blockIdx.x) * 1024 + i * 256 + threadIdx.x;
        if (at < rows * dim)
            out[at / dim * stride + at % dim] = 0;
    }
}

} // namespace lm
