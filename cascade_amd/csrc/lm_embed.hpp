// The rows of a weight for the tokens of a text, out[i] = scale * weight[token[i]], and the gradient of the weight,
//   d_weight[v] = scale * (sum over the places i of word v, in their order, of d_out[i]).
//
// Forward: bound by memory, a row read and a row written a token.
// Backward: places are put in the order of their words first, so that a row of d_weight is the sum of neighbouring entries, without atomics and in a fixed
// order. A short text is ranked in one launch: place i goes to where it has as many entries before it as there are pairs (token, place) below its own, all pairs
// compared. A longer one takes a stable sort by digits of up to 9 bits, three launches each: every wave counts the digits of a segment of its own, the counts of a digit are
// summed over the segments, and the wave moves its segment, with ballots that tell a lane how many lanes before it hold its digit.
// The order is cut into runs of RUN entries, whatever words they hold, so that frequent words are shared out: a team of lanes adds up a run's rows in 32 bits and stores
// the words that lie inside it; of a word that reaches over the run's ends it leaves a partial sum, which a second kernel joins in the order of the runs.
// Rows of words that are not there are zeros, which the workgroups behind the teams' write.
#pragma once
#include "lm_values.hpp"

namespace lm {

constexpr int PIECES_PER_GROUP = 1024;

template <class Token>
__device__ inline uint32_t word_of(const Token* tokens, int64_t i, uint32_t rows) // `rows` for what is no row
{
    const uint32_t t = static_cast<uint32_t>(tokens[i]);
    return t < rows ? t : rows;
}

template <class T, class Token>
__global__ __launch_bounds__(256) void embed_kernel(const Token* tokens, int64_t n, const T* weight, int64_t stride, uint32_t rows, int dim, float scale, T* out)
{
    constexpr int TURNS = PIECES_PER_GROUP / 256;
    const uint32_t pieces = (dim + PIECE - 1) / PIECE;
    const uint64_t first = static_cast<uint64_t>(blockIdx.x) * PIECES_PER_GROUP;
    const int64_t base = first / pieces; // this workgroup's first row, and the first of its pieces there
    const uint32_t rest = static_cast<uint32_t>(first % pieces);
    int64_t row[TURNS];
    int d[TURNS];
    uint32_t word[TURNS];
    float x[TURNS][PIECE];
#pragma unroll
    for (int j = 0; j < TURNS; ++j) {
        const uint32_t at = rest + j * 256 + threadIdx.x;
        row[j] = base + at / pieces;
        d[j] = piece_at(at % pieces * PIECE, dim).d;
        word[j] = row[j] < n ? word_of(tokens, row[j], rows) : rows;
    }
#pragma unroll
    for (int j = 0; j < TURNS; ++j)
        load8(weight + (word[j] < rows ? word[j] : 0) * stride + d[j], x[j]); // what is no row: the first one, not used
#pragma unroll
    for (int j = 0; j < TURNS; ++j) {
#pragma unroll
        for (int k = 0; k < PIECE; ++k)
            x[j][k] = word[j] < rows ? x[j][k] * scale : 0.f;
        if (row[j] < n)
            store8(out + row[j] * dim + d[j], x[j]);
    }
}

// ---- places in the order of their words ----

// 64 places a workgroup; its 16 waves share the places to compare them with.
template <class Token>
__global__ __launch_bounds__(1024) void rank_places_kernel(const Token* tokens, int n, uint32_t rows, uint32_t* words, uint32_t* places)
{
    __shared__ uint32_t counts[16][64];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, begin = blockIdx.x * 64, i = begin + lane;
    const uint32_t mine = i < n ? word_of(tokens, i, rows) : 0;
    const int share = (n + 1023) / 1024 * 64, from = wave * share, to = from + share < n ? from + share : n;
    uint32_t count = 0;
    for (int j0 = from; j0 < to; j0 += 64) {
        const uint32_t word = j0 + lane < n ? word_of(tokens, j0 + lane, rows) : 0xffffffffu; // past the end: below nothing
        if (j0 == begin) {
#pragma unroll
            for (int k = 0; k < 64; ++k) {
                const uint32_t other = __builtin_amdgcn_readlane(word, k);
                count += other < mine + (k < lane ? 1 : 0);
            }
        } else {
            const uint32_t limit = mine + (j0 < begin ? 1 : 0); // places before this one count with an equal word, too
#pragma unroll
            for (int k = 0; k < 64; ++k)
                count += static_cast<uint32_t>(__builtin_amdgcn_readlane(word, k)) < limit;
        }
    }
    counts[wave][lane] = count;
    __syncthreads();
    if (wave == 0 && i < n) {
        for (int w = 1; w < 16; ++w)
            count += counts[w][lane];
        words[count] = mine;
        places[count] = i;
    }
}

constexpr int DIGIT_BITS = 9, MOST_DIGITS = 1 << DIGIT_BITS;
constexpr uint64_t MOST_SEGMENTS = 4096;

// What a pass sorts: the text itself, or what the pass before left.
template <class Token>
struct Entries {
    const Token* tokens; // null behind the first pass
    const uint32_t *words, *places;
    int64_t n;
    uint32_t rows;
    __device__ uint32_t word(int64_t i) const { return tokens ? word_of(tokens, i, rows) : words[i]; }
    __device__ uint32_t place(int64_t i) const { return tokens ? static_cast<uint32_t>(i) : places[i]; }
};

// counts[digit][segment]; a wave a segment
template <class Token>
__global__ __launch_bounds__(256) void count_digits_kernel(Entries<Token> e, int64_t segment, uint32_t segments, int shift, uint32_t digits, uint32_t* counts)
{
    __shared__ uint32_t all[4][MOST_DIGITS];
    const uint32_t lane = threadIdx.x % 64, s = blockIdx.x * 4 + threadIdx.x / 64;
    uint32_t* mine = all[threadIdx.x / 64]; // a wave's own: no barriers
    for (uint32_t d = lane; d < digits; d += 64)
        mine[d] = 0;
    if (s >= segments)
        return;
    const int64_t begin = s * segment, end = begin + segment < e.n ? begin + segment : e.n;
    for (int64_t i = begin + lane; i < end; i += 64)
        atomicAdd(mine + (e.word(i) >> shift & (digits - 1)), 1u);
    for (uint32_t d = lane; d < digits; d += 64)
        counts[d * static_cast<uint64_t>(segments) + s] = mine[d];
}

// A digit's counts become the entries of that digit in earlier segments; totals[digit]: in all.
__global__ __launch_bounds__(256) void sum_digits_kernel(uint32_t* counts, uint32_t segments, uint32_t* totals)
{
    __shared__ uint32_t waves[2][4];
    uint32_t* mine = counts + blockIdx.x * static_cast<uint64_t>(segments);
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    uint32_t before = 0;
    int turn = 0;
    for (uint32_t s0 = 0; s0 < segments; s0 += 256, turn ^= 1) {
        const uint32_t s = s0 + threadIdx.x, x = s < segments ? mine[s] : 0;
        uint32_t sum = x;
        for (uint32_t d = 1; d < 64; d *= 2) {
            const uint32_t y = __shfl_up(sum, d);
            sum += lane >= d ? y : 0;
        }
        if (lane == 63)
            waves[turn][wave] = sum;
        __syncthreads();
        uint32_t earlier = before;
        for (uint32_t w = 0; w < 4; ++w) {
            earlier += w < wave ? waves[turn][w] : 0;
            before += waves[turn][w];
        }
        if (s < segments)
            mine[s] = earlier + sum - x;
    }
    if (threadIdx.x == 0)
        totals[blockIdx.x] = before;
}

template <class Token>
__global__ __launch_bounds__(256) void move_digits_kernel(Entries<Token> e, int64_t segment, uint32_t segments, int shift, uint32_t digits, const uint32_t* counts,
                                                          const uint32_t* totals, uint32_t* words, uint32_t* places)
{
    __shared__ uint32_t all[4][MOST_DIGITS];
    const uint32_t lane = threadIdx.x % 64, s = blockIdx.x * 4 + threadIdx.x / 64;
    uint32_t* next = all[threadIdx.x / 64]; // where the wave's next entry of a digit goes
    if (s >= segments)
        return;
    uint32_t before = 0; // entries of lower digits
    for (uint32_t d0 = 0; d0 < digits; d0 += 64) {
        const uint32_t d = d0 + lane, x = d < digits ? totals[d] : 0;
        uint32_t sum = x;
        for (uint32_t k = 1; k < 64; k *= 2) {
            const uint32_t y = __shfl_up(sum, k);
            sum += lane >= k ? y : 0;
        }
        if (d < digits)
            next[d] = before + sum - x + counts[d * static_cast<uint64_t>(segments) + s];
        before += __shfl(sum, 63);
    }
    const int64_t begin = s * segment, end = begin + segment < e.n ? begin + segment : e.n;
    for (int64_t i0 = begin; i0 < end; i0 += 64) {
        const int64_t i = i0 + lane;
        const bool there = i < end;
        const uint32_t word = there ? e.word(i) : 0, place = there ? e.place(i) : 0, digit = word >> shift & (digits - 1);
        uint64_t same = __ballot(there); // the lanes that hold this lane's digit
        for (uint32_t bit = 1; bit < digits; bit *= 2) {
            const uint64_t ones = __ballot(digit & bit);
            same &= digit & bit ? ones : ~ones;
        }
        const uint32_t rank = __popcll(same & ((1ull << lane) - 1));
        uint32_t to = 0;
        if (there)
            to = next[digit] + rank;
        __builtin_amdgcn_wave_barrier();
        if (there && rank == 0)
            next[digit] = to + __popcll(same);
        __builtin_amdgcn_wave_barrier();
        if (there) {
            words[to] = word;
            places[to] = place;
        }
    }
}

// ---- sums of neighbouring entries ----

struct EmbedSums {
    const uint32_t *words, *places; // n entries in order
    int64_t n, run, runs;           // entries of a run
    int64_t stride;                 // of d_out
    int64_t groups;                 // workgroups of teams; those behind them write zeros
    uint32_t rows, rows_each;       // of d_weight; rows that a workgroup of zeros looks after
    int dim, slices;                // slices of a row: a team's lanes take eight values each
    float scale;
    float *head, *tail;             // sums of a run's first word as far as it comes from the run before, and of its last one that begins in it and goes on
};

// The first entry whose word is not below `word`.
__device__ inline int64_t first_entry(const uint32_t* words, int64_t n, uint32_t word)
{
    int64_t lo = 0, hi = n;
    while (lo < hi) {
        const int64_t mid = (lo + hi) / 2;
        if (words[mid] < word)
            lo = mid + 1;
        else
            hi = mid;
    }
    return lo;
}

constexpr int ZERO_ROWS = 64; // that a workgroup looks after at most

template <class T, int LANES>
__global__ __launch_bounds__(256) void embed_sums_kernel(EmbedSums e, const T* d_out, T* d_weight)
{
    if (blockIdx.x >= e.groups) {
        __shared__ bool absent[ZERO_ROWS];
        const uint32_t v0 = static_cast<uint32_t>((blockIdx.x - e.groups) * e.rows_each), count = e.rows - v0 < e.rows_each ? e.rows - v0 : e.rows_each;
        if (threadIdx.x < count) {
            const int64_t at = first_entry(e.words, e.n, v0 + threadIdx.x);
            absent[threadIdx.x] = at == e.n || e.words[at] != v0 + threadIdx.x;
        }
        __syncthreads();
        const uint32_t pieces = (e.dim + PIECE - 1) / PIECE;
        const float zeros[PIECE] = {};
        for (uint32_t k = threadIdx.x; k < count * pieces; k += 256)
            if (const uint32_t v = k / pieces; absent[v])
                store8(d_weight + static_cast<int64_t>(v0 + v) * e.dim + piece_at(k % pieces * PIECE, e.dim).d, zeros);
        return;
    }
    const int64_t team = static_cast<int64_t>(blockIdx.x) * (256 / LANES) + threadIdx.x / LANES, run = team / e.slices;
    const Piece at = piece_at((static_cast<int>(team % e.slices) * LANES + threadIdx.x % LANES) * PIECE, e.dim);
    if (run >= e.runs || !at.mine)
        return;
    constexpr int AHEAD = 8;
    const int64_t begin = run * e.run, end = begin + e.run < e.n ? begin + e.run : e.n;
    uint32_t word = e.words[begin];
    bool continued = begin > 0 && e.words[begin - 1] == word; // from the run before
    float sum[PIECE] = {};
    auto close = [&](bool goes_on) { // the sum of `word` is complete as far as this run goes
        if (word >= e.rows)
            return;
        if (continued || goes_on) {
            store8((continued ? e.head : e.tail) + run * e.dim + at.d, sum);
        } else {
#pragma unroll
            for (int k = 0; k < PIECE; ++k)
                sum[k] *= e.scale;
            store8(d_weight + static_cast<int64_t>(word) * e.dim + at.d, sum);
        }
    };
    for (int64_t s = begin; s < end; s += AHEAD) {
        uint32_t words[AHEAD];
        float x[AHEAD][PIECE];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const int64_t entry = s + k < end ? s + k : end - 1; // past the end: the last one again, not used
            words[k] = e.words[entry];
            load8(d_out + e.places[entry] * e.stride + at.d, x[k]);
        }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            if (s + k >= end)
                break;
            if (words[k] != word) {
                close(false);
                word = words[k];
                continued = false;
#pragma unroll
                for (int i = 0; i < PIECE; ++i)
                    sum[i] = 0;
            }
#pragma unroll
            for (int i = 0; i < PIECE; ++i)
                sum[i] += x[k][i];
        }
    }
    close(end < e.n && e.words[end] == word);
}

// A word that goes on behind the run it begins in: the tail of that run and the heads of the next ones. A workgroup a run and slice, its teams share the heads.
template <class T, int LANES>
__global__ __launch_bounds__(256) void embed_join_kernel(EmbedSums e, T* d_weight)
{
    constexpr int TEAMS = 256 / LANES;
    __shared__ float got[TEAMS][PIECE][LANES];
    const int64_t run = blockIdx.x / e.slices, last = (run + 1) * e.run - 1; // never the last run
    const uint32_t word = e.words[last];
    if (word >= e.rows || e.words[last + 1] != word || (e.words[run * e.run] == word && run > 0 && e.words[run * e.run - 1] == word))
        return;
    int64_t lo = run + 1, hi = e.runs - 1; // the last run that begins with the word
    while (lo < hi) {
        const int64_t mid = (lo + hi + 1) / 2;
        if (e.words[mid * e.run] == word)
            lo = mid;
        else
            hi = mid - 1;
    }
    const int x = threadIdx.x % LANES, y = threadIdx.x / LANES;
    const Piece at = piece_at((static_cast<int>(blockIdx.x % e.slices) * LANES + x) * PIECE, e.dim);
    float sum[PIECE] = {};
    if (y == 0)
        load8(e.tail + run * e.dim + at.d, sum);
#pragma unroll 4
    for (int64_t r = run + 1 + y; r <= lo; r += TEAMS) {
        float more[PIECE];
        load8(e.head + r * e.dim + at.d, more);
#pragma unroll
        for (int k = 0; k < PIECE; ++k)
            sum[k] += more[k];
    }
#pragma unroll
    for (int k = 0; k < PIECE; ++k)
        got[y][k][x] = sum[k];
    __syncthreads();
    if (y || !at.mine)
        return;
    for (int t = 1; t < TEAMS; ++t)
#pragma unroll
        for (int k = 0; k < PIECE; ++k)
            sum[k] += got[t][k][x];
#pragma unroll
    for (int k = 0; k < PIECE; ++k)
        sum[k] *= e.scale;
    store8(d_weight + static_cast<int64_t>(word) * e.dim + at.d, sum);
}

} // namespace lm
