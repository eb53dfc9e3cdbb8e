// The rows of a weight for the tokens of a text, out[i] = scale * weight[token[i]], and the gradient of the weight,
//   d_weight[v] = scale * (sum over the places i of word v, in their order, of d_out[i]).
//
// Forward: bound by memory, a row read and a row written a token.
// Backward: places are put in the order of their words first, so that a row of d_weight is the sum of neighbouring entries, without atomics and in a fixed
// order. A short text is ranked in one launch: place i goes to where it has as many entries before it as there are pairs (word, place) below its own, all pairs
// compared. A longer one takes a stable sort by digits of up to 9 bits, two launches each, or three where there are many segments: workgroups count the digits of their segments, the counts of a digit
// are summed over the segments (few are by those who move them), and the workgroups move their segments, with ballots that tell a lane how many lanes before it hold its digit.
// The order is cut into runs of entries, whatever words they hold, so that frequent words are shared out: a team of lanes adds up a run's rows in 32 bits and stores
// the words that lie inside it. Of words that reach over a run's ends the teams of a workgroup join their sums in LDS, in the order of the runs, and what reaches over the ends of the
// workgroup's block of runs is left as a partial sum, which a second kernel joins in the order of the blocks.
// Rows of words that are not there are zeros. Where most words are not, all rows are written as zeros beside the kernel that begins the ordering, which leaves the memory idle; otherwise
// workgroups behind the teams' look for them.
#pragma once
#include "lm_values.hpp"

namespace lm {

template <class Token>
__device__ inline uint32_t word_of(const Token* tokens, int64_t i, uint32_t rows) // `rows` for what is no row
{
    const uint32_t t = static_cast<uint32_t>(tokens[i]);
    return t < rows ? t : rows;
}

// TURNS pieces a lane
template <class T, class Token, int TURNS, bool PAST>
__global__ __launch_bounds__(256) void embed_kernel(const Token* tokens, int64_t n, const T* weight, int64_t stride, uint32_t rows, int dim, float scale, T* out)
{
    constexpr int V = PIECE<T>;
    const uint32_t pieces = (dim + V - 1) / V;
    const uint64_t first = static_cast<uint64_t>(blockIdx.x) * (TURNS * 256);
    const int64_t base = first / pieces; // this workgroup's first row, and the first of its pieces there
    const uint32_t rest = static_cast<uint32_t>(first % pieces);
    int64_t row[TURNS];
    int d[TURNS];
    uint32_t word[TURNS];
    float x[TURNS][V];
#pragma unroll
    for (int j = 0; j < TURNS; ++j) {
        const uint32_t at = rest + j * 256 + threadIdx.x;
        row[j] = base + at / pieces;
        d[j] = piece_at<V>(at % pieces * V, dim).d;
        word[j] = row[j] < n ? word_of(tokens, row[j], rows) : rows;
    }
#pragma unroll
    for (int j = 0; j < TURNS; ++j)
        load(weight + (word[j] < rows ? word[j] : 0) * stride + d[j], x[j]); // what is no row: the first one, not used
#pragma unroll
    for (int j = 0; j < TURNS; ++j) {
#pragma unroll
        for (int k = 0; k < V; ++k)
            x[j][k] = word[j] < rows ? x[j][k] * scale : 0.f;
        if (row[j] < n)
            store<PAST>(out + row[j] * dim + d[j], x[j]);
    }
}

// ---- zeros ----

constexpr int64_t ZERO_BYTES = 65536; // that a workgroup writes

struct Zeros { // of `bytes` bytes, a multiple of two, by the workgroups behind the first `groups` of a launch
    char* to;
    int64_t bytes;
    uint32_t groups;
};

__device__ inline void write_zeros(const Zeros& z)
{
    const int64_t begin = static_cast<int64_t>(blockIdx.x - z.groups) * ZERO_BYTES, end = begin + ZERO_BYTES < z.bytes ? begin + ZERO_BYTES : z.bytes;
    const Several<uint16_t, 8> none = {};
    int64_t i = begin + threadIdx.x * 16;
    for (; i + 16 <= end; i += blockDim.x * 16)
        *reinterpret_cast<Several<uint16_t, 8>*>(z.to + i) = none;
    for (; i < end; i += 2)
        *reinterpret_cast<uint16_t*>(z.to + i) = 0;
}

// ---- places in the order of their words ----

constexpr int RANKED_EACH = 32; // places a workgroup

// RANKED_EACH places a workgroup, all compared with all REGISTERS * 1024 >= n places of the text, which lie in the registers of its 16 waves: a comparison and a count of its lanes for
// each place and 64 others. 8192 places: 10 us alone, 58 us with the zeros of 50257 rows of 4096 values (7.1 TB/s).
template <class Token, int REGISTERS>
__global__ __launch_bounds__(1024) void rank_places_kernel(const Token* tokens, int n, uint32_t rows, uint32_t* words, uint32_t* places, Zeros zeros)
{
    if (blockIdx.x >= zeros.groups) {
        write_zeros(zeros);
        return;
    }
    __shared__ int counts[16][RANKED_EACH];
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), begin = blockIdx.x * RANKED_EACH, own = begin / 64;
    int others[REGISTERS];
#pragma unroll
    for (int r = 0; r < REGISTERS; ++r) {
        const int block = wave * REGISTERS + r, j = block * 64 + lane;
        // what stands before this workgroup's block counts with an equal word, too; past the end nothing does
        others[r] = j < n ? static_cast<int>(word_of(tokens, j, rows)) - (block < own) : 0x7fffffff;
    }
    const int mine = begin + lane % RANKED_EACH < n ? static_cast<int>(word_of(tokens, begin + lane % RANKED_EACH, rows)) : 0;
    const int near = own * 64 + lane < n ? static_cast<int>(word_of(tokens, own * 64 + lane, rows)) : -1; // the block itself
    int found = 0;
    for (int p = 0; p < RANKED_EACH; ++p) {
        const int word = __builtin_amdgcn_readlane(mine, p);
        int below = 0;
#pragma unroll
        for (int r = 0; r < REGISTERS; ++r)
            below += __popcll(__ballot(others[r] < word));
        if (wave == own / REGISTERS)
            below += __popcll(__ballot(near == word) & ((1ull << (begin % 64 + p)) - 1));
        found = lane == p ? below : found;
    }
    if (lane < RANKED_EACH)
        counts[wave][lane] = found;
    __syncthreads();
    if (threadIdx.x < RANKED_EACH && begin + static_cast<int>(threadIdx.x) < n) {
        int rank = 0;
        for (int w = 0; w < 16; ++w)
            rank += counts[w][threadIdx.x];
        words[rank] = mine;
        places[rank] = begin + threadIdx.x;
    }
}

constexpr int DIGIT_BITS = 9, MOST_DIGITS = 1 << DIGIT_BITS;
constexpr int TURN_EACH = 4, TURN = 256 * TURN_EACH; // entries of a lane, and of a workgroup, at a time
constexpr uint64_t MOST_SEGMENTS = 4096;             // of whole turns

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

// counts[digit][segment]; a workgroup a segment
template <class Token>
__global__ __launch_bounds__(256) void count_digits_kernel(Entries<Token> e, int64_t segment, uint32_t segments, int shift, uint32_t digits, uint32_t* counts, Zeros zeros)
{
    if (blockIdx.x >= segments) {
        write_zeros(zeros);
        return;
    }
    __shared__ uint32_t all[MOST_DIGITS];
    for (uint32_t d = threadIdx.x; d < digits; d += 256)
        all[d] = 0;
    __syncthreads();
    const int64_t begin = blockIdx.x * segment, end = begin + segment < e.n ? begin + segment : e.n;
    for (int64_t i0 = begin; i0 < end; i0 += TURN) {
        uint32_t word[TURN_EACH];
#pragma unroll
        for (int k = 0; k < TURN_EACH; ++k) {
            const int64_t i = i0 + k * 256 + threadIdx.x;
            word[k] = e.word(i < end ? i : end - 1);
        }
#pragma unroll
        for (int k = 0; k < TURN_EACH; ++k)
            if (i0 + k * 256 + threadIdx.x < end)
                atomicAdd(all + (word[k] >> shift & (digits - 1)), 1u);
    }
    __syncthreads();
    for (uint32_t d = threadIdx.x; d < digits; d += 256)
        counts[d * static_cast<uint64_t>(segments) + blockIdx.x] = all[d];
}

// Sums of a wave's lanes up to each one.
__device__ inline uint32_t sums_to(uint32_t x)
{
    const uint32_t lane = threadIdx.x % 64;
    for (uint32_t d = 1; d < 64; d *= 2) {
        const uint32_t y = __shfl_up(x, d);
        x += lane >= d ? y : 0;
    }
    return x;
}

// A digit's counts become the entries of that digit in earlier segments; totals[digit]: in all.
__global__ __launch_bounds__(256) void sum_digits_kernel(uint32_t* counts, uint32_t segments, uint32_t* totals)
{
    __shared__ uint32_t waves[2][4];
    uint32_t* mine = counts + blockIdx.x * static_cast<uint64_t>(segments);
    const uint32_t wave = threadIdx.x / 64;
    uint32_t before = 0;
    int turn = 0;
    for (uint32_t s0 = 0; s0 < segments; s0 += 256, turn ^= 1) {
        const uint32_t s = s0 + threadIdx.x, x = s < segments ? mine[s] : 0, sum = sums_to(x);
        if (threadIdx.x % 64 == 63)
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

// A workgroup a segment, a turn at a time: each of its waves has a quarter of the turn, ranks its entries among those of their digit in that quarter and counts them, and
// begins behind the counts of the waves before it. SUMMED: counts and totals are sums over the segments; otherwise the workgroup adds up all counts itself.
template <class Token, bool SUMMED>
__global__ __launch_bounds__(256) void move_digits_kernel(Entries<Token> e, int64_t segment, uint32_t segments, int shift, uint32_t digits, const uint32_t* counts,
                                                          const uint32_t* totals, uint32_t* words, uint32_t* places)
{
    __shared__ uint32_t next[MOST_DIGITS];    // where the segment's next entry of a digit goes
    __shared__ uint32_t quarter[4][MOST_DIGITS]; // a wave's entries of a digit, then where they begin
    __shared__ uint32_t waves[4];
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int64_t begin = blockIdx.x * segment, end = begin + segment < e.n ? begin + segment : e.n;
    {
        constexpr int EACH = MOST_DIGITS / 256;
        uint32_t x[EACH], before[EACH], sum = 0;
#pragma unroll
        for (int k = 0; k < EACH; ++k) { // neighbouring digits a lane
            const uint32_t d = threadIdx.x * EACH + k;
            const uint32_t* mine = counts + d * static_cast<uint64_t>(segments);
            x[k] = before[k] = 0;
            if (SUMMED && d < digits) {
                x[k] = totals[d];
                before[k] = mine[blockIdx.x];
            } else if (d < digits) {
#pragma unroll 8
                for (uint32_t s = 0; s < segments; ++s) {
                    const uint32_t count = mine[s];
                    before[k] += s < blockIdx.x ? count : 0;
                    x[k] += count;
                }
            }
            sum += x[k];
        }
        uint32_t to = sums_to(sum);
        if (lane == 63)
            waves[wave] = to;
        __syncthreads();
        to -= sum;
        for (uint32_t w = 0; w < wave; ++w)
            to += waves[w];
#pragma unroll
        for (int k = 0; k < EACH; ++k) {
            next[threadIdx.x * EACH + k] = to + before[k];
            to += x[k];
        }
    }
    for (int64_t i0 = begin; i0 < end; i0 += TURN) {
        uint32_t word[TURN_EACH], place[TURN_EACH], rank[TURN_EACH];
#pragma unroll
        for (int k = 0; k < TURN_EACH; ++k) {
            const int64_t i = i0 + (wave * TURN_EACH + k) * 64 + lane, at = i < end ? i : end - 1;
            word[k] = e.word(at);
            place[k] = e.place(at);
        }
        for (uint32_t d = lane; d < digits; d += 64)
            quarter[wave][d] = 0;
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int k = 0; k < TURN_EACH; ++k) {
            const bool there = i0 + (wave * TURN_EACH + k) * 64 + lane < end;
            const uint32_t digit = word[k] >> shift & (digits - 1);
            uint64_t same = __ballot(there); // the lanes that hold this lane's digit
            for (uint32_t bit = 1; bit < digits; bit *= 2) {
                const uint64_t ones = __ballot(digit & bit);
                same &= digit & bit ? ones : ~ones;
            }
            const uint32_t before = there ? quarter[wave][digit] : 0, ahead = __popcll(same & ((1ull << lane) - 1));
            rank[k] = before + ahead;
            __builtin_amdgcn_wave_barrier();
            if (there && ahead == 0)
                quarter[wave][digit] = before + __popcll(same);
            __builtin_amdgcn_wave_barrier();
        }
        __syncthreads();
        for (uint32_t d = threadIdx.x; d < digits; d += 256) {
            uint32_t to = next[d];
            for (int w = 0; w < 4; ++w) {
                const uint32_t count = quarter[w][d];
                quarter[w][d] = to;
                to += count;
            }
            next[d] = to;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < TURN_EACH; ++k)
            if (i0 + (wave * TURN_EACH + k) * 64 + lane < end) {
                const uint32_t to = quarter[wave][word[k] >> shift & (digits - 1)] + rank[k];
                words[to] = word[k];
                places[to] = place[k];
            }
        __syncthreads();
    }
}

// ---- sums of neighbouring entries ----

struct EmbedSums {
    const uint32_t *words, *places; // n entries in order
    int64_t n, run, block, blocks;  // entries of a run, and of a block: a run for each team of a workgroup
    int64_t stride;                 // of d_out
    int64_t groups;                 // workgroups of teams, one a block and slice; those behind them write zeros
    uint32_t rows, rows_each;       // of d_weight; rows that a workgroup of zeros looks after
    int dim, slices;                // slices of a row: a team's lanes take a piece each
    float scale;
    float *head, *tail;             // sums of a block's first word as far as it comes from the block before, and of its last one that begins in it and goes on
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
    constexpr int V = PIECE<T>;
    if (blockIdx.x >= e.groups) {
        __shared__ bool absent[ZERO_ROWS];
        const uint32_t v0 = static_cast<uint32_t>((blockIdx.x - e.groups) * e.rows_each), count = e.rows - v0 < e.rows_each ? e.rows - v0 : e.rows_each;
        if (threadIdx.x < count) {
            const int64_t at = first_entry(e.words, e.n, v0 + threadIdx.x);
            absent[threadIdx.x] = at == e.n || e.words[at] != v0 + threadIdx.x;
        }
        __syncthreads();
        const uint32_t pieces = (e.dim + V - 1) / V;
        const float zeros[V] = {};
        for (uint32_t k = threadIdx.x; k < count * pieces; k += 256)
            if (const uint32_t v = k / pieces; absent[v])
                store(d_weight + static_cast<int64_t>(v0 + v) * e.dim + piece_at<V>(k % pieces * V, e.dim).d, zeros);
        return;
    }
    enum { HEAD = 1, THROUGH = 2, TAIL = 4 }; // the run's first word comes from the run before, and goes on behind this one; its last word begins in it and goes on
    constexpr int TEAMS = 256 / LANES, AHEAD = 8;
    __shared__ float heads[TEAMS][V][LANES];
    __shared__ int reach[TEAMS];
    const int64_t block = blockIdx.x / e.slices;
    const int team = threadIdx.x / LANES, x = threadIdx.x % LANES;
    const Piece at = piece_at<V>((static_cast<int>(blockIdx.x % e.slices) * LANES + x) * V, e.dim);
    const int64_t begin = block * e.block + team * e.run, end = begin + e.run < e.n ? begin + e.run : e.n;
    uint32_t word = e.rows;
    float sum[V] = {};
    int reaches = 0;
    if (begin < end) {
        word = e.words[begin];
        bool continued = begin > 0 && e.words[begin - 1] == word; // from the run before
        auto close = [&](bool goes_on) { // the sum of `word` is complete as far as this run goes
            if (word >= e.rows)
                return;
            if (continued) {
                reaches |= HEAD | (goes_on ? THROUGH : 0);
#pragma unroll
                for (int k = 0; k < V; ++k)
                    heads[team][k][x] = sum[k];
            } else if (goes_on) { // the last word: `sum` stays as it is, and goes on below
                reaches |= TAIL;
            } else if (at.mine) {
#pragma unroll
                for (int k = 0; k < V; ++k)
                    sum[k] *= e.scale;
                store(d_weight + static_cast<int64_t>(word) * e.dim + at.d, sum);
            }
        };
        for (int64_t s = begin; s < end; s += AHEAD) {
            uint32_t words[AHEAD];
            float more[AHEAD][V];
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) {
                const int64_t entry = s + k < end ? s + k : end - 1; // past the end: the last one again, not used
                words[k] = e.words[entry];
                load(d_out + e.places[entry] * e.stride + at.d, more[k]);
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
                    for (int i = 0; i < V; ++i)
                        sum[i] = 0;
                }
#pragma unroll
                for (int i = 0; i < V; ++i)
                    sum[i] += more[k][i];
            }
        }
        close(end < e.n && e.words[end] == word);
    }
    if (x == 0)
        reach[team] = reaches;
    __syncthreads();
    // `sum` goes on with the heads of the runs from `next` on; where that ends inside the block, it is stored at `inside`, otherwise at `over`
    auto go_on = [&](int next, float* over, auto inside) {
        for (; next < TEAMS; ++next) {
#pragma unroll
            for (int k = 0; k < V; ++k)
                sum[k] += heads[next][k][x];
            if (!(reach[next] & THROUGH)) {
                inside();
                return;
            }
        }
        if (at.mine)
            store(over + block * e.dim + at.d, sum);
    };
    if (reaches & TAIL)
        go_on(team + 1, e.tail, [&] {
#pragma unroll
            for (int k = 0; k < V; ++k)
                sum[k] *= e.scale;
            if (at.mine)
                store(d_weight + static_cast<int64_t>(word) * e.dim + at.d, sum);
        });
    if (team == 0 && reaches & HEAD) {
#pragma unroll
        for (int k = 0; k < V; ++k)
            sum[k] = 0;
        go_on(0, e.head, [&] {
            if (at.mine)
                store(e.head + block * e.dim + at.d, sum);
        });
    }
}

// The words that go on behind the block they begin in: the tail of that block and the heads of the next ones. A workgroup a block and slice, its teams share the heads.
template <class T, int LANES>
__global__ __launch_bounds__(256) void embed_join_kernel(EmbedSums e, T* d_weight)
{
    constexpr int TEAMS = 256 / LANES, V = PIECE<T>, AHEAD = 8;
    __shared__ float got[TEAMS][V][LANES];
    const int64_t block = blockIdx.x / e.slices, begin = block * e.block, end = begin + e.block; // never the last block
    const uint32_t word = e.words[end - 1], follows = e.words[end], first = e.words[begin], before = begin ? e.words[begin - 1] : e.rows;
    if (word >= e.rows || follows != word || (first == word && before == word))
        return;
    int64_t last = block; // block that begins with the word: every lane looks at another one
    for (bool more = true; more;) {
        const int64_t b = last + 1 + threadIdx.x % 64;
        const uint64_t same = __ballot(b < e.blocks && e.words[b * e.block] == word);
        last += __popcll(same);
        more = same == ~0ull;
    }
    const int x = threadIdx.x % LANES, y = threadIdx.x / LANES;
    const Piece at = piece_at<V>((static_cast<int>(blockIdx.x % e.slices) * LANES + x) * V, e.dim);
    float sum[V] = {};
    if (y == 0)
        load(e.tail + block * e.dim + at.d, sum);
    for (int64_t b = block + 1 + y; b <= last; b += AHEAD * TEAMS) {
        float head[AHEAD][V];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
            load(e.head + (b + k * TEAMS <= last ? b + k * TEAMS : b) * e.dim + at.d, head[k]);
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i)
                sum[i] += b + k * TEAMS <= last ? head[k][i] : 0.f;
    }
#pragma unroll
    for (int k = 0; k < V; ++k)
        got[y][k][x] = sum[k];
    __syncthreads();
    if (y || !at.mine)
        return;
    for (int t = 1; t < TEAMS; ++t)
#pragma unroll
        for (int k = 0; k < V; ++k)
            sum[k] += got[t][k][x];
#pragma unroll
    for (int k = 0; k < V; ++k)
        sum[k] *= e.scale;
    store(d_weight + static_cast<int64_t>(word) * e.dim + at.d, sum);
}

} // namespace lm
