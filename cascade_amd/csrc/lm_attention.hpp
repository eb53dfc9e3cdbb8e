// Attention of every position over a span of keys, and its gradients:
//   z[i][j] = scale q_i . k_j, bent to cap tanh(z / cap) where cap > 0, less slope |i - j|;   p = softmax of z over j in [lo_i, hi_i);
//   out_i = sum_j p v_j, lse_i = ln sum_j exp z;
//   D_i = d_out_i . out_i, ds = p (d_out_i . v_j - D_i) (1 - tanh^2), d_q = scale ds k, d_k = scale ds^T q, d_v = p^T d_out.
// A span is two numbers a row: causal, documents, prefixes seen both ways and windows are all spans, and so is no key at all.
//
// All three kernels keep the scores on the side where they are needed next. The matrix unit leaves column lane % 32 and rows
// 8 (r / 4) + 4 (lane / 32) + r % 4 in a lane's sixteen registers; taken as the second operand of the next product, whose sum runs
// over those rows, they are two fragments as they stand, if the first operand's values come in the same order: its LDS reads are transposed
// ones of four rows each, so the order costs nothing. Scores therefore never pass through LDS.
//   forward and d_q: a lane holds one row i; its keys run along the registers (scores transposed: K Q^T), so the softmax's maximum, sum,
//                    mask and distance are a lane's own, with one exchange between the halves of the wave.
//   d_k and d_v:     a lane holds one key and rows run along the registers; a workgroup owns its keys and walks the rows of all heads that share
//                    them, or a part of those that is joined with the others' in a fixed order, so nothing is added by atomics and the results do not depend on the order of workgroups. The scores are
//                    computed twice for that, once here and once for d_q, which also takes its score gradients in two halves (eight products instead of five).
// Tiles of keys or rows come straight from memory into LDS, one tile ahead. The 16-byte pieces of a tile's row stand at
// places that keep both kinds of reads, sixteen rows' same piece and four rows' neighbouring pieces, in different banks.
//
// Measured on 12289 causal tokens, 16 heads of 128 that share 2 (bfloat16, averages of six passes, the first of them cold): forward 0.66 ms, 940 TFLOP/s of what is seen;
// d_q 1.12 ms, 1110; d_k and d_v 1.41 ms, 880; the fastest passes 0.62, 1.08 and 1.31. Bound by the matrix units (busy 57, 68 and 53 % of the three kernels' time) and the vector
// instructions beside them (52, 58 and 35 %), which the two waves of a SIMD overlap little; LDS is busy 26 to 41 % without conflicts. A large product of the library does 1390.
#pragma once
#include "lm_common.hpp"

namespace lm {

struct Heads {
    const void* data;
    int64_t token, head; // values between tokens and between heads
};

struct Attention {
    Heads q, k, v;
    const int32_t *lo, *hi;
    const float* slope; // of each head of q, or null
    int64_t tokens;
    uint32_t q_heads, group; // group: heads of q that share one of k and v
    int dim;
    float scale, cap;
};

// x, as something that the compiler cannot tell from a new value: what is made of it is made again where it is used instead of being kept in
// registers throughout a loop.
__device__ inline int again(int x)
{
    asm volatile("" : "+v"(x));
    return x;
}

// The thread and the workgroup, for the first or the second time that a kernel does its work: the second one, which few calls need, makes all it needs by itself and
// leaves the first one its registers.
template <bool SECOND>
__device__ inline int thread_id()
{
    return SECOND ? again(threadIdx.x) : threadIdx.x;
}
template <bool SECOND>
__device__ inline uint32_t group_id()
{
    return SECOND ? __builtin_amdgcn_readfirstlane(again(blockIdx.x)) : blockIdx.x;
}
// A kernel's only argument, with which its argument segment begins, read once more.
template <class Call>
__device__ inline Call call_again()
{
    auto from = (const __attribute__((address_space(4))) char*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(from));
    Call call;
    __builtin_memcpy(&call, from, sizeof(call));
    return call;
}

template <int DIM>
struct HeadTile {
    static constexpr int PIECES = DIM / 8;
    // Place of a row's 16-byte piece. LDS serves 256 bytes at a time: sixteen lanes that read the same piece of sixteen rows meet sixteen places
    // of it, and so do 32 lanes that read half pieces, two by two pieces of four rows.
    static __device__ int place(int row, int piece)
    {
        const int turn = row >> 2 & 3;
        return piece ^ (PIECES == 16 ? (row & 3) * 4 | turn : PIECES == 8 ? (row >> 1 & 1) * 4 | turn : turn);
    }
    // A lane's reads start at two places of a tile. `place` changes bits of the piece within a run of `TURN + 1` values only, and a row is a whole
    // number of runs, so the pieces of a row are reached by flipping bits of the place and by offsets that instructions hold.
    static constexpr int TURN = PIECES == 16 ? 127 : PIECES == 8 ? 63 : 31;
    int along_, across_;
    __device__ explicit HeadTile(int lane)
    {
        const int row = lane % 32, g = lane / 16, j = lane % 16, line = 4 * (g / 2) + j / 4, col = (g % 2) * 16 + 4 * (j % 4);
        along_ = row * DIM + place(row, lane / 32) * 8;
        across_ = line * DIM + place(line, col / 8) * 8 + col % 8;
    }
    __device__ HeadTile(int along, int across) : along_(along), across_(across) {}
    __device__ HeadTile afresh() const { return {again(along_), again(across_)}; }
    // Operand with the head's values along k: rows row0 ... row0 + 31, values 16 step ... of them
    __device__ s16x8 along(const short* tile, int row0, int step) const
    {
        return read16(tile + (along_ ^ (step * 16 & TURN)) + (step * 16 & ~TURN) + row0 * DIM);
    }
    // Operand with the rows along k in the order of the registers above: values 32 e ... 32 e + 31 of the head, rows row0 ... row0 + 15
    __device__ s16x8 across(const short* tile, int row0, int e) const
    {
        const short* p = tile + (e * 32 & ~TURN) + row0 * DIM;
        const int at = across_ ^ (e * 32 & TURN); // eight rows on, `turn` differs by 2
        return join(read_turned(p + at), read_turned(p + (at ^ 16) + 8 * DIM));
    }
};

// ROWS rows of one head, padded to DIM values with zeros, by WAVES waves. Where the waves' loads together cover whole rows, sixteen or a multiple, a
// lane's place within them is the same every time, and one register holds it; heads of 12 pieces need one a load.
template <int ROWS, int DIM, int WAVES>
struct HeadLoader {
    static constexpr int TOTAL = ROWS * DIM / 8 / 64, LOADS = (TOTAL + WAVES - 1) / WAVES; // instructions, of all waves and of one
    static constexpr int STEP = WAVES * 64 * 8 / DIM;                                      // rows of an instruction of all waves
    static constexpr bool SAME = WAVES * 64 * 8 % DIM == 0 && STEP % 16 == 0;
    static_assert(ROWS * DIM / 8 % 64 == 0, "whole waves");
    int64_t line; // bytes
    uint32_t offset[SAME ? 1 : LOADS];
    __device__ void begin(const Heads& h, int dim, int wave, int lane)
    {
        line = h.token * 2;
        for (int j = 0; j < (SAME ? 1 : LOADS); ++j) {
            const int at = (j * WAVES + wave) * 64 + lane, row = at / (DIM / 8), piece = HeadTile<DIM>::place(row, at % (DIM / 8));
            offset[j] = piece * 8 < dim ? static_cast<uint32_t>(row * line + piece * 16) : OUTSIDE;
        }
    }
    // rows row0 ... of the head that `base` points at, of `rows`; those past the end are zeros
    __device__ void load(const char* base, int64_t row0, int64_t rows, short* tile, int wave) const
    {
        int left = static_cast<int>(rows - row0 < ROWS ? rows - row0 : ROWS);
        const char* from = base + row0 * line;
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const buffer_t w = window(from, left > 0 ? static_cast<uint32_t>(left) * static_cast<uint32_t>(line) : 0);
            if (TOTAL % WAVES == 0 || j * WAVES + wave < TOTAL)
                load_to_lds(w, tile + (j * WAVES + wave) * 512, offset[SAME ? 0 : j]);
            if (SAME) {
                left -= STEP;
                from += STEP * line;
            }
        }
    }
};

// A row's fragments of 16 values a step, from memory: zeros past `dim` and for rows past the end.
template <int DIM>
__device__ inline void read_rows(const Heads& h, uint32_t head, int64_t row, int64_t rows, int dim, int lane, s16x8 (&f)[DIM / 16])
{
    const short* p = static_cast<const short*>(h.data) + head * h.head + row * h.token;
#pragma unroll
    for (int s = 0; s < DIM / 16; ++s) {
        const int at = s * 16 + lane / 32 * 8;
        f[s] = row < rows && at < dim ? *reinterpret_cast<const s16x8*>(p + at) : s16x8{};
    }
}

__device__ inline int wave_min(int x)
{
    for (int d = 32; d; d /= 2)
        x = min(x, __shfl_xor(x, d));
    return x;
}
__device__ inline int wave_most(int x)
{
    for (int d = 32; d; d /= 2)
        x = max(x, __shfl_xor(x, d));
    return x;
}

constexpr int NONE = 0x7fffffff; // lo of a row that sees nothing, whose hi is 0: it lowers no minimum and raises no maximum

// lo and hi as given, to what of them there is
__device__ inline void narrow(const Attention& a, int& lo, int& hi)
{
    lo = max(lo, 0);
    hi = static_cast<int>(min(static_cast<int64_t>(hi), a.tokens));
    if (lo >= hi) {
        lo = NONE;
        hi = 0;
    }
}

__device__ inline void span_of(const Attention& a, int64_t i, int& lo, int& hi)
{
    lo = NONE;
    hi = 0;
    if (i < a.tokens) {
        lo = a.lo ? a.lo[i] : 0;
        hi = a.hi ? a.hi[i] : static_cast<int>(i) + 1;
        narrow(a, lo, hi);
    }
}

template <class Type>
__device__ inline s16x8 round8(const f32x16& x, int u)
{
    s16x8 y;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        y[i] = to16<Type>(x[8 * u + i]);
    return y;
}

// Workgroup's tile of rows and head. Neighbouring workgroup ids run on different XCDs: where there are eight heads or a multiple, an XCD gets
// neighbouring heads, which share keys and values in its L2. Tiles come in `order`, the most work first; without one the last tile comes
// first: in a causal text it sees most.
__device__ inline void place_of(uint32_t id, uint32_t heads, uint32_t tiles, const uint32_t* order, uint32_t& head, uint32_t& tile)
{
    const uint32_t in = id % heads, at = id / heads;
    head = heads % 8 == 0 ? in % 8 * (heads / 8) + in / 8 : in;
    tile = order ? order[at] : tiles - 1 - at;
}

// What round8 left of registers 8 u ... 8 u + 7 (zeros elsewhere)
template <class Type>
__device__ inline f32x16 widen(const s16x8& x, int u)
{
    f32x16 y = {};
#pragma unroll
    for (int i = 0; i < 8; ++i)
        y[8 * u + i] = to32<Type>(x[i]);
    return y;
}

// Order for the stretch of code before it: AHEAD LDS reads first, then EACH of them behind every matrix instruction as long as there are any, so that
// an operand is on its way while the ones before it are multiplied.
template <int READS, int PRODUCTS, int AHEAD, int EACH>
__device__ inline void read_ahead()
{
    constexpr int TURNS = (READS - AHEAD) / EACH;
    static_assert(TURNS <= PRODUCTS && (READS - AHEAD) % EACH == 0, "reads are shared out");
    __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
    for (int i = 0; i < TURNS; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, EACH, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x8, PRODUCTS - TURNS, 0);
}

// How scores are bent. Kernels of each kind are compiled without the code of the others, which costs them registers even where it does not run.
enum Bend : int {
    STRAIGHT, // neither a cap nor a slope
    PLAIN,    // a cap of CAP_PLAIN at most, a slope, or both
    FAR_CAP   // a larger cap, perhaps with a slope
};

// cap tanh(y), y = score / cap. As 1 - 2 / (1 + e^2y) a tanh is off by 1.5e-7 whatever y is, and the score by that part of the cap: 1e-5 at CAP_PLAIN, far below what 16-bit
// operands leave of a score, but 0.1 at a cap of 1e6. With larger caps |y| < 1/2 takes y times tanh(y) / y, a polynomial in y^2 (interpolated at Chebyshev's points, off by 6e-8), so that a score is
// off by 5e-7 of itself. Caps of CAP_PLAIN and less do not, which would cost them: 6000 tokens, 16 heads of 128 values trained 0.98 ms, with the polynomial 1.19 ms.
constexpr float CAP_PLAIN = 64.f;

// A product s bent, still to be multiplied by scale: s tanh(y) / y, y = s in. in: scale / cap, out: its inverse, finite.
__device__ inline float bend_far(float s, float in, float out)
{
    const float y = s * in, y2 = y * y;
    const float ratio = 1.f + y2 * (-0.333330679f + y2 * (0.133247505f + y2 * (-0.0529842388f + y2 * 0.0171313444f)));
    return fabsf(y) < 0.5f ? s * ratio : out - 2.f * out * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(y * (2.f * LOG2E)));
}
__device__ inline float near_in(const Attention& a) { return fminf(2.f * LOG2E * a.scale / a.cap, 3e38f); } // finite, so that a product of 0 stays 0
__device__ inline float far_out(const Attention& a) { return fminf(a.cap / a.scale, 1e38f); }

// ---- what a row may not see ----
//
// A score that a row may not see becomes a probability of 0, but 0 times an infinity or NaN that stands there is none. What no row of a workgroup sees is
// not loaded at all (padding behind a text may hold anything). Where a sum has become infinite or NaN all the same, the workgroup goes through its tiles once more, what is
// not finite in them replaced by zeros, and what sees nothing of that takes its second result: documents next to one that has gone wrong, and rows before a bad one, stay as
// they are. What does see it keeps the first, infinite or NaN, perhaps in all its values. 4096 tokens, 8 heads of 128 values trained: 0.30 ms, with one infinite row of d_out 0.57, with nothing but NaN 0.89.

template <int N>
__device__ inline bool all_finite(const f32x16 (&x)[N])
{
    float worst = 0.f;
#pragma unroll
    for (int e = 0; e < N; ++e)
#pragma unroll
        for (int r = 0; r < 16; ++r)
            worst = fmaxf(worst, x[e][r] - x[e][r] == 0.f ? 0.f : 1.f);
    return worst == 0.f;
}

template <class Type>
__device__ inline bool is_finite(short x) // of a 16-bit pattern
{
    return (x & Type::EXPONENT) != Type::EXPONENT;
}
__device__ inline bool is_finite(float x) { return x - x == 0.f; }

// Whether a lane of any of the workgroup's four waves says so. `votes` is used once.
__device__ inline bool anybody(bool mine, int (&votes)[4])
{
    const int some = __any(mine);
    if (threadIdx.x % 64 == 0)
        votes[threadIdx.x / 64] = some;
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(votes[0] | votes[1] | votes[2] | votes[3]);
}

// Zeros in place of what is not finite in a tile of 64 keys, by all waves, and whether this lane's row, which sees [lo, hi), sees any of these keys.
template <class Type, int DIM>
__device__ inline bool clear_tile(short* tile, uint32_t (&bad)[2], int key0, int lo, int hi)
{
    const int me = threadIdx.x;
    if (me < 2)
        bad[me] = 0;
    wait_for_lds();
    meet();
    for (int at = me; at < 64 * DIM / 8; at += 256) {
        s16x8 x = read16(tile + at * 8);
        bool fine = true;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (!is_finite<Type>(x[i])) {
                x[i] = 0;
                fine = false;
            }
        if (!fine) {
            const int key = at / (DIM / 8);
            *reinterpret_cast<s16x8*>(tile + at * 8) = x;
            atomicOr(bad + key / 32, 1u << key % 32);
        }
    }
    wait_for_lds();
    meet();
    const uint64_t keys = bad[0] | static_cast<uint64_t>(bad[1]) << 32;
    const int from = max(lo - key0, 0), to = min(hi - key0, 64);
    return from < to && keys >> from << (64 - (to - from)) != 0;
}

constexpr int ROWS_PER_GROUP = 128, KEYS_PER_TILE = 64;

// The part [start, stop) of the keys [lo, hi) that one of `shares` workgroups walks, whole tiles but for the last.
__device__ inline void share_of(int lo, int hi, uint32_t share, uint32_t shares, int& start, int& stop)
{
    const int64_t tiles = lo < hi ? (hi - lo + KEYS_PER_TILE - 1) / KEYS_PER_TILE : 0;
    start = lo + static_cast<int>(tiles * share / shares) * KEYS_PER_TILE;
    stop = min(hi, lo + static_cast<int>(tiles * (share + 1) / shares) * KEYS_PER_TILE);
    if (!tiles)
        start = stop = 0;
}

// Scores of a tile, still raw products: to exponents of 2 less nothing, with `unit` left to multiply. Returns with z = s * unit.
template <int BEND, int TILES>
__device__ inline void bend(const Attention& a, f32x16 (&s)[TILES], float& unit, float slope2, int row, int key0, int half)
{
    unit = a.scale * LOG2E;
    if (BEND == STRAIGHT)
        return;
    if (BEND == FAR_CAP) {
        const float in = a.scale / a.cap, back = far_out(a);
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                s[t][r] = bend_far(s[t][r], in, back);
    } else if (a.cap > 0.f) {
        const float in = near_in(a), cap2 = a.cap * LOG2E;
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) // tanh y = 1 - 2 / (1 + e^2y)
                s[t][r] = cap2 - 2.f * cap2 * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(s[t][r] * in));
        unit = 1.f;
    }
    if (a.slope) {
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int key = key0 + 32 * t + 8 * (r / 4) + 4 * half + r % 4;
                s[t][r] = s[t][r] * unit - slope2 * fabsf(static_cast<float>(row - key));
            }
        unit = 1.f;
    }
}

struct ForwardCall {
    Attention a;
    const uint32_t* order;
    uint32_t shares;
    float* parts;
    float2* stats;
    short* out;
    int64_t out_token;
    int64_t out_head;
    float* lse;
};

// The work of a workgroup, and whether the lane's row came out infinite or NaN. SECOND: once more for such rows (`lost`), with zeros in place of what is not finite.
template <class Type, int DIM, int BEND, bool SECOND>
__device__ __attribute__((always_inline)) inline bool forward_rows(const ForwardCall& call, short (&k0s)[KEYS_PER_TILE * DIM], short (&v0s)[KEYS_PER_TILE * DIM],
    short (&k1s)[KEYS_PER_TILE * DIM], short (&v1s)[KEYS_PER_TILE * DIM], uint32_t (&bad)[2], bool lost)
{
    const Attention& a = call.a;
    const uint32_t* const order = call.order;
    const uint32_t shares = call.shares;
    float* const parts = call.parts;
    float2* const stats = call.stats;
    short* const out = call.out;
    const int64_t out_token = call.out_token;
    const int64_t out_head = call.out_head;
    float* const lse = call.lse;
    const int thread = thread_id<SECOND>();
    const HeadTile<DIM> lane_at(thread % 64);
    constexpr int KT = KEYS_PER_TILE;
    const int lane = thread % 64, half = lane / 32, wave = __builtin_amdgcn_readfirstlane(thread / 64);
    uint32_t unit, tile;
    place_of(group_id<SECOND>(), a.q_heads * shares, gridDim.x / (a.q_heads * shares), order, unit, tile);
    const uint32_t head = unit / shares;
    const int64_t first = static_cast<int64_t>(tile) * ROWS_PER_GROUP, row = first + wave * 32 + lane % 32;

    // The keys that this workgroup's rows see, this wave's rows see, and all of this wave's rows see.
    int lo, hi, l2, h2;
    span_of(a, first + lane, lo, hi);
    span_of(a, first + 64 + lane, l2, h2);
    const int group_lo = __builtin_amdgcn_readfirstlane(wave_min(min(lo, l2))), group_hi = __builtin_amdgcn_readfirstlane(wave_most(max(hi, h2)));
    int start, stop;
    share_of(group_lo, group_hi, unit % shares, shares, start, stop);
    span_of(a, row, lo, hi);
    const int wave_lo = __builtin_amdgcn_readfirstlane(wave_min(lo)), wave_hi = __builtin_amdgcn_readfirstlane(wave_most(hi));
    const int all_lo = __builtin_amdgcn_readfirstlane(wave_most(lo)), all_hi = __builtin_amdgcn_readfirstlane(wave_min(hi));

    s16x8 q[DIM / 16];
    read_rows<DIM>(a.q, head, row, a.tokens, a.dim, lane, q);
    const uint32_t kv = head / a.group;
    const char* kb = reinterpret_cast<const char*>(static_cast<const short*>(a.k.data) + kv * a.k.head);
    const char* vb = reinterpret_cast<const char*>(static_cast<const short*>(a.v.data) + kv * a.v.head);
    HeadLoader<KT, DIM, 4> kl, vl;
    kl.begin(a.k, a.dim, wave, lane);
    vl.begin(a.v, a.dim, wave, lane);
    const float slope2 = a.slope ? a.slope[head] * LOG2E : 0.f;

    f32x16 o[DIM / 32];
#pragma unroll
    for (int e = 0; e < DIM / 32; ++e)
        o[e] = f32x16{};
    float top = -3.0e38f, sum = 0.f; // the running maximum may lag behind by 2^8, which spares most rescalings
    bool hit = false;                // the lane's row sees something that is not finite

    auto turn = [&](const short* ks, const short* vs, int key0) __attribute__((always_inline)) {
        if (key0 + KT <= wave_lo || key0 >= wave_hi)
            return;
        const HeadTile<DIM> tiles_at = lane_at.afresh();
        f32x16 s[2];
#pragma unroll
        for (int t = 0; t < 2; ++t)
            s[t] = f32x16{};
#pragma unroll
        for (int d = 0; d < DIM / 16; ++d)
#pragma unroll
            for (int t = 0; t < 2; ++t)
                s[t] = Type::mfma32(tiles_at.along(ks, 32 * t, d), q[d], s[t]);
        read_ahead<DIM / 8, DIM / 8, 4, 1>();
        float unit;
        bend<BEND>(a, s, unit, slope2, static_cast<int>(row), key0, half);
        if (key0 < all_lo || key0 + KT > all_hi) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int key = key0 + 32 * t + 8 * (r / 4) + 4 * half + r % 4;
                    s[t][r] = key >= lo && key < hi ? s[t][r] : -INFINITY;
                }
        }
        float most = s[0][0];
#pragma unroll
        for (int r = 1; r < 16; ++r)
            most = fmaxf(most, s[0][r]);
#pragma unroll
        for (int r = 0; r < 16; ++r)
            most = fmaxf(most, s[1][r]);
        most = fmaxf(most, other_half(most)) * unit;
        if (__any(most > top + 8.f)) {
            const float high = fmaxf(top, most), down = __builtin_amdgcn_exp2f(top - high);
            top = high;
            sum *= down;
#pragma unroll
            for (int e = 0; e < DIM / 32; ++e)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    o[e][r] *= down;
        }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[t][r] = __builtin_amdgcn_exp2f(s[t][r] * unit - top);
                sum += s[t][r];
            }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const s16x8 p = round8<Type>(s[t], u);
#pragma unroll
                for (int e = 0; e < DIM / 32; ++e)
                    o[e] = Type::mfma32(tiles_at.across(vs, 32 * t + 16 * u, e), p, o[e]);
            }
        read_ahead<DIM / 4, DIM / 8, 6, 2>();
    };

    if (start < stop) {
        kl.load(kb, start, stop, k0s, wave);
        vl.load(vb, start, stop, v0s, wave);
        for (int key0 = start; key0 < stop; key0 += 2 * KT) {
            wait_for_all();
            meet();
            kl.load(kb, key0 + KT, stop, k1s, wave);
            vl.load(vb, key0 + KT, stop, v1s, wave);
            if (SECOND)
                hit |= clear_tile<Type, DIM>(v0s, bad, key0, lo, hi);
            turn(k0s, v0s, key0);
            wait_for_all();
            meet();
            kl.load(kb, key0 + 2 * KT, stop, k0s, wave);
            vl.load(vb, key0 + 2 * KT, stop, v0s, wave);
            if (key0 + KT < stop) {
                if (SECOND)
                    hit |= clear_tile<Type, DIM>(v1s, bad, key0 + KT, lo, hi);
                turn(k1s, v1s, key0 + KT);
            }
        }
        wait_for_all();
    }
    sum += other_half(sum);
    const bool mine = row < a.tokens && (!SECOND || (lost && !hit));
    const int64_t place = (static_cast<int64_t>(unit % shares) * a.q_heads + head) * a.tokens + row;
    if (mine && shares > 1) { // shares leave their sums as they are, for the kernel that joins them
#pragma unroll
        for (int e = 0; e < DIM / 32; ++e)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<f32x4*>(parts + place * DIM + 32 * e + 8 * g + 4 * half) = f32x4{o[e][4 * g], o[e][4 * g + 1], o[e][4 * g + 2], o[e][4 * g + 3]};
        if (half == 0)
            stats[place] = make_float2(top, sum);
    } else if (mine) {
        const bool any = sum > 0.f || sum != sum;
        const float share = any ? 1.f / sum : 0.f;
        short* to = out + head * out_head + row * out_token;
#pragma unroll
        for (int e = 0; e < DIM / 32; ++e)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int d = 32 * e + 8 * g + 4 * half;
                if (d < a.dim) {
                    s16x4 y;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        y[i] = to16<Type>(o[e][4 * g + i] * share);
                    *reinterpret_cast<s16x4*>(to + d) = y;
                }
            }
        if (half == 0)
            lse[head * a.tokens + row] = any ? (top + __builtin_amdgcn_logf(sum)) * LN2 : -INFINITY;
    }
    lost = !all_finite(o);
    return lost || other_half(lost ? 1.f : 0.f) != 0.f;
}

// Up to three workgroups a compute unit where heads of 64 values are neither capped nor biased: the second pass would take registers for two (12289 tokens of 16 heads 376 us and 393). Bent ones
// are shorter with two (8191 capped tokens of 16 heads 259 us and 282); those of 96 fit three as they are, those of 128 two, by their LDS.
template <class Type, int DIM, int BEND>
__global__ __launch_bounds__(256, DIM == 64 && BEND == STRAIGHT ? 3 : 2) void attention_forward_kernel(ForwardCall call)
{
    constexpr int KT = KEYS_PER_TILE;
    __shared__ __attribute__((aligned(16))) short k0s[KT * DIM], v0s[KT * DIM], k1s[KT * DIM], v1s[KT * DIM];
    __shared__ uint32_t bad[2];
    __shared__ int votes[4];
    const bool lost = forward_rows<Type, DIM, BEND, false>(call, k0s, v0s, k1s, v1s, bad, false);
    if (anybody(lost, votes))
        forward_rows<Type, DIM, BEND, true>(call_again<ForwardCall>(), k0s, v0s, k1s, v1s, bad, lost);
}

// out and lse of a row from its shares, four values a thread: sums of exponentials of different maxima.
template <class Type>
__global__ __launch_bounds__(256) void join_rows_kernel(const float* parts, const float2* stats, uint32_t shares, int64_t tokens, int dim, int width, short* out,
                                                        int64_t out_token, int64_t out_head, float* lse)
{
    const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const int quads = dim / 4;
    if (at >= tokens * quads)
        return;
    const int64_t row = at / quads;
    const int d = static_cast<int>(at % quads) * 4;
    const uint32_t head = blockIdx.y, heads = gridDim.y;
    float high = -3.0e38f;
    for (uint32_t i = 0; i < shares; ++i)
        high = fmaxf(high, stats[(static_cast<int64_t>(i) * heads + head) * tokens + row].x);
    float sum = 0.f;
    f32x4 x = {};
    for (uint32_t i = 0; i < shares; ++i) {
        const int64_t place = (static_cast<int64_t>(i) * heads + head) * tokens + row;
        const float2 v = stats[place];
        const float factor = __builtin_amdgcn_exp2f(v.x - high);
        sum += v.y * factor;
        x += *reinterpret_cast<const f32x4*>(parts + place * width + d) * factor;
    }
    const bool any = sum > 0.f || sum != sum;
    const float share = any ? 1.f / sum : 0.f;
    s16x4 y;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        y[i] = to16<Type>(any ? x[i] * share : 0.f);
    *reinterpret_cast<s16x4*>(out + head * out_head + row * out_token + d) = y;
    if (d == 0)
        lse[head * tokens + row] = any ? (high + __builtin_amdgcn_logf(sum)) * LN2 : -INFINITY;
}

// ---- backward ----


// What the backward kernels read of 32 rows of a head: 32 values each of lse in base 2 (infinite for rows that see nothing: their
// probabilities are zeros), D, lo and hi. The block of (head, tile) is 512 bytes, one load of half a wave.
constexpr int BLOCK_ROWS = 32;
struct RowBlock {
    float lse2[BLOCK_ROWS], delta[BLOCK_ROWS];
    int lo[BLOCK_ROWS], hi[BLOCK_ROWS];
};

// The least lo and the largest hi of every 32 rows.
__global__ __launch_bounds__(64) void span_bounds_kernel(Attention a, int2* bounds)
{
    int lo, hi;
    span_of(a, static_cast<int64_t>(blockIdx.x) * 64 + threadIdx.x, lo, hi);
    for (int d = 16; d; d /= 2) {
        lo = min(lo, __shfl_xor(lo, d));
        hi = max(hi, __shfl_xor(hi, d));
    }
    if (threadIdx.x % 32 == 0) {
        const int64_t tile = blockIdx.x * 2 + threadIdx.x / 32;
        if (tile * BLOCK_ROWS < a.tokens)
            bounds[tile] = make_int2(lo, hi);
    }
}

template <class Type>
__device__ inline float dot16(const short* x, const short* y, int dim, int lane16)
{
    float sum = 0.f;
    const int d = lane16 * 8;
    if (d < dim) {
        const s16x8 a = *reinterpret_cast<const s16x8*>(x + d), b = *reinterpret_cast<const s16x8*>(y + d);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            sum += to32<Type>(a[i]) * to32<Type>(b[i]);
    }
    for (int k = 8; k; k /= 2)
        sum += __shfl_xor(sum, k);
    return sum;
}

// Row blocks of every head: sixteen lanes a row, sixteen rows a workgroup at a time.
template <class Type>
__global__ __launch_bounds__(256) void row_blocks_kernel(Attention a, Heads out, Heads d_out, const float* lse, RowBlock* blocks)
{
    const uint32_t head = blockIdx.y, tile = blockIdx.x;
    RowBlock& to = blocks[static_cast<int64_t>(head) * gridDim.x + tile];
    const int lane16 = threadIdx.x % 16;
    for (int r = threadIdx.x / 16; r < BLOCK_ROWS; r += 16) {
        const int64_t row = static_cast<int64_t>(tile) * BLOCK_ROWS + r;
        float delta = 0.f;
        if (row < a.tokens)
            delta = dot16<Type>(static_cast<const short*>(out.data) + head * out.head + row * out.token,
                                static_cast<const short*>(d_out.data) + head * d_out.head + row * d_out.token, a.dim, lane16);
        if (lane16 == 0) {
            int lo, hi;
            span_of(a, row, lo, hi);
            to.lse2[r] = lo < hi ? lse[head * a.tokens + row] * LOG2E : INFINITY;
            to.delta[r] = lo < hi ? delta : 0.f;
            to.lo[r] = lo;
            to.hi[r] = hi;
        }
    }
}

// In half precision ds is rounded to 16 bits times a power of two, and p times 2^15 in the sums for d_v: small gradients and probabilities would otherwise vanish.
// The inverse is applied in 32 bits. The power is a lane's own, that is of one row (d_q) or one key (d_k), and follows the largest ds that the lane has met: what other rows
// and keys hold, and what nobody sees, takes no bits from it. It starts too large and only becomes smaller, by which the lane's sums are then multiplied, as for the
// running maximum of a softmax; 2^3 of headroom make that rare. (6000 tokens, 16 heads of 128 values trained 0.91 ms, with one power for the whole call 0.90; 3001 tokens of 12 heads 177 us and
// 180, since that power took the norms of all rows.)
template <class Type>
struct Growth {
    float by = Type::wide_range ? 1.f : 0x1p100f;
    // ds times the power, the lane's sums brought to it. Lanes l and l ^ 32 hold parts of one row's or key's ds.
    template <int N>
    __device__ void apply(f32x16& ds, f32x16 (&sums)[N])
    {
        if (Type::wide_range)
            return;
        float most = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r)
            most = fmaxf(most, fabsf(ds[r]));
        most = fmaxf(most, other_half(most));
        if (__any(most * by > 0x1p15f && most < INFINITY)) { // an infinity is in the sums whatever the power is
            const int e = max(12 - ilogb(most), -100);
            const float less = most * by > 0x1p15f && most < INFINITY ? __builtin_amdgcn_ldexpf(1.f, e) : by, down = less / by;
            by = less;
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    sums[n][r] *= down;
        }
#pragma unroll
        for (int r = 0; r < 16; ++r)
            ds[r] *= by;
    }
    static __device__ int ilogb(float x) { return __builtin_amdgcn_frexp_expf(x) - 1; }
};
template <class Type>
constexpr float P_SHIFT = Type::wide_range ? 0.f : 15.f;

// p and ds of 32 x 32 scores: s and dp in, p and ds (both times 2^shift) out. `lse2(r)`, `delta(r)`, `distance(r)`, `seen(r)` of register r.
// With REST, returns the sum of p (dp - delta) over the lane's registers, times 2^shift.
template <int BEND, bool REST, class L, class D, class X, class S>
__device__ inline float score_gradients(const Attention& a, f32x16& s, f32x16& dp, float slope2, float shift, bool masked, L lse2, D delta, X distance,
                                        S seen)
{
    f32x16 bent;
#pragma unroll
    for (int r = 0; r < 16; ++r)
        dp[r] -= delta(r);
    float unit = a.scale * LOG2E;
    if (BEND == FAR_CAP) {
        const float in = a.scale / a.cap, back = far_out(a);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[r] = bend_far(s[r], in, back);
            const float t = s[r] * in;
            if (REST)
                bent[r] = 1.f - t * t;
            else
                dp[r] *= 1.f - t * t;
        }
    } else if (BEND == PLAIN && a.cap > 0.f) {
        const float in = near_in(a), cap2 = a.cap * LOG2E;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float t = 1.f - 2.f * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(s[r] * in));
            s[r] = cap2 * t;
            if (REST)
                bent[r] = 1.f - t * t;
            else
                dp[r] *= 1.f - t * t;
        }
        unit = 1.f;
    }
    if (BEND != STRAIGHT && a.slope) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
            s[r] = s[r] * unit - slope2 * fabsf(distance(r));
        unit = 1.f;
    }
    if (masked) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const bool there = seen(r);
            s[r] = there ? s[r] : -INFINITY;
            dp[r] = there ? dp[r] : 0.f;
            if (REST && BEND != STRAIGHT)
                bent[r] = there ? bent[r] : 0.f;
        }
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        s[r] = __builtin_amdgcn_exp2f(s[r] * unit - (lse2(r) - shift));
        dp[r] *= s[r];
    }
    float sum = 0.f;
    if (!REST)
        return sum;
#pragma unroll
    for (int r = 0; r < 16; ++r)
        sum += dp[r];
    if (BEND != STRAIGHT && a.cap > 0.f) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
            dp[r] *= bent[r];
    }
    return sum;
}

struct QueryCall {
    Attention a;
    const uint32_t* order;
    uint32_t shares;
    float* parts;
    float* rests;
    Heads d_out;
    RowBlock* blocks;
    uint32_t blocks_per_head;
    short* d_q;
    int64_t out_token;
    int64_t out_head;
};

// The work of a workgroup, and whether the lane's row came out infinite or NaN. SECOND: once more for such rows (`lost`), with zeros in place of what is not finite.
template <class Type, int DIM, int BEND, bool SECOND>
__device__ __attribute__((always_inline)) inline bool d_q_rows(const QueryCall& call, short (&k0s)[KEYS_PER_TILE * DIM], short (&v0s)[KEYS_PER_TILE * DIM],
    short (&k1s)[KEYS_PER_TILE * DIM], short (&v1s)[KEYS_PER_TILE * DIM], uint32_t (&bad)[2], bool lost)
{
    const Attention& a = call.a;
    const uint32_t* const order = call.order;
    const uint32_t shares = call.shares;
    float* const parts = call.parts;
    float* const rests = call.rests;
    const Heads& d_out = call.d_out;
    RowBlock* const blocks = call.blocks;
    const uint32_t blocks_per_head = call.blocks_per_head;
    short* const d_q = call.d_q;
    const int64_t out_token = call.out_token;
    const int64_t out_head = call.out_head;
    const int thread = thread_id<SECOND>();
    const HeadTile<DIM> lane_at(thread % 64);
    constexpr int KT = KEYS_PER_TILE;
    const int lane = thread % 64, half = lane / 32, wave = __builtin_amdgcn_readfirstlane(thread / 64);
    uint32_t unit, tile;
    place_of(group_id<SECOND>(), a.q_heads * shares, gridDim.x / (a.q_heads * shares), order, unit, tile);
    const uint32_t head = unit / shares;
    const int64_t first = static_cast<int64_t>(tile) * ROWS_PER_GROUP, row = first + wave * 32 + lane % 32;
    int lo, hi, l2, h2;
    span_of(a, first + lane, lo, hi);
    span_of(a, first + 64 + lane, l2, h2);
    const int group_lo = __builtin_amdgcn_readfirstlane(wave_min(min(lo, l2))), group_hi = __builtin_amdgcn_readfirstlane(wave_most(max(hi, h2)));
    int start, stop;
    share_of(group_lo, group_hi, unit % shares, shares, start, stop);
    span_of(a, row, lo, hi);
    const int wave_lo = __builtin_amdgcn_readfirstlane(wave_min(lo)), wave_hi = __builtin_amdgcn_readfirstlane(wave_most(hi));
    const int all_lo = __builtin_amdgcn_readfirstlane(wave_most(lo)), all_hi = __builtin_amdgcn_readfirstlane(wave_min(hi));

    s16x8 q[DIM / 16], g[DIM / 16];
    read_rows<DIM>(a.q, head, row, a.tokens, a.dim, lane, q);
    read_rows<DIM>(d_out, head, row, a.tokens, a.dim, lane, g);
    float lse2 = INFINITY, delta = 0.f;
    if (row < a.tokens) {
        const RowBlock& b = blocks[static_cast<int64_t>(head) * blocks_per_head + row / BLOCK_ROWS];
        lse2 = b.lse2[row % BLOCK_ROWS];
        delta = b.delta[row % BLOCK_ROWS]; // the second time it is the corrected one, if this kernel corrects it
    }
    const uint32_t kv = head / a.group;
    const char* kb = reinterpret_cast<const char*>(static_cast<const short*>(a.k.data) + kv * a.k.head);
    const char* vb = reinterpret_cast<const char*>(static_cast<const short*>(a.v.data) + kv * a.v.head);
    HeadLoader<KT, DIM, 4> kl, vl;
    kl.begin(a.k, a.dim, wave, lane);
    vl.begin(a.v, a.dim, wave, lane);
    const float slope2 = a.slope ? a.slope[head] * LOG2E : 0.f;
    f32x16 o[DIM / 32];
#pragma unroll
    for (int e = 0; e < DIM / 32; ++e)
        o[e] = f32x16{};
    float rest = 0.f; // sum of p (dp - D), which would be 0 if D were exact
    bool hit = false; // the lane's row sees something that is not finite
    Growth<Type> grow;

    auto turn = [&](const short* ks, const short* vs, int key0) __attribute__((always_inline)) {
        if (key0 + KT <= wave_lo || key0 >= wave_hi)
            return;
        const bool masked = key0 < all_lo || key0 + KT > all_hi;
        const HeadTile<DIM> tiles_at = lane_at.afresh();
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            f32x16 s = {}, dp = {};
#pragma unroll
            for (int d = 0; d < DIM / 16; ++d) {
                s = Type::mfma32(tiles_at.along(ks, 32 * t, d), q[d], s);
                dp = Type::mfma32(tiles_at.along(vs, 32 * t, d), g[d], dp);
            }
            read_ahead<DIM / 8, DIM / 8, 4, 1>();
            const int key = key0 + 32 * t + 4 * half, i = static_cast<int>(row);
            rest += score_gradients<BEND, true>(
                a, s, dp, slope2, 0.f, masked, [&](int) { return lse2; }, [&](int) { return delta; },
                [&](int r) { return static_cast<float>(i - (key + 8 * (r / 4) + r % 4)); },
                [&](int r) { const int k = key + 8 * (r / 4) + r % 4; return k >= lo && k < hi; });
            grow.apply(dp, o);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const s16x8 ds = round8<Type>(dp, u), low = round8<Type>(dp - widen<Type>(ds, u), u);
#pragma unroll
                for (int e = 0; e < DIM / 32; ++e) {
                    const s16x8 f = tiles_at.across(ks, 32 * t + 16 * u, e);
                    o[e] = Type::mfma32(f, ds, o[e]);
                    o[e] = Type::mfma32(f, low, o[e]);
                }
            }
            read_ahead<DIM / 4, DIM / 4, 6, 1>();
        }
    };

    if (start < stop) {
        kl.load(kb, start, stop, k0s, wave);
        vl.load(vb, start, stop, v0s, wave);
        for (int key0 = start; key0 < stop; key0 += 2 * KT) {
            wait_for_all();
            meet();
            kl.load(kb, key0 + KT, stop, k1s, wave);
            vl.load(vb, key0 + KT, stop, v1s, wave);
            if (SECOND)
                hit |= clear_tile<Type, DIM>(k0s, bad, key0, lo, hi);
            turn(k0s, v0s, key0);
            wait_for_all();
            meet();
            kl.load(kb, key0 + 2 * KT, stop, k0s, wave);
            vl.load(vb, key0 + 2 * KT, stop, v0s, wave);
            if (key0 + KT < stop) {
                if (SECOND)
                    hit |= clear_tile<Type, DIM>(k1s, bad, key0 + KT, lo, hi);
                turn(k1s, v1s, key0 + KT);
            }
        }
        wait_for_all();
    }
    rest += other_half(rest);
    const bool mine = row < a.tokens && (!SECOND || (lost && !hit));
    const float back = a.scale / grow.by;
    const int64_t place = (static_cast<int64_t>(unit % shares) * a.q_heads + head) * a.tokens + row;
    if (mine && shares > 1) { // A share knows only its own part of what D is off by: the kernel that joins them corrects D for the kernel of d_k.
#pragma unroll
        for (int e = 0; e < DIM / 32; ++e)
#pragma unroll
            for (int k = 0; k < 4; ++k)
                *reinterpret_cast<f32x4*>(parts + place * DIM + 32 * e + 8 * k + 4 * half) =
                    f32x4{o[e][4 * k], o[e][4 * k + 1], o[e][4 * k + 2], o[e][4 * k + 3]} * back;
        if (half == 0)
            rests[place] = rest;
    } else if (mine) {
        if (half == 0)
            blocks[static_cast<int64_t>(head) * blocks_per_head + row / BLOCK_ROWS].delta[row % BLOCK_ROWS] = delta + rest;
        short* to = d_q + head * out_head + row * out_token;
#pragma unroll
        for (int e = 0; e < DIM / 32; ++e)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int d = 32 * e + 8 * k + 4 * half;
                if (d < a.dim) {
                    s16x4 y;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        y[i] = to16<Type>(o[e][4 * k + i] * back);
                    *reinterpret_cast<s16x4*>(to + d) = y;
                }
            }
    }
    lost = !all_finite(o);
    return lost || other_half(lost ? 1.f : 0.f) != 0.f;
}

template <class Type, int DIM, int BEND>
__global__ __launch_bounds__(256, 2) void attention_d_q_kernel(QueryCall call)
{
    constexpr int KT = KEYS_PER_TILE;
    __shared__ __attribute__((aligned(16))) short k0s[KT * DIM], v0s[KT * DIM], k1s[KT * DIM], v1s[KT * DIM];
    __shared__ uint32_t bad[2];
    __shared__ int votes[4];
    const bool lost = d_q_rows<Type, DIM, BEND, false>(call, k0s, v0s, k1s, v1s, bad, false);
    if (anybody(lost, votes))
        d_q_rows<Type, DIM, BEND, true>(call_again<QueryCall>(), k0s, v0s, k1s, v1s, bad, lost);
}

// d_q of a row from its shares, four values a thread, and D of the row corrected.
template <class Type>
__global__ __launch_bounds__(256) void join_d_q_kernel(const float* parts, const float* rests, uint32_t shares, int64_t tokens, int dim, int width, RowBlock* blocks,
                                                       uint32_t blocks_per_head, short* d_q, int64_t out_token, int64_t out_head)
{
    const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const int quads = dim / 4;
    if (at >= tokens * quads)
        return;
    const int64_t row = at / quads;
    const int d = static_cast<int>(at % quads) * 4;
    const uint32_t head = blockIdx.y, heads = gridDim.y;
    f32x4 x = {};
    float rest = 0.f;
    for (uint32_t i = 0; i < shares; ++i) {
        const int64_t place = (static_cast<int64_t>(i) * heads + head) * tokens + row;
        x += *reinterpret_cast<const f32x4*>(parts + place * width + d);
        rest += rests[place];
    }
    s16x4 y;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        y[i] = to16<Type>(x[i]);
    *reinterpret_cast<s16x4*>(d_q + head * out_head + row * out_token + d) = y;
    if (d == 0)
        blocks[static_cast<int64_t>(head) * blocks_per_head + row / BLOCK_ROWS].delta[row % BLOCK_ROWS] += rest;
}

constexpr int KEYS_PER_GROUP = 128;

// The workgroup's 128 keys by 32 rows a turn, 32 keys a wave. Two waves of a SIMD have 256 registers each: at 128 values a head the sums of d_k and
// d_v take 128 of them, the wave's keys 32 and the scores 32; the wave's values therefore stay in LDS and are read again every turn.
struct KeyCall {
    Attention a;
    const uint32_t* order;
    Heads d_out;
    const RowBlock* blocks;
    const int2* bounds;
    uint32_t tiles;
    uint32_t shares;
    float* parts;
    short* d_k;
    int64_t dk_token;
    int64_t dk_head;
    short* d_v;
    int64_t dv_token;
    int64_t dv_head;
};

template <class Type, int DIM, int BEND, bool SECOND>
__device__ __attribute__((always_inline)) inline bool d_kv_keys(const KeyCall& call, short (&q0s)[BLOCK_ROWS * DIM], short (&g0s)[BLOCK_ROWS * DIM],
    short (&q1s)[BLOCK_ROWS * DIM], short (&g1s)[BLOCK_ROWS * DIM], short (&vs)[KEYS_PER_GROUP * DIM], RowBlock (&b0s)[2], RowBlock (&b1s)[2], int (&ends)[8],
    bool lost)
{
    const Attention& a = call.a;
    const uint32_t* const order = call.order;
    const Heads& d_out = call.d_out;
    const RowBlock* const blocks = call.blocks;
    const int2* const bounds = call.bounds;
    const uint32_t tiles = call.tiles;
    const uint32_t shares = call.shares;
    float* const parts = call.parts;
    short* const d_k = call.d_k;
    const int64_t dk_token = call.dk_token;
    const int64_t dk_head = call.dk_head;
    short* const d_v = call.d_v;
    const int64_t dv_token = call.dv_token;
    const int64_t dv_head = call.dv_head;
    const int thread = thread_id<SECOND>();
    const HeadTile<DIM> lane_at(thread % 64);
    constexpr int RT = BLOCK_ROWS;
    // A wave goes first while it feeds the matrix unit. Whole calls: 12289 tokens, 16 heads of 128 values 2.98 -> 2.94 ms; 8000 tokens, 16 heads of 96 1.060 -> 1.037;
    // with 64 values it costs: 20000 tokens, 8 heads 2.17 -> 2.28 ms; 3001 tokens, 12 heads 174 -> 181 us. The other two kernels gain nothing by it.
    constexpr bool FIRST = DIM > 64;
    const int lane = thread % 64, half = lane / 32, wave = __builtin_amdgcn_readfirstlane(thread / 64);
    const uint32_t kv_heads = a.q_heads / a.group, units = kv_heads * shares;
    uint32_t unit, which;
    place_of(group_id<SECOND>(), units, gridDim.x / units, order, unit, which);
    if (!order)
        which = gridDim.x / units - 1 - which; // the first keys, which most rows of a causal text see, first
    const uint32_t kv = unit / shares;
    const int first = static_cast<int>(which) * KEYS_PER_GROUP, last = min(first + KEYS_PER_GROUP, static_cast<int>(a.tokens)); // keys [first, last)
    const int wave_key = first + wave * 32, key = wave_key + lane % 32;

    // The first and the last tile of rows that sees any of these keys.
    int from = NONE, to = -1;
    for (uint32_t t = thread; t < tiles; t += 256) {
        const int2 b = bounds[t];
        if (b.x < last && b.y > first) {
            from = min(from, static_cast<int>(t));
            to = max(to, static_cast<int>(t));
        }
    }
    from = wave_min(from);
    to = wave_most(to);
    if (lane == 0) {
        ends[wave] = from;
        ends[4 + wave] = to;
    }
    __syncthreads();
    from = __builtin_amdgcn_readfirstlane(min(min(ends[0], ends[1]), min(ends[2], ends[3])));
    to = __builtin_amdgcn_readfirstlane(max(max(ends[4], ends[5]), max(ends[6], ends[7])));

    s16x8 k[DIM / 16];
    read_rows<DIM>(a.k, kv, key, a.tokens, a.dim, lane, k);
    {
        HeadLoader<KEYS_PER_GROUP, DIM, 4> vl;
        vl.begin(a.v, a.dim, wave, lane);
        vl.load(reinterpret_cast<const char*>(static_cast<const short*>(a.v.data) + kv * a.v.head), first, a.tokens, vs, wave);
    }
    HeadLoader<RT, DIM, 4> ql, gl;
    ql.begin(a.q, a.dim, wave, lane);
    gl.begin(d_out, a.dim, wave, lane);
    Growth<Type> grow; // of ds times 2^15, as it comes with p
    f32x16 ok[DIM / 32], ov[DIM / 32];
#pragma unroll
    for (int e = 0; e < DIM / 32; ++e)
        ok[e] = ov[e] = f32x16{};

    // Turns: the heads that share these keys, and of each the tiles from `from` to `to`; this workgroup's are `mine` of them, `begin` the first.
    const int count = from <= to ? to - from + 1 : 0;
    const int64_t turns = static_cast<int64_t>(count) * a.group, share = unit % shares;
    const int begin = static_cast<int>(turns * share / shares), mine = static_cast<int>(turns * (share + 1) / shares) - begin;
    const uint32_t first_head = kv * a.group + (count ? begin / count : 0);
    const int first_tile = from + (count ? begin % count : 0);
    int to_load = mine, load_tile = first_tile;
    uint32_t load_head = first_head;
    auto load = [&](short* qs, short* gs, RowBlock* bs) {
        const bool there = to_load > 0;
        const int64_t row0 = there ? static_cast<int64_t>(load_tile) * RT : a.tokens; // past the last one: an empty window
        const uint32_t head = there ? load_head : first_head;
        ql.load(reinterpret_cast<const char*>(static_cast<const short*>(a.q.data) + head * a.q.head), row0, a.tokens, qs, wave);
        gl.load(reinterpret_cast<const char*>(static_cast<const short*>(d_out.data) + head * d_out.head), row0, a.tokens, gs, wave);
        if (wave == 0)
            load_to_lds(window(blocks + static_cast<int64_t>(head) * tiles + load_tile, there ? sizeof(RowBlock) : 0), bs, lane * 16);
        --to_load;
        load_head += load_tile == to;
        load_tile = load_tile < to ? load_tile + 1 : from;
    };
    uint32_t head = first_head;
    int tile = first_tile;
    bool hit = false; // a row that sees the lane's key is not finite
    auto turn = [&](short* qs, short* gs, RowBlock& bs) __attribute__((always_inline)) {
        // which of the rows see any of the wave's 32 keys, and which do not see all of them
        const int lo = bs.lo[lane % 32], hi = bs.hi[lane % 32];
        // Rows that see nothing may hold anything: they become zeros, by all waves, before the tile is used. The second time so do rows that are not finite.
        bool out = lo == NONE && tile * RT + lane % 32 < static_cast<int>(a.tokens);
        if (SECOND) {
            const int r = lane % 32;
            bool fine = lo == NONE || (is_finite(bs.lse2[r]) && is_finite(bs.delta[r]));
            for (int d = 0; d < DIM && lo != NONE; d += 8) {
                const s16x8 x = read16((half ? gs : qs) + r * DIM + d);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    fine &= is_finite<Type>(x[i]);
            }
            const uint64_t gone = __ballot(!fine);
            for (uint32_t rows = static_cast<uint32_t>(gone | gone >> 32); rows; rows &= rows - 1) {
                const int c = __builtin_ctz(rows);
                hit |= key >= bs.lo[c] && key < bs.hi[c];
                out |= c == r;
            }
        }
        if (uint32_t empty = static_cast<uint32_t>(__ballot(out))) {
            if (SECOND)
                meet(); // everybody has looked at the rows
            for (; empty; empty &= empty - 1) {
                const int r = __builtin_ctz(empty), at = r * DIM + static_cast<int>(thread % (DIM / 8)) * 8;
                if (thread < DIM / 4)
                    *reinterpret_cast<s16x8*>((thread < DIM / 8 ? qs : gs) + at) = s16x8{};
                if (SECOND && thread == 0) {
                    bs.lse2[r] = INFINITY;
                    bs.delta[r] = 0.f;
                }
            }
            wait_for_lds();
            meet();
        }
        if (!__any(lo < wave_key + 32 && hi > wave_key))
            return;
        const bool masked = __any(lo > wave_key || hi < wave_key + 32);
        const HeadTile<DIM> tiles_at = lane_at.afresh();
        if (FIRST)
            __builtin_amdgcn_s_setprio(1);
        f32x16 s = {}, dp = {};
#pragma unroll
        for (int d = 0; d < DIM / 16; ++d) {
            s = Type::mfma32(tiles_at.along(qs, 0, d), k[d], s);
            dp = Type::mfma32(tiles_at.along(gs, 0, d), tiles_at.along(vs, 32 * wave, d), dp);
        }
        read_ahead<3 * DIM / 16, DIM / 8, 4, 2>();
        if (FIRST)
            __builtin_amdgcn_s_setprio(0);
        const float slope2 = a.slope ? a.slope[head] * LOG2E : 0.f;
        const int row = tile * RT + 4 * half;
        score_gradients<BEND, false>(
            a, s, dp, slope2, P_SHIFT<Type>, masked, [&](int r) { return bs.lse2[4 * half + 8 * (r / 4) + r % 4]; },
            [&](int r) { return bs.delta[4 * half + 8 * (r / 4) + r % 4]; }, [&](int r) { return static_cast<float>(row + 8 * (r / 4) + r % 4 - key); },
            [&](int r) {
                const int at = 4 * half + 8 * (r / 4) + r % 4;
                return key >= bs.lo[at] && key < bs.hi[at];
            });
        grow.apply(dp, ok);
        if (FIRST)
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const s16x8 p = round8<Type>(s, u), ds = round8<Type>(dp, u);
#pragma unroll
            for (int e = 0; e < DIM / 32; ++e) {
                ov[e] = Type::mfma32(tiles_at.across(gs, 16 * u, e), p, ov[e]);
                ok[e] = Type::mfma32(tiles_at.across(qs, 16 * u, e), ds, ok[e]);
            }
        }
        read_ahead<DIM / 4, DIM / 8, 6, 2>();
        if (FIRST)
            __builtin_amdgcn_s_setprio(0);
    };
    auto next = [&] {
        head += tile == to;
        tile = tile < to ? tile + 1 : from;
    };

    if (mine > 0) {
        load(q0s, g0s, b0s);
        for (int n = 0; n < mine; n += 2) {
            wait_for_all();
            meet();
            load(q1s, g1s, b1s);
            turn(q0s, g0s, b0s[0]);
            next();
            wait_for_all();
            meet();
            load(q0s, g0s, b0s);
            if (n + 1 < mine) {
                turn(q1s, g1s, b1s[0]);
                next();
            }
        }
    }
    wait_for_all();
    const bool writes = key < a.tokens && (!SECOND || (lost && !hit));
    const float back_v = Type::wide_range ? 1.f : 0x1p-15f, back_k = a.scale / grow.by * back_v;
    if (writes && shares > 1) {
        float* part = parts + (static_cast<int64_t>(unit) * 2 * a.tokens + key) * DIM;
#pragma unroll
        for (int e = 0; e < DIM / 32; ++e)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                f32x4 y, z;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    y[i] = ok[e][4 * x + i] * back_k;
                    z[i] = ov[e][4 * x + i] * back_v;
                }
                const int d = 32 * e + 8 * x + 4 * half;
                *reinterpret_cast<f32x4*>(part + d) = y;
                *reinterpret_cast<f32x4*>(part + a.tokens * DIM + d) = z;
            }
    } else if (writes) {
        short* kt = d_k + kv * dk_head + static_cast<int64_t>(key) * dk_token;
        short* vt = d_v + kv * dv_head + static_cast<int64_t>(key) * dv_token;
#pragma unroll
        for (int e = 0; e < DIM / 32; ++e)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int d = 32 * e + 8 * x + 4 * half;
                if (d < a.dim) {
                    s16x4 y, z;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        y[i] = to16<Type>(ok[e][4 * x + i] * back_k);
                        z[i] = to16<Type>(ov[e][4 * x + i] * back_v);
                    }
                    *reinterpret_cast<s16x4*>(kt + d) = y;
                    *reinterpret_cast<s16x4*>(vt + d) = z;
                }
            }
    }
    lost = !all_finite(ok) || !all_finite(ov);
    return lost || other_half(lost ? 1.f : 0.f) != 0.f;
}

template <class Type, int DIM, int BEND>
__global__ __launch_bounds__(256, 2) void attention_d_kv_kernel(KeyCall call)
{
    constexpr int RT = BLOCK_ROWS;
    __shared__ __attribute__((aligned(16))) short q0s[RT * DIM], g0s[RT * DIM], q1s[RT * DIM], g1s[RT * DIM], vs[KEYS_PER_GROUP * DIM];
    __shared__ __attribute__((aligned(16))) RowBlock b0s[2], b1s[2]; // the second of each is where the load's other half wave puts zeros
    __shared__ int ends[8], votes[4];
    const bool lost = d_kv_keys<Type, DIM, BEND, false>(call, q0s, g0s, q1s, g1s, vs, b0s, b1s, ends, false);
    if (anybody(lost, votes))
        d_kv_keys<Type, DIM, BEND, true>(call_again<KeyCall>(), q0s, g0s, q1s, g1s, vs, b0s, b1s, ends, lost);
}

// The order of tiles by work, most first, for texts whose spans are given: documents differ in length by more than workgroups can make up for by
// their number (six texts of 16384 tokens and documents of lognormal lengths: the last workgroup ends 10 to 25 % earlier). One workgroup
// reads all spans once, or what span_bounds_kernel has left of them if `bounds` is there, and ranks tiles by the 64-key tiles that their rows see, and by
// the 32-row tiles that see their keys. What it waits for is memory, so loads are as wide as they can be, two on their way
// together (8192 tokens: 5.4 us, four single values a load 8.6; 16384 tokens with their keys: 8.8 us from spans, 6.2 from bounds, as single values 18).
constexpr int ORDER_TILES = 1024; // of 128 rows or keys

__global__ __launch_bounds__(1024) void tile_order_kernel(Attention a, const int2* bounds, uint32_t* row_order, uint32_t* key_order)
{
    __shared__ int los[ORDER_TILES], his[ORDER_TILES]; // of the rows of a tile
    __shared__ int change[ORDER_TILES + 1];            // of the number of 32-row tiles that see a tile of keys, from the tile before it
    __shared__ __attribute__((aligned(16))) int work[ORDER_TILES];
    __shared__ int sums[16];
    const int t = threadIdx.x, lane = t % 64, tiles = static_cast<int>((a.tokens + ROWS_PER_GROUP - 1) / ROWS_PER_GROUP);
    los[t] = NONE;
    his[t] = change[t] = 0;
    __syncthreads();
    auto count = [&](int tile, int lo, int hi) { // of the rows of a 32-row tile
        if (lo < hi) {
            atomicMin(los + tile / (ROWS_PER_GROUP / BLOCK_ROWS), lo);
            atomicMax(his + tile / (ROWS_PER_GROUP / BLOCK_ROWS), hi);
            atomicAdd(change + lo / KEYS_PER_GROUP, 1);
            atomicAdd(change + (hi - 1) / KEYS_PER_GROUP + 1, -1);
        }
    };
    if (bounds) {
        const int blocks = static_cast<int>((a.tokens + BLOCK_ROWS - 1) / BLOCK_ROWS);
        for (int tile = t; tile < blocks; tile += 1024)
            count(tile, bounds[tile].x, bounds[tile].y);
    } else {
        constexpr int MINE = 4, TURNS = 2; // neighbouring rows of a lane, eight lanes to a 32-row tile, and loads of them at a time
        const bool wide = (reinterpret_cast<uintptr_t>(a.lo) | reinterpret_cast<uintptr_t>(a.hi)) % 16 == 0;
        for (int64_t first = t * MINE; first < tiles * ROWS_PER_GROUP; first += 1024 * MINE * TURNS) {
            int lo[TURNS], hi[TURNS];
#pragma unroll
            for (int u = 0; u < TURNS; ++u) {
                lo[u] = NONE;
                hi[u] = 0;
                const int64_t row = first + u * 1024 * MINE;
                int l[MINE] = {}, h[MINE];
#pragma unroll
                for (int k = 0; k < MINE; ++k)
                    h[k] = static_cast<int>(row) + k + 1;
                if (wide && row + MINE <= a.tokens) {
                    if (a.lo)
                        __builtin_memcpy(l, __builtin_assume_aligned(a.lo + row, 16), 16);
                    if (a.hi)
                        __builtin_memcpy(h, __builtin_assume_aligned(a.hi + row, 16), 16);
                }
#pragma unroll
                for (int k = 0; k < MINE; ++k) {
                    if (wide && row + MINE <= a.tokens)
                        narrow(a, l[k], h[k]);
                    else
                        span_of(a, row + k, l[k], h[k]);
                    lo[u] = min(lo[u], l[k]);
                    hi[u] = max(hi[u], h[k]);
                }
            }
#pragma unroll
            for (int u = 0; u < TURNS; ++u) {
                for (int d = 1; d < BLOCK_ROWS / MINE; d *= 2) {
                    lo[u] = min(lo[u], __shfl_xor(lo[u], d));
                    hi[u] = max(hi[u], __shfl_xor(hi[u], d));
                }
                if (t % (BLOCK_ROWS / MINE) == 0)
                    count(static_cast<int>((first + u * 1024 * MINE) / BLOCK_ROWS), lo[u], hi[u]);
            }
        }
    }
    __syncthreads();
    int lanes = 1;
    while (lanes < 64 && lanes * 2 * tiles <= 1024)
        lanes *= 2;
    for (int keys = 0; keys < (key_order ? 2 : 1); ++keys) {
        int mine = 0;
        if (keys) { // the running sum of the changes
            mine = change[t];
            for (int d = 1; d < 64; d *= 2) {
                const int below = __shfl_up(mine, d);
                mine += lane >= d ? below : 0;
            }
            if (lane == 63)
                sums[t / 64] = mine;
            __syncthreads();
            for (int w = 0; w < t / 64; ++w)
                mine += sums[w];
        } else if (los[t] < his[t]) {
            mine = (his[t] - los[t] + KEYS_PER_TILE - 1) / KEYS_PER_TILE;
        }
        work[t] = mine;
        __syncthreads();
        if (t / lanes < tiles) { // `lanes` of them for a tile
            const int tile = t / lanes;
            const uint32_t own = work[tile];
            int rank = 0;
            for (int other = t % lanes * 4; other < tiles; other += lanes * 4) {
                const u32x4 w = *reinterpret_cast<const u32x4*>(work + other); // tiles that are not there have no work and come later
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    rank += w[k] > own || (w[k] == own && other + k < tile);
            }
            for (int d = 1; d < lanes; d *= 2)
                rank += __shfl_xor(rank, d);
            if (t % lanes == 0)
                (keys ? key_order : row_order)[rank] = tile;
        }
        __syncthreads();
    }
}

// d_k (blockIdx.z 0) and d_v (1) of a head from its shares, four values a thread.
template <class Type>
__global__ __launch_bounds__(256) void join_parts_kernel(const float* parts, uint32_t shares, int64_t tokens, int dim, int width, short* d_k, int64_t dk_token,
                                                         int64_t dk_head, short* d_v, int64_t dv_token, int64_t dv_head)
{
    const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const int quads = dim / 4;
    if (at >= tokens * quads)
        return;
    const int64_t token = at / quads;
    const int d = static_cast<int>(at % quads) * 4;
    const uint32_t kv = blockIdx.y, which = blockIdx.z;
    f32x4 sum = {};
    for (uint32_t i = 0; i < shares; ++i)
        sum += *reinterpret_cast<const f32x4*>(parts + ((static_cast<int64_t>(kv * shares + i) * 2 + which) * tokens + token) * width + d);
    s16x4 y;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        y[i] = to16<Type>(sum[i]);
    short* to = which ? d_v + kv * dv_head + token * dv_token : d_k + kv * dk_head + token * dk_token;
    *reinterpret_cast<s16x4*>(to + d) = y;
}

} // namespace lm
