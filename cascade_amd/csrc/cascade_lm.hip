// Host side of the language-model operators: argument checks, launch shapes and the C ABI declared in include/cascade_lm.h. gfx950 only.
#include "../../include/cascade_lm.h"

#include "lm_attention.hpp"
#include "lm_clip.hpp"
#include "lm_cross_entropy.hpp"
#include "lm_spans.hpp"

#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <cstdlib>

using namespace lm;

namespace {

thread_local char g_err[512] = "";

int fail(int code, const char* fmt, ...)
{
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof(g_err), fmt, ap);
    va_end(ap);
    return code;
}

int launched(const char* who)
{
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? CSA_OK : fail(CSA_ERR_HIP, "%s: a launch failed: %s", who, hipGetErrorString(e));
}

uint64_t up(uint64_t x, uint64_t to) { return (x + to - 1) / to * to; }
uint64_t parts_of(uint64_t x, uint64_t size) { return (x + size - 1) / size; }
// HIP starts fewer than 2^32 threads along an axis. What would need more is refused before the call's first launch.
bool launchable(uint64_t groups, uint64_t threads) { return groups < (1ull << 32) / threads; }
bool aligned(const void* p, uint64_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

// Hands out the pieces of a workspace, or only adds them up.
struct Carver {
    char* base;
    uint64_t used = 0;
    template <class T>
    T* take(uint64_t count)
    {
        T* at = base ? reinterpret_cast<T*>(base + used) : nullptr;
        used = up(used + count * sizeof(T), 256);
        return at;
    }
};

int check_work(const char* who, const void* work, uint64_t have, uint64_t need)
{
    if (need && (!work || !aligned(work, 256)))
        return fail(CSA_ERR_ARG, "%s: the workspace is null or not aligned to 256 bytes", who);
    if (have < need)
        return fail(CSA_ERR_ARG, "%s: a workspace of %llu bytes where %llu are needed", who, (unsigned long long)have, (unsigned long long)need);
    return CSA_OK;
}

// ---- spans ----

uint64_t span_tile(uint64_t n)
{
    return up(parts_of(n, SPAN_TILES), SPAN_TURN);
}

// ---- attention ----

int check_heads(const char* who, const char* what, const csa_lm_heads& h, const csa_lm_attention& a)
{
    if (!h.data || !aligned(h.data, 16))
        return fail(CSA_ERR_ARG, "%s: %s is null or not aligned to 16 bytes", who, what);
    if (h.token_stride % 8 || h.head_stride % 8 || h.token_stride < static_cast<int64_t>(a.head_dim) || h.token_stride >= 1 << 22 || h.head_stride < 0)
        return fail(CSA_ERR_ARG, "%s: strides of %s (%lld between tokens, %lld between heads) have to be multiples of 8, the first at least head_dim and below 2^22",
                    who, what, (long long)h.token_stride, (long long)h.head_stride);
    return CSA_OK;
}

int check_attention(const char* who, const csa_lm_attention* a, bool backward)
{
    if (!a)
        return fail(CSA_ERR_ARG, "%s: null description", who);
    if (a->type != CSA_LM_BF16 && a->type != CSA_LM_F16)
        return fail(CSA_ERR_ARG, "%s: type %d is neither CSA_LM_BF16 nor CSA_LM_F16", who, a->type);
    if (!a->kv_heads || !a->q_heads || a->q_heads % a->kv_heads || a->q_heads > 65535)
        return fail(CSA_ERR_ARG, "%s: %u heads of q do not share %u heads of k and v", who, a->q_heads, a->kv_heads);
    if (a->head_dim < 8 || a->head_dim > 128 || a->head_dim % 8)
        return fail(CSA_ERR_ARG, "%s: head_dim = %u is no multiple of 8 in [8, 128]", who, a->head_dim);
    if (a->tokens > 1u << 30)
        return fail(CSA_ERR_TOO_LARGE, "%s: %llu tokens", who, (unsigned long long)a->tokens);
    if (!(a->scale > 0.f) || a->scale > 3e38f)
        return fail(CSA_ERR_ARG, "%s: scale = %g is not positive and finite", who, a->scale);
    if (!(a->cap >= 0.f) || a->cap > 3e38f)
        return fail(CSA_ERR_ARG, "%s: cap = %g is neither 0 nor positive and finite", who, a->cap);
    if (a->tokens) {
        if (int rc = check_heads(who, "q", a->q, *a))
            return rc;
        if (int rc = check_heads(who, "k", a->k, *a))
            return rc;
        if (int rc = check_heads(who, "v", a->v, *a))
            return rc;
    }
    if (!launchable(parts_of(a->tokens, ROWS_PER_GROUP) * a->q_heads, 256) || (backward && !launchable(parts_of(a->tokens, BLOCK_ROWS), 256)))
        return fail(CSA_ERR_TOO_LARGE, "%s: %llu tokens of %u heads", who, (unsigned long long)a->tokens, a->q_heads);
    return CSA_OK;
}

Heads heads(const csa_lm_heads& h) { return {h.data, h.token_stride, h.head_stride}; }

Attention attention(const csa_lm_attention& a)
{
    return {heads(a.q), heads(a.k), heads(a.v), a.d_lo, a.d_hi, a.d_slope, static_cast<int64_t>(a.tokens), a.q_heads, a.q_heads / a.kv_heads,
            static_cast<int>(a.head_dim), a.scale, a.cap};
}

// The rows that a tile of keys meets are shared out over workgroups, each with sums of its own that are joined at the end, until there are
// KV_GROUPS workgroups (a workgroup takes half a compute unit), or up to twice as many where a share would otherwise hold more than KV_LONG tiles of rows: the
// workgroups of a long document are the last ones to end. A share has KV_TURNS tiles of rows at least, and where it can be, whole heads: workgroups next to
// each other then read the same rows (12289 tokens, 16 heads of 2: 8 shares 2.91 ms, 11 shares 3.03 ms; 16384 tokens of documents, 16 heads of 4: 4 shares 1.05 ms,
// 3 shares 1.15 ms, 2 shares 1.36 ms; 3001 tokens, 12 heads of 12: 8 shares 0.26 ms, none 0.34 ms).
// A workgroup's sums take 128 KB at 128 values a head. Rounded up to a number of shares for each group of keys, KV_GROUPS of them are less than 2 * KV_GROUPS (268 MB), twice as many
// less than 4 * KV_GROUPS (537 MB: 262016 tokens of 1 head of keys), and whole heads make half as much again of those at most (805 MB).
constexpr uint64_t KV_GROUPS = 1024, KV_LONG = 512, KV_TURNS = 16;

// The keys that a tile of rows sees are shared out in the same way where there are too few tiles for two workgroups a compute unit; a share has five tiles of
// keys at least if its rows see the whole text (4000 tokens of 4 heads trained 186 -> 113 us, 3001 of 12 heads 264 -> 215, 1000 of 8 heads 98 -> 81;
// a share of four tiles and 768 workgroups: 2000 tokens of documents of 8 heads 136 where these take 120).
constexpr uint64_t ROW_GROUPS = 512, ROW_KEYS = 5 * KEYS_PER_TILE;

uint64_t shares_of_rows(uint64_t tokens, uint64_t q_heads)
{
    const uint64_t groups = parts_of(tokens, ROWS_PER_GROUP) * q_heads;
    if (!groups || groups >= ROW_GROUPS)
        return 1;
    const uint64_t want = parts_of(ROW_GROUPS, groups), most = tokens / ROW_KEYS;
    return want < most ? want : most > 1 ? most : 1;
}

int head_width(uint64_t dim) { return dim <= 64 ? 64 : dim <= 96 ? 96 : 128; }

// Tiles are put in order where spans are given (a causal text is in order the other way round), where not all workgroups run at once anyway
// (two or three fit a compute unit), and where one workgroup can rank them.
bool may_be_ordered(uint64_t tokens, uint64_t q_heads)
{
    const uint64_t tiles = parts_of(tokens, ROWS_PER_GROUP);
    return tiles <= ORDER_TILES && tiles * q_heads > 512;
}
bool in_order(const csa_lm_attention& a) { return (a.d_lo || a.d_hi) && may_be_ordered(a.tokens, a.q_heads); }

struct AttentionWork {
    int2* bounds;
    RowBlock* blocks;
    float* parts;
    uint32_t *row_order, *key_order; // null where there is none
    uint32_t shares, row_shares;
    float* row_parts;
    float2* row_stats;
    uint64_t bytes;
    AttentionWork(void* base, uint64_t tokens, uint64_t q_heads, uint64_t kv_heads, uint64_t dim, bool backward)
    {
        Carver c{static_cast<char*>(base)};
        row_order = c.take<uint32_t>(may_be_ordered(tokens, q_heads) ? ORDER_TILES : 0);
        row_shares = static_cast<uint32_t>(shares_of_rows(tokens, q_heads));
        row_parts = c.take<float>(row_shares > 1 ? row_shares * q_heads * tokens * head_width(dim) : 0);
        row_stats = c.take<float2>(row_shares > 1 ? row_shares * q_heads * tokens : 0);
        if (!backward) {
            bytes = c.used;
            return;
        }
        key_order = c.take<uint32_t>(may_be_ordered(tokens, q_heads) ? ORDER_TILES : 0);
        const uint64_t tiles = parts_of(tokens, BLOCK_ROWS), group = q_heads / kv_heads, groups = parts_of(tokens, KEYS_PER_GROUP) * kv_heads;
        uint64_t want = groups ? parts_of(KV_GROUPS, groups) : 1;
        const uint64_t long_ones = parts_of(group * tiles, KV_LONG), twice = groups ? parts_of(2 * KV_GROUPS, groups) : 1, most = group * tiles / KV_TURNS;
        if (want < long_ones)
            want = long_ones < twice ? long_ones : twice;
        const uint64_t whole = want > group ? want / group * group : parts_of(group, group / want); // as many shares as heads, or as groups of heads
        if (whole <= 2 * want)
            want = whole;
        shares = static_cast<uint32_t>(want < most ? want : most > 1 ? most : 1);
        parts = c.take<float>(shares > 1 ? 2 * shares * kv_heads * tokens * head_width(dim) : 0);
        bounds = c.take<int2>(tiles);
        blocks = c.take<RowBlock>(tiles * q_heads);
        bytes = c.used;
    }
};

template <class Type, int DIM, int BEND>
void forward(const csa_lm_attention& a, const AttentionWork& w, const csa_lm_heads& out, float* lse, hipStream_t s)
{
    const bool order = in_order(a);
    if (order)
        tile_order_kernel<<<1, 1024, 0, s>>>(attention(a), nullptr, w.row_order, nullptr);
    attention_forward_kernel<Type, DIM, BEND><<<static_cast<uint32_t>(parts_of(a.tokens, ROWS_PER_GROUP) * a.q_heads * w.row_shares), 256, 0, s>>>(
        ForwardCall{attention(a), order ? w.row_order : nullptr, w.row_shares, w.row_parts, w.row_stats, static_cast<short*>(out.data), out.token_stride,
                    out.head_stride, lse});
    if (w.row_shares > 1)
        join_rows_kernel<Type><<<dim3(static_cast<uint32_t>(parts_of(a.tokens * (a.head_dim / 4), 256)), a.q_heads), 256, 0, s>>>(
            w.row_parts, w.row_stats, w.row_shares, static_cast<int64_t>(a.tokens), static_cast<int>(a.head_dim), DIM, static_cast<short*>(out.data),
            out.token_stride, out.head_stride, lse);
}

template <class Type, int DIM, int BEND>
void backward(const csa_lm_attention& a, const csa_lm_heads& out, const float* lse, const csa_lm_heads& d_out, const csa_lm_heads& d_q, const csa_lm_heads& d_k,
              const csa_lm_heads& d_v, const AttentionWork& w, hipStream_t s)
{
    const Attention at = attention(a);
    const uint32_t tiles = static_cast<uint32_t>(parts_of(a.tokens, BLOCK_ROWS));
    span_bounds_kernel<<<static_cast<uint32_t>(parts_of(a.tokens, 64)), 64, 0, s>>>(at, w.bounds);
    const bool order = in_order(a);
    if (order)
        tile_order_kernel<<<1, 1024, 0, s>>>(at, w.bounds, w.row_order, w.key_order);
    row_blocks_kernel<Type><<<dim3(tiles, a.q_heads), 256, 0, s>>>(at, heads(out), heads(d_out), lse, w.blocks);
    float* rests = reinterpret_cast<float*>(w.row_stats);
    attention_d_q_kernel<Type, DIM, BEND><<<static_cast<uint32_t>(parts_of(a.tokens, ROWS_PER_GROUP) * a.q_heads * w.row_shares), 256, 0, s>>>(
        QueryCall{at, order ? w.row_order : nullptr, w.row_shares, w.row_parts, rests, heads(d_out), w.blocks, tiles, static_cast<short*>(d_q.data),
                  d_q.token_stride, d_q.head_stride});
    if (w.row_shares > 1)
        join_d_q_kernel<Type><<<dim3(static_cast<uint32_t>(parts_of(a.tokens * (a.head_dim / 4), 256)), a.q_heads), 256, 0, s>>>(
            w.row_parts, rests, w.row_shares, at.tokens, at.dim, DIM, w.blocks, tiles, static_cast<short*>(d_q.data), d_q.token_stride, d_q.head_stride);
    attention_d_kv_kernel<Type, DIM, BEND><<<static_cast<uint32_t>(parts_of(a.tokens, KEYS_PER_GROUP) * a.kv_heads * w.shares), 256, 0, s>>>(
        KeyCall{at, order ? w.key_order : nullptr, heads(d_out), w.blocks, w.bounds, tiles, w.shares, w.parts, static_cast<short*>(d_k.data), d_k.token_stride,
                d_k.head_stride, static_cast<short*>(d_v.data), d_v.token_stride, d_v.head_stride});
    if (w.shares > 1)
        join_parts_kernel<Type><<<dim3(static_cast<uint32_t>(parts_of(a.tokens * (a.head_dim / 4), 256)), a.kv_heads, 2), 256, 0, s>>>(
            w.parts, w.shares, at.tokens, at.dim, DIM, static_cast<short*>(d_k.data), d_k.token_stride, d_k.head_stride, static_cast<short*>(d_v.data),
            d_v.token_stride, d_v.head_stride);
}

template <class F>
void with_type(int type, F f)
{
    if (type == CSA_LM_F16)
        f(F16());
    else
        f(Bf16());
}

// f(type, head width, how scores are bent) as types
template <class F>
void with_kind(const csa_lm_attention& a, F f)
{
    with_type(a.type, [&](auto type) {
        auto with_width = [&](auto width) {
            if (a.cap > CAP_PLAIN)
                f(type, width, std::integral_constant<int, FAR_CAP>());
            else if (a.cap > 0.f || a.d_slope)
                f(type, width, std::integral_constant<int, PLAIN>());
            else
                f(type, width, std::integral_constant<int, STRAIGHT>());
        };
        if (head_width(a.head_dim) == 64)
            with_width(std::integral_constant<int, 64>());
        else if (head_width(a.head_dim) == 96)
            with_width(std::integral_constant<int, 96>());
        else
            with_width(std::integral_constant<int, 128>());
    });
}

// ---- cross entropy ----

// Tiles of 256 x 256 use the matrix units best, one workgroup a compute unit. Where fewer than half of the places that they would take in whole
// rounds over the compute units hold words and tokens, smaller ones take less time (1024 values a row, 50257 words, forward: 200 tokens, 60 % of the
// places, 36 us and 44 in small tiles; 300 tokens, 45 %, 64 us and 49).
template <class Type>
using WideLogits = Product<Type, 256, 256, 2, 4, false, false>;
template <class Type>
using NarrowLogits = Product<Type, 128, 64, 2, 2, false, false>;
template <class Type>
using WideWeights = Product<Type, 256, 256, 2, 4, true, true>;
template <class Type>
using NarrowWeights = Product<Type, 128, 64, 2, 2, true, true>;
template <class Type>
using WideHidden = Product<Type, 256, 256, 2, 4, false, true>;
template <class Type>
using NarrowHidden = Product<Type, 64, 256, 1, 4, false, true>;

constexpr uint64_t UNITS = 256;               // compute units
constexpr uint64_t PIECE_BYTES = 256ull << 20; // of P
constexpr uint64_t PIECE_TILES = 8192;         // of 256 words: 256 rows of P, of half as much again at most, lie within 2^31 bytes
constexpr uint64_t SHARE_BYTES = 128ull << 20; // of d_hidden's shares beside the first

struct EntropyPlan {
    uint64_t padded_dim, words, piece_words, pieces; // words: of the largest piece
    uint64_t shares, share_words;
    bool narrow_logits, narrow_hidden;
    EntropyPlan(uint64_t tokens, uint64_t dim, uint64_t vocab, bool backward)
    {
        padded_dim = up(dim, 8);
        const uint64_t tiles256 = parts_of(vocab, 256);
        narrow_logits = tokens * vocab * 2 < up(tiles256 * parts_of(tokens, 256), UNITS) * 65536;
        const uint64_t fit = PIECE_BYTES / (512 * (tokens ? tokens : 1)), most_tiles = tiles256 < PIECE_TILES ? tiles256 : PIECE_TILES;
        const uint64_t per = fit && fit < most_tiles ? fit : fit ? most_tiles : 1;
        pieces = tiles256 / per;
        if (tiles256 % per * 2 >= per) // a rest of less than half a piece goes with the last one
            ++pieces;
        piece_words = per * 256;
        words = pieces * per >= tiles256 ? piece_words : (tiles256 - (pieces - 1) * per) * 256;

        narrow_hidden = tokens <= 128;
        shares = 1;
        share_words = words;
        if (!backward)
            return;
        // d_hidden has few tiles where there are few tokens: its sum over the words of a piece is then shared out, so that workgroups fill the
        // compute units (two small ones fit one) in whole rounds as well as shares can.
        const uint64_t tiles = parts_of(tokens, narrow_hidden ? 64 : 256) * parts_of(padded_dim, 256), slots = narrow_hidden ? 2 * UNITS : UNITS;
        const uint64_t room = SHARE_BYTES / (4 * (tokens * padded_dim ? tokens * padded_dim : 1)) + 1, longest = parts_of(words, 4 * SLICE);
        const uint64_t most = room < longest ? room : longest;
        double best = 0;
        for (uint64_t n = 1; n <= most && tiles && n * tiles <= 2 * slots; ++n) {
            const double used = static_cast<double>(n * tiles) / up(n * tiles, slots);
            if (used > best + 0.05) {
                best = used;
                shares = n;
            }
        }
        share_words = up(parts_of(words, shares), 2 * SLICE);
        shares = parts_of(words, share_words);
    }
};

struct EntropyWork {
    short *hidden, *weight, *kept, *p;
    float2* part;
    float *target_logit, *scale, *shares;
    uint64_t bytes;
    EntropyWork(void* base, const EntropyPlan& plan, uint64_t tokens, uint64_t vocab, bool backward, bool copies)
    {
        Carver c{static_cast<char*>(base)};
        hidden = c.take<short>(copies ? tokens * plan.padded_dim : 0);
        weight = c.take<short>(copies ? vocab * plan.padded_dim : 0);
        if (backward) {
            kept = c.take<short>(tokens * plan.padded_dim);
            p = c.take<short>(tokens * plan.words);
            shares = c.take<float>(plan.shares * tokens * plan.padded_dim);
            scale = c.take<float>(2);
        } else {
            part = c.take<float2>(parts_of(vocab, 256) * 4 * tokens);
            target_logit = c.take<float>(tokens);
        }
        bytes = c.used;
    }
};

bool walks(const void* p, int64_t stride, uint64_t dim) { return aligned(p, 16) && stride % 8 == 0 && dim % 8 == 0; }

// Whether the operator's launches all hold less than they may. copied: the rows of the larger array that has to be laid out first.
bool entropy_fits(uint64_t tokens, uint64_t dim, uint64_t vocab, bool backward, uint64_t copied)
{
    if (tokens > 1u << 30 || vocab > 1u << 30 || dim >= 1u << 22)
        return false;
    const EntropyPlan plan(tokens, dim, vocab, false); // shares of d_hidden are few workgroups: they need no check
    const uint64_t words = backward ? plan.words : vocab, values = tokens * plan.padded_dim;
    const bool logits = plan.narrow_logits ? launchable(parts_of(words, 128) * parts_of(tokens, 64), 256) : launchable(parts_of(words, 256) * parts_of(tokens, 256), 512);
    const bool copies = launchable(parts_of((backward && copied < tokens ? tokens : copied) * (plan.padded_dim / 8), 256), 256);
    if (!backward)
        return logits && copies && launchable(parts_of(tokens, tokens <= 512 ? 4 : 16), 256);
    return logits && copies && launchable(parts_of(dim, 256) * parts_of(words, 256), 512) &&
           launchable(parts_of(tokens, plan.narrow_hidden ? 64 : 256) * parts_of(dim, 256), 512) && launchable(parts_of(values / 4, 256), 256) &&
           launchable(parts_of(vocab * dim, 1024), 256);
}

int check_entropy(const char* who, bool backward, int type, const void* hidden, int64_t hidden_stride, const void* weight, int64_t weight_stride, const void* target,
                  uint64_t tokens, uint64_t dim, uint64_t vocab)
{
    if (type != CSA_LM_BF16 && type != CSA_LM_F16)
        return fail(CSA_ERR_ARG, "%s: type %d is neither CSA_LM_BF16 nor CSA_LM_F16", who, type);
    if (!dim || !vocab)
        return fail(CSA_ERR_ARG, "%s: %llu values a row, %llu words", who, (unsigned long long)dim, (unsigned long long)vocab);
    const uint64_t hidden_rows = walks(hidden, hidden_stride, dim) ? 0 : tokens, weight_rows = walks(weight, weight_stride, dim) ? 0 : vocab;
    if (!entropy_fits(tokens, dim, vocab, backward, hidden_rows > weight_rows ? hidden_rows : weight_rows))
        return fail(CSA_ERR_TOO_LARGE, "%s: %llu tokens by %llu words of %llu values in one call", who, (unsigned long long)tokens, (unsigned long long)vocab,
                    (unsigned long long)dim);
    if (!weight || !aligned(weight, 2) || (tokens && (!hidden || !aligned(hidden, 2) || !target)))
        return fail(CSA_ERR_ARG, "%s: a null or odd address", who);
    if (hidden_stride < static_cast<int64_t>(dim) || weight_stride < static_cast<int64_t>(dim) || hidden_stride >= 1 << 22 || weight_stride >= 1 << 22)
        return fail(CSA_ERR_ARG, "%s: strides of %lld and %lld values for rows of %llu", who, (long long)hidden_stride, (long long)weight_stride,
                    (unsigned long long)dim);
    return CSA_OK;
}

void lay_out(const void* in, int64_t in_stride, uint64_t rows, uint64_t dim, const int32_t* target, uint64_t vocab, short* out, uint64_t stride, hipStream_t s)
{
    if (const uint64_t threads = rows * (stride / 8))
        lay_out_rows_kernel<<<static_cast<uint32_t>(parts_of(threads, 256)), 256, 0, s>>>(static_cast<const short*>(in), in_stride, rows, dim, target, vocab, out, stride,
                                                                                          walks(in, in_stride, dim));
}

template <class Type>
void entropy_forward(const EntropyPlan& plan, const EntropyWork& w, const Operand& hidden, const Operand& weight, const int32_t* target, float* loss, float* lse,
                     hipStream_t s)
{
    typedef WideLogits<Type> W;
    typedef NarrowLogits<Type> N;
    const uint32_t mt = static_cast<uint32_t>(parts_of(weight.rows, plan.narrow_logits ? N::BM : W::BM)), nt = static_cast<uint32_t>(parts_of(hidden.rows, plan.narrow_logits ? N::BN : W::BN));
    const Logits l{weight, hidden, static_cast<int64_t>(plan.padded_dim), mt, nt, target, 0};
    if (plan.narrow_logits)
        logit_sums_kernel<N><<<mt * nt, N::THREADS, 0, s>>>(l, w.part, w.target_logit);
    else
        logit_sums_kernel<W><<<mt * nt, W::THREADS, 0, s>>>(l, w.part, w.target_logit);
    // few tokens: more runs for each, the sums would otherwise be one lane's work after the other
    const int64_t parts = mt * static_cast<int64_t>(plan.narrow_logits ? N::WM : W::WM);
    if (hidden.rows <= 512)
        join_sums_kernel<4><<<static_cast<uint32_t>(parts_of(hidden.rows, 4)), 256, 0, s>>>(w.part, parts, w.target_logit, target, hidden.rows, weight.rows, loss, lse);
    else
        join_sums_kernel<16><<<static_cast<uint32_t>(parts_of(hidden.rows, 16)), 256, 0, s>>>(w.part, parts, w.target_logit, target, hidden.rows, weight.rows, loss, lse);
}

template <class Type>
void entropy_backward(const EntropyPlan& plan, const EntropyWork& w, const Operand& hidden, const Operand& weight, const int32_t* target, const float* lse,
                      const float* d_loss, uint64_t dim, short* d_hidden, int64_t d_hidden_stride, short* d_weight, int64_t d_weight_stride, hipStream_t s)
{
    typedef WideLogits<Type> WL;
    typedef NarrowLogits<Type> NL;
    typedef WideWeights<Type> WW;
    typedef NarrowWeights<Type> NW;
    typedef WideHidden<Type> WH;
    typedef NarrowHidden<Type> NH;
    const int64_t tokens = hidden.rows, vocab = weight.rows, d = static_cast<int64_t>(dim), pd = static_cast<int64_t>(plan.padded_dim);
    const bool wide = d_weight && aligned(d_weight, 16) && d_weight_stride % 8 == 0;
    loss_scale_kernel<<<1, 1024, 0, s>>>(d_loss, target, tokens, vocab, Type::wide_range ? 1.f : 16384.f, w.scale);
    const uint32_t dt = static_cast<uint32_t>(parts_of(dim, WH::BN)), tt = static_cast<uint32_t>(parts_of(tokens, plan.narrow_hidden ? NH::BM : WH::BM));
    for (uint64_t piece = 0; piece < plan.pieces; ++piece) {
        const int64_t first = static_cast<int64_t>(piece * plan.piece_words), words = piece + 1 < plan.pieces ? static_cast<int64_t>(plan.piece_words) : vocab - first;
        const Operand part{static_cast<const short*>(weight.data) + first * weight.stride, weight.stride, words};
        const int64_t ps = static_cast<int64_t>(up(words, 8)); // rows of P
        const uint32_t lt = static_cast<uint32_t>(parts_of(words, plan.narrow_logits ? NL::BM : WL::BM)), nt = static_cast<uint32_t>(parts_of(tokens, plan.narrow_logits ? NL::BN : WL::BN));
        const Logits l{part, hidden, pd, lt, nt, target, first};
        if (plan.narrow_logits)
            logit_gradients_kernel<NL, Type><<<lt * nt, NL::THREADS, 0, s>>>(l, lse, d_loss, w.scale, vocab, w.p, ps);
        else
            logit_gradients_kernel<WL, Type><<<lt * nt, WL::THREADS, 0, s>>>(l, lse, d_loss, w.scale, vocab, w.p, ps);
        if (d_weight) {
            const Operand p{w.p, ps, words}, kept{w.kept, pd, d};
            short* to = d_weight + first * d_weight_stride;
            // small tiles where large ones would leave half of the compute units without work
            const uint32_t dw = static_cast<uint32_t>(parts_of(dim, WW::BM)), ww = static_cast<uint32_t>(parts_of(words, WW::BN));
            const uint32_t dn = static_cast<uint32_t>(parts_of(dim, NW::BM)), wn = static_cast<uint32_t>(parts_of(words, NW::BN));
            if (static_cast<uint64_t>(dw) * ww * 2 > UNITS)
                weight_gradients_kernel<WW, Type><<<dw * ww, WW::THREADS, 0, s>>>(kept, p, tokens, dw, ww, w.scale, to, d_weight_stride, wide);
            else
                weight_gradients_kernel<NW, Type><<<dn * wn, NW::THREADS, 0, s>>>(kept, p, tokens, dn, wn, w.scale, to, d_weight_stride, wide);
        }
        if (d_hidden) {
            const Operand p{w.p, ps, tokens}, across{part.data, part.stride, d};
            const uint32_t shares = static_cast<uint32_t>(plan.shares), groups = tt * dt * shares;
            if (plan.narrow_hidden)
                hidden_gradients_kernel<NH><<<groups, NH::THREADS, 0, s>>>(p, across, words, plan.share_words, tt, dt, w.shares, pd, piece > 0);
            else
                hidden_gradients_kernel<WH><<<groups, WH::THREADS, 0, s>>>(p, across, words, plan.share_words, tt, dt, w.shares, pd, piece > 0);
        }
    }
    if (d_hidden) {
        const uint64_t quads = static_cast<uint64_t>(tokens * pd / 4);
        const uint32_t shares = static_cast<uint32_t>(plan.shares);
        if (shares > 16) // many shares of few values: sixteen lanes add up those of four
            join_shares_kernel<Type, 16><<<static_cast<uint32_t>(parts_of(quads, 16)), 256, 0, s>>>(w.shares, shares, tokens, d, pd, w.scale, d_hidden, d_hidden_stride);
        else
            join_shares_kernel<Type, 1><<<static_cast<uint32_t>(parts_of(quads, 256)), 256, 0, s>>>(w.shares, shares, tokens, d, pd, w.scale, d_hidden, d_hidden_stride);
    }
}

// ---- clipping ----

// The first array of the list that is written where another one (or its own `in`, but for the same place) lies: workgroups would read it before or after, as it happens.
// `count` if there is none, `count + 1` if there is no memory to find out.
uint32_t first_overlap(const csa_lm_values* list, uint32_t count)
{
    struct Span {
        uintptr_t begin, end;
        uint32_t index;
        bool written;
    };
    Span few[128];
    Span* spans = count <= 64 ? few : static_cast<Span*>(malloc(2 * sizeof(Span) * count));
    if (!spans)
        return count + 1;
    uint32_t n = 0;
    for (uint32_t i = 0; i < count; ++i) {
        const uint64_t bytes = list[i].n * (list[i].type == CSA_LM_F32 ? 4 : 2);
        const uintptr_t in = reinterpret_cast<uintptr_t>(list[i].in), out = reinterpret_cast<uintptr_t>(list[i].out);
        if (!bytes)
            continue;
        spans[n++] = {out, out + bytes, i, true};
        if (in != out)
            spans[n++] = {in, in + bytes, i, false};
    }
    std::sort(spans, spans + n, [](const Span& a, const Span& b) { return a.begin < b.begin; });
    uintptr_t written_to = 0, read_to = 0; // where what begins earlier ends
    uint32_t found = count;
    for (uint32_t k = 0; k < n && found == count; ++k) {
        const Span& x = spans[k];
        if (x.begin < written_to || (x.written && x.begin < read_to))
            found = x.index;
        uintptr_t& to = x.written ? written_to : read_to;
        to = to < x.end ? x.end : to;
    }
    if (spans != few)
        free(spans);
    return found;
}

} // namespace

extern "C" {

const char* csa_lm_last_error(void) { return g_err; }

uint64_t csa_lm_spans_workspace(uint64_t n) { return n > SPAN_TURN ? SPAN_TILES * sizeof(int32_t) : 0; }

int csa_lm_spans_u16_dev(const uint16_t* d_text, uint64_t n, uint32_t separator, int32_t* d_lo, int32_t* d_hi, int32_t* d_target, void* d_work,
                         uint64_t work_bytes, void* stream)
{
    const char* who = "csa_lm_spans_u16_dev";
    if (n > CSA_MAX_PART_SZ)
        return fail(CSA_ERR_TOO_LARGE, "%s: %llu symbols", who, (unsigned long long)n);
    if (separator > 0xFFFF)
        return fail(CSA_ERR_ARG, "%s: separator %u is no uint16", who, separator);
    if (n == 0)
        return CSA_OK;
    if (!d_text || !d_lo || !d_hi || !d_target || !aligned(d_text, 2) || !aligned(d_lo, 4) || !aligned(d_hi, 4) || !aligned(d_target, 4))
        return fail(CSA_ERR_ARG, "%s: a null or unaligned buffer", who);
    if (int rc = check_work(who, d_work, work_bytes, csa_lm_spans_workspace(n)))
        return rc;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const uint64_t tile = span_tile(n);
    const uint32_t tiles = static_cast<uint32_t>(parts_of(n, tile));
    const bool wide = aligned(d_text, 16) && aligned(d_lo, 16) && aligned(d_hi, 16) && aligned(d_target, 16);
    if (tiles > 1)
        last_separators_kernel<<<tiles, 256, 0, s>>>(d_text, n, static_cast<uint16_t>(separator), tile, wide, static_cast<int32_t*>(d_work));
    spans_kernel<<<tiles, 256, 0, s>>>(d_text, n, static_cast<uint16_t>(separator), tile, wide, static_cast<int32_t*>(d_work), d_lo, d_hi, d_target);
    return launched(who);
}

int csa_lm_attention_forward_dev(const csa_lm_attention* a, csa_lm_heads out, float* d_lse, void* d_work, uint64_t work_bytes, void* stream)
{
    const char* who = "csa_lm_attention_forward_dev";
    if (int rc = check_attention(who, a, false))
        return rc;
    if (a->tokens == 0)
        return CSA_OK;
    if (int rc = check_heads(who, "out", out, *a))
        return rc;
    if (!d_lse || !aligned(d_lse, 4))
        return fail(CSA_ERR_ARG, "%s: d_lse is null or unaligned", who);
    const AttentionWork w(d_work, a->tokens, a->q_heads, a->kv_heads, a->head_dim, false);
    if (int rc = check_work(who, d_work, work_bytes, w.bytes))
        return rc;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    with_kind(*a, [&](auto type, auto width, auto bend) { forward<decltype(type), width(), bend()>(*a, w, out, d_lse, s); });
    return launched(who);
}

uint64_t csa_lm_attention_workspace(uint64_t tokens, uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim, uint32_t flags)
{
    return kv_heads && q_heads >= kv_heads ? AttentionWork(nullptr, tokens, q_heads, kv_heads, head_dim, flags & CSA_LM_BACKWARD).bytes : 0;
}

int csa_lm_attention_backward_dev(const csa_lm_attention* a, csa_lm_heads out, const float* d_lse, csa_lm_heads d_out, csa_lm_heads d_q, csa_lm_heads d_k,
                                  csa_lm_heads d_v, void* d_work, uint64_t work_bytes, void* stream)
{
    const char* who = "csa_lm_attention_backward_dev";
    if (int rc = check_attention(who, a, true))
        return rc;
    if (a->tokens == 0)
        return CSA_OK;
    const struct {
        const char* name;
        const csa_lm_heads& h;
    } arrays[] = {{"out", out}, {"d_out", d_out}, {"d_q", d_q}, {"d_k", d_k}, {"d_v", d_v}};
    for (const auto& x : arrays)
        if (int rc = check_heads(who, x.name, x.h, *a))
            return rc;
    if (!d_lse || !aligned(d_lse, 4))
        return fail(CSA_ERR_ARG, "%s: d_lse is null or unaligned", who);
    const AttentionWork w(d_work, a->tokens, a->q_heads, a->kv_heads, a->head_dim, true);
    if (int rc = check_work(who, d_work, work_bytes, w.bytes))
        return rc;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    with_kind(*a, [&](auto type, auto width, auto bend) { backward<decltype(type), width(), bend()>(*a, out, d_lse, d_out, d_q, d_k, d_v, w, s); });
    return launched(who);
}

uint64_t csa_lm_cross_entropy_workspace(uint64_t tokens, uint64_t dim, uint64_t vocab, uint32_t flags)
{
    const bool copies = flags & CSA_LM_COPY_ROWS || dim % 8;
    if (!dim || !vocab || !entropy_fits(tokens, dim, vocab, flags & CSA_LM_BACKWARD, !copies ? 0 : tokens > vocab ? tokens : vocab))
        return 0;
    return EntropyWork(nullptr, EntropyPlan(tokens, dim, vocab, flags & CSA_LM_BACKWARD), tokens, vocab, flags & CSA_LM_BACKWARD, copies).bytes;
}

int csa_lm_cross_entropy_forward_dev(int type, const void* d_hidden, int64_t hidden_stride, const void* d_weight, int64_t weight_stride, const int32_t* d_target,
                                     uint64_t tokens, uint64_t dim, uint64_t vocab, float* d_loss, float* d_lse, void* d_work, uint64_t work_bytes, void* stream)
{
    const char* who = "csa_lm_cross_entropy_forward_dev";
    if (int rc = check_entropy(who, false, type, d_hidden, hidden_stride, d_weight, weight_stride, d_target, tokens, dim, vocab))
        return rc;
    if (tokens == 0)
        return CSA_OK;
    if (!d_loss || !d_lse || !aligned(d_loss, 4) || !aligned(d_lse, 4))
        return fail(CSA_ERR_ARG, "%s: d_loss or d_lse is null or unaligned", who);
    const EntropyPlan plan(tokens, dim, vocab, false);
    const bool copies = !walks(d_hidden, hidden_stride, dim) || !walks(d_weight, weight_stride, dim);
    const EntropyWork w(d_work, plan, tokens, vocab, false, copies);
    if (int rc = check_work(who, d_work, work_bytes, w.bytes))
        return rc;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    Operand hidden{d_hidden, hidden_stride, static_cast<int64_t>(tokens)}, weight{d_weight, weight_stride, static_cast<int64_t>(vocab)};
    if (!walks(d_hidden, hidden_stride, dim)) {
        lay_out(d_hidden, hidden_stride, tokens, dim, nullptr, vocab, w.hidden, plan.padded_dim, s);
        hidden = {w.hidden, static_cast<int64_t>(plan.padded_dim), hidden.rows};
    }
    if (!walks(d_weight, weight_stride, dim)) {
        lay_out(d_weight, weight_stride, vocab, dim, nullptr, vocab, w.weight, plan.padded_dim, s);
        weight = {w.weight, static_cast<int64_t>(plan.padded_dim), weight.rows};
    }
    with_type(type, [&](auto t) { entropy_forward<decltype(t)>(plan, w, hidden, weight, d_target, d_loss, d_lse, s); });
    return launched(who);
}

int csa_lm_cross_entropy_backward_dev(int type, const void* d_hidden, int64_t hidden_stride, const void* d_weight, int64_t weight_stride, const int32_t* d_target,
                                      const float* d_lse, const float* d_loss_grad, uint64_t tokens, uint64_t dim, uint64_t vocab, void* d_hidden_grad,
                                      int64_t hidden_grad_stride, void* d_weight_grad, int64_t weight_grad_stride, void* d_work, uint64_t work_bytes, void* stream)
{
    const char* who = "csa_lm_cross_entropy_backward_dev";
    if (int rc = check_entropy(who, true, type, d_hidden, hidden_stride, d_weight, weight_stride, d_target, tokens, dim, vocab))
        return rc;
    if (tokens && (!d_lse || !d_loss_grad || !aligned(d_lse, 4) || !aligned(d_loss_grad, 4)))
        return fail(CSA_ERR_ARG, "%s: d_lse or d_loss_grad is null or unaligned", who);
    if ((d_hidden_grad && (!aligned(d_hidden_grad, 2) || hidden_grad_stride < static_cast<int64_t>(dim))) ||
        (d_weight_grad && (!aligned(d_weight_grad, 2) || weight_grad_stride < static_cast<int64_t>(dim))))
        return fail(CSA_ERR_ARG, "%s: a gradient's address is odd or its stride below its rows' length", who);
    const EntropyPlan plan(tokens, dim, vocab, true);
    const EntropyWork w(d_work, plan, tokens, vocab, true, !walks(d_weight, weight_stride, dim));
    if (int rc = check_work(who, d_work, work_bytes, w.bytes))
        return rc;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (tokens == 0) { // the sum over no tokens
        if (d_weight_grad)
            zero_rows_kernel<<<static_cast<uint32_t>(parts_of(vocab * dim, 1024)), 256, 0, s>>>(static_cast<short*>(d_weight_grad), weight_grad_stride, vocab, dim);
        return launched(who);
    }
    Operand weight{d_weight, weight_stride, static_cast<int64_t>(vocab)};
    lay_out(d_hidden, hidden_stride, tokens, dim, d_target, vocab, w.kept, plan.padded_dim, s);
    const Operand hidden{w.kept, static_cast<int64_t>(plan.padded_dim), static_cast<int64_t>(tokens)};
    if (!walks(d_weight, weight_stride, dim)) {
        lay_out(d_weight, weight_stride, vocab, dim, nullptr, vocab, w.weight, plan.padded_dim, s);
        weight = {w.weight, static_cast<int64_t>(plan.padded_dim), weight.rows};
    }
    with_type(type, [&](auto t) {
        entropy_backward<decltype(t)>(plan, w, hidden, weight, d_target, d_lse, d_loss_grad, dim, static_cast<short*>(d_hidden_grad), hidden_grad_stride,
                                      static_cast<short*>(d_weight_grad), weight_grad_stride, s);
    });
    return launched(who);
}

uint64_t csa_lm_clip_workspace(uint32_t count) { return parts_of(count, CLIP_TENSORS) * CLIP_GROUPS * sizeof(double); }

int csa_lm_clip_dev(const csa_lm_values* list, uint32_t count, float max_norm, float* d_norm, void* d_work, uint64_t work_bytes, void* stream)
{
    const char* who = "csa_lm_clip_dev";
    if (!list && count)
        return fail(CSA_ERR_ARG, "%s: null list", who);
    if (!(max_norm >= 0.f))
        return fail(CSA_ERR_ARG, "%s: max_norm = %g", who, max_norm);
    if (d_norm && !aligned(d_norm, 4))
        return fail(CSA_ERR_ARG, "%s: d_norm is unaligned", who);
    for (uint32_t i = 0; i < count; ++i) {
        const csa_lm_values& v = list[i];
        if (v.type != CSA_LM_BF16 && v.type != CSA_LM_F16 && v.type != CSA_LM_F32)
            return fail(CSA_ERR_ARG, "%s: array %u has type %d", who, i, v.type);
        const uint64_t size = v.type == CSA_LM_F32 ? 4 : 2;
        if (v.n && (!v.in || !v.out || !aligned(v.in, size) || !aligned(v.out, size)))
            return fail(CSA_ERR_ARG, "%s: array %u is null or not aligned to its type", who, i);
        if (v.n > 1ull << 40)
            return fail(CSA_ERR_TOO_LARGE, "%s: array %u has %llu values", who, i, (unsigned long long)v.n);
    }
    if (const uint32_t which = first_overlap(list, count); which < count)
        return fail(CSA_ERR_ARG, "%s: array %u lies where another one, or its other address, is written", who, which);
    else if (which > count)
        return fail(CSA_ERR_ARG, "%s: no memory to look over %u arrays", who, count);
    for (uint32_t begin = 0; begin < count; begin += CLIP_TENSORS) {
        uint64_t chunks = 0;
        for (uint32_t i = begin; i < count && i < begin + CLIP_TENSORS; ++i)
            chunks += parts_of(list[i].n, CLIP_CHUNK);
        if (chunks > 0x7fffffffu)
            return fail(CSA_ERR_TOO_LARGE, "%s: too many values", who);
    }
    if (int rc = check_work(who, d_work, work_bytes, csa_lm_clip_workspace(count)))
        return rc;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    double* partial = static_cast<double*>(d_work);
    uint32_t partials = 0;
    // Twice the list, as many arrays a launch as its arguments hold: all sums first, then all products.
    for (int way = 0; way < 2; ++way)
        for (uint32_t begin = 0; begin < count || (way == 1 && begin == 0); begin += CLIP_TENSORS) {
            ClipList c;
            c.count = 0;
            uint64_t chunks = 0;
            for (uint32_t i = begin; i < count && i < begin + CLIP_TENSORS; ++i)
                if (list[i].n) {
                    c.in[c.count] = list[i].in;
                    c.out[c.count] = list[i].out;
                    c.n[c.count] = list[i].n;
                    c.type[c.count] = static_cast<uint8_t>(list[i].type);
                    c.wide[c.count] = aligned(list[i].in, 16) && aligned(list[i].out, 16);
                    c.first[c.count++] = static_cast<uint32_t>(chunks);
                    chunks += parts_of(list[i].n, CLIP_CHUNK);
                }
            c.first[c.count] = static_cast<uint32_t>(chunks);
            const uint32_t groups = static_cast<uint32_t>(chunks < CLIP_GROUPS ? chunks : CLIP_GROUPS);
            if (way == 0 && groups) {
                squares_kernel<<<groups, 256, 0, s>>>(c, partial + partials);
                partials += groups;
            } else if (way == 1 && (groups || begin == 0)) { // the norm is written even of nothing
                clip_kernel<<<groups ? groups : 1, 256, 0, s>>>(c, partial, partials, max_norm, begin == 0 ? d_norm : nullptr);
            }
        }
    return launched(who);
}

} // extern "C"
