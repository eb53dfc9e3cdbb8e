// Host side of the language-model operators that go row by row: embeddings and norms. gfx950 only.
#include "lm_host.hpp"

#include "lm_embed.hpp"
#include "lm_norm.hpp"

#include <algorithm>
#include <cmath>
#include <type_traits>

using namespace lm;

namespace {

template <class F>
void with_values(int type, F f)
{
    if (type == CSA_LM_F32)
        f(float());
    else if (type == CSA_LM_F16)
        f(f16_t());
    else
        f(bf16_t());
}

bool is_type(int type) { return type == CSA_LM_BF16 || type == CSA_LM_F16 || type == CSA_LM_F32; }
uint64_t size_of(int type) { return type == CSA_LM_F32 ? 4 : 2; }

// Rows of an array that is read: null and unaligned addresses, and strides that do not hold a row, are refused.
int check_rows(const char* who, const char* what, const void* p, int64_t stride, uint64_t dim, int type)
{
    if (!p || !aligned(p, size_of(type)))
        return fail(CSA_ERR_ARG, "%s: %s is null or unaligned", who, what);
    if (stride < static_cast<int64_t>(dim) || stride >= 1 << 22)
        return fail(CSA_ERR_ARG, "%s: a stride of %lld values for rows of %llu of %s", who, (long long)stride, (unsigned long long)dim, what);
    return CSA_OK;
}

int check_result(const char* who, const char* what, const void* p, int type)
{
    return p && aligned(p, size_of(type)) ? CSA_OK : fail(CSA_ERR_ARG, "%s: %s is null or unaligned", who, what);
}

// Results of more bytes go past the caches, the last of which holds 256 MB: nobody would find them there.
constexpr uint64_t CACHED = 128ull << 20;

// ---- embeddings ----

constexpr uint64_t MOST_ROWS = 1ull << 31, MOST_DIM = 1 << 22;

template <class F>
void with_tokens(uint32_t bytes, F f)
{
    if (bytes == 2)
        f(uint16_t());
    else
        f(int32_t());
}

uint64_t pieces_of(int type, uint64_t dim) { return parts_of(dim, 16 / size_of(type)); }
// Up to FEW pieces a lane takes one of them, beyond four, whose loads are under way together.
constexpr uint64_t FEW = 1ull << 23;
int embed_turns(int type, uint64_t n, uint64_t dim) { return n * pieces_of(type, dim) <= FEW ? 1 : 4; }
uint64_t embed_groups(int type, uint64_t n, uint64_t dim) { return parts_of(n * pieces_of(type, dim), 256 * embed_turns(type, n, dim)); }

int check_embed(const char* who, int type, const void* tokens, uint32_t token_bytes, uint64_t n, uint64_t rows, uint64_t dim, float scale)
{
    if (!is_type(type))
        return fail(CSA_ERR_ARG, "%s: type %d", who, type);
    if (token_bytes != 2 && token_bytes != 4)
        return fail(CSA_ERR_ARG, "%s: tokens of %u bytes", who, token_bytes);
    if (!rows || dim < LEAST_DIM)
        return fail(CSA_ERR_ARG, "%s: %llu rows of %llu values; a row has at least 8", who, (unsigned long long)rows, (unsigned long long)dim);
    if (!std::isfinite(scale))
        return fail(CSA_ERR_ARG, "%s: scale = %g", who, scale);
    if (n && (!tokens || !aligned(tokens, token_bytes)))
        return fail(CSA_ERR_ARG, "%s: tokens are null or unaligned", who);
    if (n >= 1ull << 31 || rows >= MOST_ROWS || dim >= MOST_DIM || !launchable(embed_groups(type, n, dim), 256))
        return fail(CSA_ERR_TOO_LARGE, "%s: %llu tokens, %llu rows of %llu values", who, (unsigned long long)n, (unsigned long long)rows, (unsigned long long)dim);
    return CSA_OK;
}

constexpr uint64_t RANKED = 8192; // tokens at most whose places are ranked in one launch
// Up to as many segments the moving workgroups add up the counts of all themselves, which takes less than another launch (of 512 bfloat16 values, trained: 8193 tokens 41 -> 37 us,
// 32768 53 -> 51; with 64 segments 50000 would take 67 instead of 65).
constexpr uint32_t FEW_SEGMENTS = 32;

// How a weight's gradient is made.
struct EmbedPlan {
    uint64_t lanes, slices, run, block, blocks, groups, rows_each, zero_groups;
    bool sorted;     // by digits
    bool zero_first; // all of the gradient, beside the ordering's first kernel; otherwise the rows of words that are not there, beside the sums
    int passes, bits;
    uint64_t segment, segments;
    EmbedPlan(int type, uint64_t n, uint64_t rows, uint64_t dim)
    {
        const uint64_t pieces = pieces_of(type, dim);
        for (lanes = 8; lanes < 64 && lanes < pieces; lanes *= 2) {
        }
        slices = parts_of(pieces, lanes);
        // runs of 8 to 64 entries, so that there are about 2048 waves where the text has as many
        for (run = 8; run < 64 && parts_of(n, 2 * run) * slices * lanes >= 2048 * 64; run *= 2) {
        }
        block = run * (256 / lanes);
        blocks = parts_of(n, block);
        groups = blocks * slices;
        rows_each = 16384 / dim;
        rows_each = rows_each < 1 ? 1 : rows_each > ZERO_ROWS ? ZERO_ROWS : rows_each;
        sorted = n > RANKED;
        zero_first = n && (!sorted || rows >= 2 * n); // at most half of the rows are written twice
        zero_groups = zero_first ? parts_of(rows * dim * size_of(type), ZERO_BYTES) : parts_of(rows, rows_each);
        int all = 1; // bits of a word, and of `rows`, which stands for what is none
        while (rows >> all)
            ++all;
        passes = (all + DIGIT_BITS - 1) / DIGIT_BITS;
        bits = (all + passes - 1) / passes;
        segment = TURN;
        while (parts_of(n, segment) > MOST_SEGMENTS)
            segment += TURN;
        segments = parts_of(n, segment);
    }
    bool fits() const { return launchable(groups + zero_groups, 256) && launchable(zero_groups + RANKED, 1024); }
};

struct EmbedWork {
    uint32_t *words[2], *places[2], *counts, *totals;
    float *head, *tail;
    uint64_t bytes;
    EmbedWork(void* base, const EmbedPlan& plan, uint64_t n, uint64_t dim)
    {
        Carver c{static_cast<char*>(base)};
        for (int i = 0; i < 2; ++i) {
            words[i] = c.take<uint32_t>(i == 0 || (plan.sorted && plan.passes > 1) ? n : 0);
            places[i] = c.take<uint32_t>(i == 0 || (plan.sorted && plan.passes > 1) ? n : 0);
        }
        counts = c.take<uint32_t>(plan.sorted ? plan.segments << plan.bits : 0);
        totals = c.take<uint32_t>(plan.sorted ? 1ull << plan.bits : 0);
        head = c.take<float>(plan.blocks > 1 ? plan.blocks * dim : 0);
        tail = c.take<float>(plan.blocks > 1 ? plan.blocks * dim : 0);
        bytes = c.used;
    }
};

// The places of the text in the order of their words, and zeros in d_weight where the plan says so; which of the two arrays they end up in.
template <class Token>
int put_in_order(const Token* tokens, uint64_t n, uint64_t rows, const EmbedPlan& plan, const EmbedWork& w, void* d_weight, uint64_t bytes, hipStream_t s)
{
    const uint32_t zero_groups = plan.zero_first ? static_cast<uint32_t>(plan.zero_groups) : 0;
    if (!plan.sorted) {
        const uint32_t groups = static_cast<uint32_t>(parts_of(n, RANKED_EACH));
        const auto launch = [&](auto registers) {
            rank_places_kernel<Token, registers()><<<groups + zero_groups, 1024, 0, s>>>(tokens, static_cast<int>(n), static_cast<uint32_t>(rows), w.words[0], w.places[0],
                                                                                         Zeros{static_cast<char*>(d_weight), static_cast<int64_t>(bytes), groups});
        };
        if (n <= 1024)
            launch(std::integral_constant<int, 1>());
        else if (n <= 2048)
            launch(std::integral_constant<int, 2>());
        else
            launch(std::integral_constant<int, RANKED / 1024>());
        return 0;
    }
    const uint32_t digits = 1u << plan.bits, segments = static_cast<uint32_t>(plan.segments);
    const int64_t segment = static_cast<int64_t>(plan.segment);
    int to = plan.passes % 2 ? 0 : 1;
    for (int pass = 0; pass < plan.passes; ++pass, to ^= 1) {
        const Entries<Token> e{pass ? nullptr : tokens, w.words[to ^ 1], w.places[to ^ 1], static_cast<int64_t>(n), static_cast<uint32_t>(rows)};
        const Zeros zeros{static_cast<char*>(d_weight), static_cast<int64_t>(bytes), segments};
        count_digits_kernel<<<segments + (pass ? 0 : zero_groups), 256, 0, s>>>(e, segment, segments, pass * plan.bits, digits, w.counts, zeros);
        if (segments > FEW_SEGMENTS) {
            sum_digits_kernel<<<digits, 256, 0, s>>>(w.counts, segments, w.totals);
            move_digits_kernel<Token, true><<<segments, 256, 0, s>>>(e, segment, segments, pass * plan.bits, digits, w.counts, w.totals, w.words[to], w.places[to]);
        } else {
            move_digits_kernel<Token, false><<<segments, 256, 0, s>>>(e, segment, segments, pass * plan.bits, digits, w.counts, nullptr, w.words[to], w.places[to]);
        }
    }
    return to ^ 1;
}

template <class T, int LANES>
void embed_sums(const EmbedPlan& plan, const EmbedSums& e, const T* d_out, T* d_weight, hipStream_t s)
{
    embed_sums_kernel<T, LANES><<<static_cast<uint32_t>(plan.groups + (plan.zero_first ? 0 : plan.zero_groups)), 256, 0, s>>>(e, d_out, d_weight);
    if (plan.blocks > 1)
        embed_join_kernel<T, LANES><<<static_cast<uint32_t>((plan.blocks - 1) * plan.slices), 256, 0, s>>>(e, d_weight);
}

// ---- norms ----

int check_norm(const char* who, int type, int stream_type, uint64_t tokens, uint64_t dim)
{
    if (!is_type(type) || (stream_type != type && stream_type != CSA_LM_F32))
        return fail(CSA_ERR_ARG, "%s: values of type %d beside a residual of type %d", who, type, stream_type);
    if (dim < LEAST_DIM || dim > NORM_DIM)
        return fail(CSA_ERR_ARG, "%s: rows of %llu values; 8 to %llu are possible", who, (unsigned long long)dim, (unsigned long long)NORM_DIM);
    if (!launchable(tokens, dim <= 2048 ? 256 : 1024)) // of a row, at most
        return fail(CSA_ERR_TOO_LARGE, "%s: %llu tokens", who, (unsigned long long)tokens);
    return CSA_OK;
}

// f(type, type of the residual, waves a row, pieces a lane) as types: pieces are of sixteen bytes of the residual, and a row has more than half as many as fit (lm_norm.hpp counts on
// it). Lanes without a piece wait with the others, so counts in between pay: three a lane instead of lanes of four times as many waves (bfloat16, trained: 27272 rows of 1100 values
// 115 -> 88 us, 5859 of 5120 109 -> 89; float32, 2500 of 12000 222 -> 191), but for a wave's rows of float32 (42857 of 700 values 178 -> 192). Four a lane of four waves: 3662 rows of 8192
// bfloat16 values 95 us by sixteen waves, 92 by four.
template <class F>
void with_norm(int type, int stream_type, uint64_t dim, F f)
{
    with_values(type, [&](auto t) {
        auto sized = [&](auto s) {
            typedef std::integral_constant<int, 1> One;
            typedef std::integral_constant<int, 2> Two;
            typedef std::integral_constant<int, 3> Three;
            typedef std::integral_constant<int, 4> Four;
            typedef std::integral_constant<int, 16> Sixteen;
            constexpr uint64_t V = PIECE<decltype(s)>;
            if constexpr (sizeof(t) == 2)
                if (dim > 128 * V && dim <= 192 * V)
                    return f(t, s, One(), Three());
            if (dim <= 64 * V)
                f(t, s, One(), One());
            else if (dim <= 128 * V)
                f(t, s, One(), Two());
            else if (dim <= 256 * V)
                f(t, s, Four(), One());
            else if (dim <= 512 * V)
                f(t, s, Four(), Two());
            else if (dim <= 768 * V)
                f(t, s, Four(), Three());
            else if (dim <= 1024 * V)
                f(t, s, Four(), Four());
            else if (V == 8 || dim <= 2048 * V)
                f(t, s, Sixteen(), Two());
            else if constexpr (V == 4) {
                if (dim <= 3 * 1024 * V)
                    f(t, s, Sixteen(), Three());
                else
                    f(t, s, Sixteen(), Four());
            }
        };
        if (stream_type == CSA_LM_F32)
            sized(float());
        else
            sized(t);
    });
}

uint64_t norm_rows(int waves) { return waves == 1 ? 4 : 1; } // of a workgroup at a time
uint64_t norm_sums(uint64_t tokens) { return tokens < NORM_GROUPS ? tokens : NORM_GROUPS; } // rows of d_gain's sums that the workspace holds

// Workgroups of the backward kernel, each with sums of d_gain of its own: as many as fit the compute units at once, or half as many where the sums would otherwise cost more than is
// won (30000 rows of 100 values: 768 32 us, 512 34 us; 8192 of 4096: 512 95 us, 768 99 us; 5859 of 5120: 512 89 us, 768 100 us; 3662 of 8192: 512 92 us, 256 108 us; 2500 of 12000:
// 256 98 us, 512 105 us).
uint64_t norm_groups(uint64_t tokens, int waves, int items)
{
    const uint64_t all = parts_of(tokens, norm_rows(waves)), most = waves == 16 ? 256 : items == 1 ? NORM_GROUPS : 512;
    return std::min({all, most, norm_sums(tokens)});
}

} // namespace

extern "C" {

int csa_lm_embed_forward_dev(int type, const void* d_tokens, uint32_t token_bytes, uint64_t n, const void* d_weight, int64_t weight_stride, uint64_t rows, uint64_t dim,
                             float scale, void* d_out, void* stream)
{
    const char* who = "csa_lm_embed_forward_dev";
    if (int rc = check_embed(who, type, d_tokens, token_bytes, n, rows, dim, scale))
        return rc;
    if (int rc = check_rows(who, "the weight", d_weight, weight_stride, dim, type))
        return rc;
    if (n == 0)
        return CSA_OK;
    if (int rc = check_result(who, "out", d_out, type))
        return rc;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    with_values(type, [&](auto value) {
        with_tokens(token_bytes, [&](auto token) {
            typedef decltype(value) T;
            typedef decltype(token) Token;
            const auto launch = [&](auto turns, auto past) {
                embed_kernel<T, Token, turns(), past()><<<static_cast<uint32_t>(embed_groups(type, n, dim)), 256, 0, s>>>(
                    static_cast<const Token*>(d_tokens), static_cast<int64_t>(n), static_cast<const T*>(d_weight), weight_stride, static_cast<uint32_t>(rows),
                    static_cast<int>(dim), scale, static_cast<T*>(d_out));
            };
            if (embed_turns(type, n, dim) == 1)
                launch(std::integral_constant<int, 1>(), std::false_type());
            else if (n * dim * sizeof(T) <= CACHED)
                launch(std::integral_constant<int, 4>(), std::false_type());
            else
                launch(std::integral_constant<int, 4>(), std::true_type());
        });
    });
    return launched(who);
}

uint64_t csa_lm_embed_backward_workspace(int type, uint64_t n, uint64_t rows, uint64_t dim)
{
    if (!is_type(type) || n >= 1ull << 31 || !rows || rows >= MOST_ROWS || dim < LEAST_DIM || dim >= MOST_DIM)
        return 0;
    const EmbedPlan plan(type, n, rows, dim);
    return plan.fits() ? EmbedWork(nullptr, plan, n, dim).bytes : 0;
}

int csa_lm_embed_backward_dev(int type, const void* d_tokens, uint32_t token_bytes, uint64_t n, const void* d_out_grad, int64_t out_grad_stride, uint64_t rows, uint64_t dim,
                              float scale, void* d_weight_grad, void* d_work, uint64_t work_bytes, void* stream)
{
    const char* who = "csa_lm_embed_backward_dev";
    if (int rc = check_embed(who, type, d_tokens, token_bytes, n, rows, dim, scale))
        return rc;
    if (n)
        if (int rc = check_rows(who, "the gradient of out", d_out_grad, out_grad_stride, dim, type))
            return rc;
    if (int rc = check_result(who, "the gradient of the weight", d_weight_grad, type))
        return rc;
    const EmbedPlan plan(type, n, rows, dim);
    if (!plan.fits())
        return fail(CSA_ERR_TOO_LARGE, "%s: %llu tokens, %llu rows of %llu values", who, (unsigned long long)n, (unsigned long long)rows, (unsigned long long)dim);
    const EmbedWork w(d_work, plan, n, dim);
    if (int rc = check_work(who, d_work, work_bytes, w.bytes))
        return rc;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    int in = 0;
    if (n)
        with_tokens(token_bytes, [&](auto token) {
            in = put_in_order(static_cast<const decltype(token)*>(d_tokens), n, rows, plan, w, d_weight_grad, rows * dim * size_of(type), s);
        });
    const EmbedSums e{w.words[in], w.places[in], static_cast<int64_t>(n), static_cast<int64_t>(plan.run), static_cast<int64_t>(plan.block), static_cast<int64_t>(plan.blocks), out_grad_stride,
                      static_cast<int64_t>(plan.groups), static_cast<uint32_t>(rows), static_cast<uint32_t>(plan.rows_each), static_cast<int>(dim),
                      static_cast<int>(plan.slices), scale, w.head, w.tail};
    with_values(type, [&](auto value) {
        typedef decltype(value) T;
        const T* d_out = static_cast<const T*>(d_out_grad);
        T* d_weight = static_cast<T*>(d_weight_grad);
        if (plan.lanes == 8)
            embed_sums<T, 8>(plan, e, d_out, d_weight, s);
        else if (plan.lanes == 16)
            embed_sums<T, 16>(plan, e, d_out, d_weight, s);
        else if (plan.lanes == 32)
            embed_sums<T, 32>(plan, e, d_out, d_weight, s);
        else
            embed_sums<T, 64>(plan, e, d_out, d_weight, s);
    });
    return launched(who);
}

int csa_lm_norm_forward_dev(int type, int stream_type, const void* d_x, int64_t x_stride, const void* d_residual, int64_t residual_stride, const void* d_gain, float eps,
                            uint64_t tokens, uint64_t dim, void* d_out, void* d_total, float* d_rstd, void* stream)
{
    const char* who = "csa_lm_norm_forward_dev";
    if (int rc = check_norm(who, type, stream_type, tokens, dim))
        return rc;
    if (!(eps > 0.f) || !std::isfinite(eps))
        return fail(CSA_ERR_ARG, "%s: eps = %g is not positive and finite", who, eps);
    if (!d_residual && stream_type != type)
        return fail(CSA_ERR_ARG, "%s: without a residual its type is that of x", who);
    if (d_gain && !aligned(d_gain, size_of(type)))
        return fail(CSA_ERR_ARG, "%s: the gain is unaligned", who);
    if (tokens == 0)
        return CSA_OK;
    if (int rc = check_rows(who, "x", d_x, x_stride, dim, type))
        return rc;
    if (d_residual) {
        if (int rc = check_rows(who, "the residual", d_residual, residual_stride, dim, stream_type))
            return rc;
        if (int rc = check_result(who, "total", d_total, stream_type))
            return rc;
    }
    if (int rc = check_result(who, "out", d_out, type))
        return rc;
    if (int rc = check_result(who, "rstd", d_rstd, CSA_LM_F32))
        return rc;
    const NormCall c{d_x, d_residual, d_gain, x_stride, residual_stride, static_cast<int64_t>(tokens), static_cast<int>(dim), eps, d_out, d_total, d_rstd,
                     tokens * dim * (size_of(type) + (d_residual ? size_of(stream_type) : 0)) > CACHED};
    with_norm(type, stream_type, dim, [&](auto t, auto s, auto waves, auto items) {
        norm_forward_kernel<decltype(t), decltype(s), waves(), items()>
            <<<static_cast<uint32_t>(parts_of(tokens, norm_rows(waves()))), NORM_THREADS<waves()>, 0, static_cast<hipStream_t>(stream)>>>(c);
    });
    return launched(who);
}

uint64_t csa_lm_norm_backward_workspace(uint64_t tokens, uint64_t dim)
{
    return dim < LEAST_DIM || dim > NORM_DIM ? 0 : up(norm_sums(tokens) * dim * sizeof(float), 256);
}

int csa_lm_norm_backward_dev(int type, int stream_type, const void* d_out_grad, int64_t out_grad_stride, const void* d_total, int64_t total_stride, const float* d_rstd,
                             const void* d_gain, const void* d_total_grad, int64_t total_grad_stride, uint64_t tokens, uint64_t dim, void* d_x_grad, void* d_residual_grad,
                             void* d_gain_grad, void* d_work, uint64_t work_bytes, void* stream)
{
    const char* who = "csa_lm_norm_backward_dev";
    if (int rc = check_norm(who, type, stream_type, tokens, dim))
        return rc;
    if ((d_gain && !aligned(d_gain, size_of(type))) || !aligned(d_gain_grad, size_of(type)) || !aligned(d_x_grad, size_of(type)) ||
        !aligned(d_residual_grad, size_of(stream_type)))
        return fail(CSA_ERR_ARG, "%s: the gain or a gradient is unaligned", who);
    if (tokens) {
        if (int rc = check_rows(who, "the gradient of out", d_out_grad, out_grad_stride, dim, type))
            return rc;
        if (int rc = check_rows(who, "total", d_total, total_stride, dim, stream_type))
            return rc;
        if (d_total_grad)
            if (int rc = check_rows(who, "the gradient of total", d_total_grad, total_grad_stride, dim, stream_type))
                return rc;
        if (int rc = check_result(who, "rstd", d_rstd, CSA_LM_F32))
            return rc;
    }
    if (d_gain_grad)
        if (int rc = check_work(who, d_work, work_bytes, csa_lm_norm_backward_workspace(tokens, dim)))
            return rc;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    uint64_t groups = 0;
    float* parts = d_gain_grad ? static_cast<float*>(d_work) : nullptr;
    const NormGradients c{d_out_grad, d_total, d_gain, d_total_grad, d_rstd, out_grad_stride, total_stride, total_grad_stride, static_cast<int64_t>(tokens),
                          static_cast<int>(dim), d_x_grad, d_residual_grad,
                          tokens * dim * ((d_x_grad ? size_of(type) : 0) + (d_residual_grad ? size_of(stream_type) : 0)) > CACHED, parts};
    if (tokens)
        with_norm(type, stream_type, dim, [&](auto t, auto r, auto waves, auto items) {
            groups = norm_groups(tokens, waves(), items());
            norm_backward_kernel<decltype(t), decltype(r), waves(), items()><<<static_cast<uint32_t>(groups), NORM_THREADS<waves()>, 0, s>>>(c);
        });
    if (d_gain_grad)
        with_values(type, [&](auto t) {
            norm_gain_kernel<<<static_cast<uint32_t>(parts_of(dim, 16)), 256, 0, s>>>(parts, static_cast<int64_t>(groups), static_cast<int>(dim),
                                                                                     static_cast<decltype(t)*>(d_gain_grad));
        });
    return launched(who);
}

} // extern "C"
