// The root-mean-square norm with the addition of the residual in front of it:
//   total = x + residual, as it is kept;  rstd = (mean of total^2 + eps)^-1/2;  out = total * rstd * gain,
// and its gradients: with g = d_out * gain and u = total * rstd,
//   d_total = rstd * (g - u * mean of g u) + what flows into total from elsewhere;  d_gain = sum over rows of d_out * u.
//
// Bound by memory: a row is read once and stays in registers, in pieces, between the sum over it and the product. A row of up to 1536 values of 16 bits, or 512 of 32 (768 of
// 16 beside a stream of 32), is one wave's, longer ones a workgroup's: four waves up to 8192 values, or 4096 where x or the stream has 32 bits, sixteen from there on. Squares are summed in 64 bits, so that no value that the type holds overflows or
// vanishes. 8192 rows of 4096 bfloat16 values with a residual: forward 45 us, 5.9 TB/s, gradients 47 us, 5.7 TB/s.
// The rows of d_gain are added up by the workgroup that meets them, in registers, and the workgroups' sums by a second kernel in a fixed order.
#pragma once
#include "lm_values.hpp"

namespace lm {

constexpr uint64_t NORM_DIM = 16384;    // values of a row that a workgroup's registers hold
constexpr uint32_t NORM_GROUPS = 768;   // of the backward kernel at most: sums of d_gain that are added up behind it

struct NormCall {
    const void *x, *residual, *gain; // gain, residual: or null
    int64_t x_stride, residual_stride, rows;
    int dim;
    double eps;
    void *out, *total;
    float* rstd;
    bool past; // results go past the caches
};

// Rows go to workgroups of four waves, a wave or all four a row, or of sixteen.
template <int WAVES>
constexpr int NORM_THREADS = WAVES == 16 ? 1024 : 256;

// The sum over a row's lanes. lds: of a place for each wave, not that of the sum before.
template <int WAVES, class X>
__device__ inline X row_sum(X x, X* lds)
{
    x = wave_sum(x);
    if (WAVES == 1)
        return x;
    if (threadIdx.x % 64 == 0)
        lds[threadIdx.x / 64] = x;
    __syncthreads();
    x = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w)
        x += lds[w];
    return x;
}

// A lane's i-th piece. A row that has ITEMS pieces a lane is longer than half as many: the first half of them is whole.
template <int V, int LANES, int ITEMS>
__device__ inline Piece piece_of_row(int i, int dim)
{
    const int first = (i * LANES + threadIdx.x % LANES) * V;
    return i < ITEMS / 2 ? Piece{first, 0, true} : piece_at<V>(first, dim);
}

template <class T, int V>
__device__ inline void store_result(bool past, T* p, const float (&x)[V])
{
    if (past)
        store<true>(p, x);
    else
        store(p, x);
}

// T: of x, gain and out, S: of residual and total. WAVES of a row, ITEMS pieces a lane.
template <class T, class S, int WAVES, int ITEMS>
__global__ __launch_bounds__(NORM_THREADS<WAVES>) void norm_forward_kernel(NormCall c)
{
    constexpr int V = PIECE<S>;
    constexpr int LANES = WAVES * 64;
    __shared__ double lds[WAVES];
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (WAVES == 1 ? 4 : 1) + (WAVES == 1 ? threadIdx.x / 64 : 0);
    if (row >= c.rows)
        return;
    const T* x = static_cast<const T*>(c.x) + row * c.x_stride;
    Piece at[ITEMS];
    float t[ITEMS][V];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        at[i] = piece_of_row<V, LANES, ITEMS>(i, c.dim);
        load(x + at[i].d, t[i]);
    }
    if (c.residual) {
        const S* residual = static_cast<const S*>(c.residual) + row * c.residual_stride;
        S* total = static_cast<S*>(c.total) + row * c.dim;
        float r[ITEMS][V];
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
            load(residual + at[i].d, r[i]);
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
#pragma unroll
            for (int k = 0; k < V; ++k)
                t[i][k] = static_cast<float>(static_cast<S>(t[i][k] + r[i][k])); // the norm is that of the sum as it is kept, which is what the gradients see
            if (at[i].mine)
                store_result(c.past, total + at[i].d, t[i]);
        }
    }
    double sum = 0;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const double y = k < at[i].skip ? 0.f : t[i][k];
            sum = fma(y, y, sum);
        }
    sum = row_sum<WAVES>(sum, lds);
    const float rstd = static_cast<float>(1.0 / sqrt(sum / c.dim + c.eps));
    if (threadIdx.x % LANES == 0)
        c.rstd[row] = rstd;
    T* out = static_cast<T*>(c.out) + row * c.dim;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        float g[V];
#pragma unroll
        for (int k = 0; k < V; ++k)
            g[k] = 1;
        if (c.gain)
            load(static_cast<const T*>(c.gain) + at[i].d, g);
#pragma unroll
        for (int k = 0; k < V; ++k)
            t[i][k] = t[i][k] * rstd * g[k];
        if (at[i].mine)
            store_result(c.past, out + at[i].d, t[i]);
    }
}

struct NormGradients {
    const void *d_out, *total, *gain, *d_total; // gain, d_total: or null
    const float* rstd;
    int64_t d_out_stride, total_stride, d_total_stride, rows;
    int dim;
    void *d_x, *d_residual; // of T and S; or null
    bool past;              // these go past the caches
    float* parts;           // a row of dim sums of d_gain for every workgroup; null: not wanted
};

// A row's values stay as they lie in memory until they are used, before the sum over the row and after it. (The next row on its way while one is worked on took more registers than it gave:
// 8192 values 84 -> 85 us, 12000 138 -> 188.)
template <class T, class S, int WAVES, int ITEMS>
__global__ __launch_bounds__(NORM_THREADS<WAVES>) void norm_backward_kernel(NormGradients c)
{
    constexpr int V = PIECE<S>, LANES = WAVES * 64;
    __shared__ float lds[2][WAVES];
    Piece at[ITEMS];
    Raw<T, V> gain[ITEMS];
    float sums[ITEMS][V];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        at[i] = piece_of_row<V, LANES, ITEMS>(i, c.dim);
#pragma unroll
        for (int k = 0; k < V; ++k)
            sums[i][k] = 0;
        if (c.gain)
            gain[i] = load_raw<T, V>(static_cast<const T*>(c.gain) + at[i].d);
    }
    struct Row {
        Raw<T, V> d_out[ITEMS];
        Raw<S, V> total[ITEMS], d_total[ITEMS];
        float rstd;
    } now;
    auto load_row = [&](Row& to, int64_t row) {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            to.d_out[i] = load_raw<T, V>(static_cast<const T*>(c.d_out) + row * c.d_out_stride + at[i].d);
            to.total[i] = load_raw<S, V>(static_cast<const S*>(c.total) + row * c.total_stride + at[i].d);
        }
        if (c.d_total)
#pragma unroll
            for (int i = 0; i < ITEMS; ++i)
                to.d_total[i] = load_raw<S, V>(static_cast<const S*>(c.d_total) + row * c.d_total_stride + at[i].d);
        to.rstd = c.rstd[row];
    };
    // g and u of a piece
    auto unpacked = [&](const Row& row, int i, float (&d_out)[V], float (&g)[V], float (&u)[V]) {
        unpack<T, V>(row.d_out[i], d_out);
        unpack<S, V>(row.total[i], u);
        float a[V];
        if (c.gain)
            unpack<T, V>(gain[i], a);
#pragma unroll
        for (int k = 0; k < V; ++k) {
            u[k] *= row.rstd;
            g[k] = c.gain ? d_out[k] * a[k] : d_out[k];
        }
    };
    int turn = 0;
    const int64_t begin = static_cast<int64_t>(blockIdx.x) * (WAVES == 1 ? 4 : 1) + (WAVES == 1 ? threadIdx.x / 64 : 0), step = static_cast<int64_t>(gridDim.x) * (WAVES == 1 ? 4 : 1);
    for (int64_t row = begin; row < c.rows; row += step, turn ^= 1) {
        load_row(now, row);
        float sum = 0, d_out[V], g[V], u[V];
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            unpacked(now, i, d_out, g, u);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                sums[i][k] += d_out[k] == 0.f ? 0.f : d_out[k] * u[k]; // what no gradient reaches (padding) may hold anything
                sum += k < at[i].skip ? 0.f : g[k] * u[k];
            }
        }
        sum = row_sum<WAVES>(sum, lds[turn]) / static_cast<float>(c.dim);
        T* d_x = static_cast<T*>(c.d_x) + row * c.dim;
        S* d_residual = static_cast<S*>(c.d_residual) + row * c.dim;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            asm volatile("" : "+v"(now.d_out[i]), "+v"(now.total[i])); // unpacked anew: kept, they would take twice the registers over the sum
            unpacked(now, i, d_out, g, u);
#pragma unroll
            for (int k = 0; k < V; ++k)
                g[k] = now.rstd * (g[k] - u[k] * sum);
            if (c.d_total) {
                float more[V];
                unpack<S, V>(now.d_total[i], more);
#pragma unroll
                for (int k = 0; k < V; ++k)
                    g[k] += more[k];
            }
            if (at[i].mine && c.d_x)
                store_result(c.past, d_x + at[i].d, g);
            if (at[i].mine && c.d_residual)
                store_result(c.past, d_residual + at[i].d, g);
        }
    }
    if (!c.parts)
        return;
    float* part = c.parts + static_cast<int64_t>(blockIdx.x) * c.dim;
    if (WAVES == 1) { // the four waves' sums of the same values
        __shared__ float all[4][ITEMS * 64 * V];
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
            if (at[i].mine)
#pragma unroll
                for (int k = 0; k < V; ++k)
                    all[threadIdx.x / 64][at[i].d + k] = sums[i][k];
        __syncthreads();
        for (int d = threadIdx.x; d < c.dim; d += 256)
            part[d] = (all[0][d] + all[1][d]) + (all[2][d] + all[3][d]);
    } else {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
            if (at[i].mine)
                store(part + at[i].d, sums[i]);
    }
}

// d_gain from the workgroups' sums: 16 values by 16 runs of them a workgroup.
template <class T>
__global__ __launch_bounds__(256) void norm_gain_kernel(const float* parts, int64_t count, int dim, T* d_gain)
{
    __shared__ float got[16][17];
    const int x = threadIdx.x % 16, y = threadIdx.x / 16, d = blockIdx.x * 16 + x;
    float sum = 0;
    if (d < dim)
#pragma unroll 8
        for (int64_t p = y; p < count; p += 16)
            sum += parts[p * dim + d];
    got[y][x] = sum;
    __syncthreads();
    if (y == 0 && d < dim) {
        for (int k = 1; k < 16; ++k)
            sum += got[k][x];
        d_gain[d] = static_cast<T>(sum);
    }
}

} // namespace lm
