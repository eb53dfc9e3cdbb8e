// The root-mean-square norm with the addition of the residual in front of it:
//   total = x + residual, as it is kept;  rstd = (mean of total^2 + eps)^-1/2;  out = total * rstd * gain,
// and its gradients: with g = d_out * gain and u = total * rstd,
//   d_total = rstd * (g - u * mean of g u) + what flows into total from elsewhere;  d_gain = sum over rows of d_out * u.
//
// Bound by memory: a row is read once and stays in registers, in pieces, between the sum over it and the product. A row of up to 1024 values is one
// wave's, longer ones a workgroup's. Squares are summed in 64 bits, so that no value that the type holds overflows or vanishes.
// The rows of d_gain are added up by the workgroup that meets them, in registers, and the workgroups' sums by a second kernel in a fixed order.
#pragma once
#include "lm_values.hpp"

namespace lm {

constexpr uint64_t NORM_DIM = 16384;    // values of a row that a workgroup's registers hold
constexpr uint32_t NORM_GROUPS = 512;   // of the backward kernel: sums of d_gain that are added up behind it

struct NormCall {
    const void *x, *residual, *gain; // gain, residual: or null
    int64_t x_stride, residual_stride, rows;
    int dim;
    double eps;
    void *out, *total;
    float* rstd;
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
        at[i] = piece_at<V>((i * LANES + threadIdx.x % LANES) * V, c.dim);
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
                store(total + at[i].d, t[i]);
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
            store(out + at[i].d, t[i]);
    }
}

struct NormGradients {
    const void *d_out, *total, *gain, *d_total; // gain, d_total: or null
    const float* rstd;
    int64_t d_out_stride, total_stride, d_total_stride, rows;
    int dim;
    void *d_x, *d_residual; // of T and S; or null
    float* parts;           // a row of dim sums of d_gain for every workgroup; null: not wanted
};

template <class T, class S, int WAVES, int ITEMS>
__global__ __launch_bounds__(NORM_THREADS<WAVES>) void norm_backward_kernel(NormGradients c)
{
    constexpr int V = PIECE<S>;
    constexpr int LANES = WAVES * 64;
    __shared__ float lds[2][WAVES];
    Piece at[ITEMS];
    float gain[ITEMS][V], sums[ITEMS][V];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        at[i] = piece_at<V>((i * LANES + threadIdx.x % LANES) * V, c.dim);
#pragma unroll
        for (int k = 0; k < V; ++k)
            gain[i][k] = 1, sums[i][k] = 0;
        if (c.gain)
            load(static_cast<const T*>(c.gain) + at[i].d, gain[i]);
    }
    int turn = 0;
    const int64_t begin = static_cast<int64_t>(blockIdx.x) * (WAVES == 1 ? 4 : 1) + (WAVES == 1 ? threadIdx.x / 64 : 0), step = static_cast<int64_t>(gridDim.x) * (WAVES == 1 ? 4 : 1);
    for (int64_t row = begin; row < c.rows; row += step, turn ^= 1) {
        const T* d_out = static_cast<const T*>(c.d_out) + row * c.d_out_stride;
        const S* total = static_cast<const S*>(c.total) + row * c.total_stride;
        const S* d_total = static_cast<const S*>(c.d_total) + row * c.d_total_stride;
        float g[ITEMS][V], u[ITEMS][V], more[ITEMS][V] = {}, sum = 0;
        const float rstd = c.rstd[row];
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            load(d_out + at[i].d, g[i]);
            load(total + at[i].d, u[i]);
        }
        if (c.d_total)
#pragma unroll
            for (int i = 0; i < ITEMS; ++i)
                load(d_total + at[i].d, more[i]);
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                u[i][k] *= rstd;
                sums[i][k] += g[i][k] * u[i][k];
                g[i][k] *= gain[i][k];
                sum += k < at[i].skip ? 0.f : g[i][k] * u[i][k];
            }
        sum = row_sum<WAVES>(sum, lds[turn]) / static_cast<float>(c.dim);
        T* d_x = static_cast<T*>(c.d_x) + row * c.dim;
        S* d_residual = static_cast<S*>(c.d_residual) + row * c.dim;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
#pragma unroll
            for (int k = 0; k < V; ++k)
                g[i][k] = rstd * (g[i][k] - u[i][k] * sum) + more[i][k];
            if (at[i].mine && c.d_x)
                store(d_x + at[i].d, g[i]);
            if (at[i].mine && c.d_residual)
                store(d_residual + at[i].d, g[i]);
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
