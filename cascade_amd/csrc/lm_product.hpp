// C = A B^T of 16-bit operands with 32-bit sums, the tile product under the cross entropy: C[m][n] = sum_k A(m, k) B(n, k), either
// operand with k along its rows in memory or across them, and what becomes of C left to the caller.
//
// A workgroup owns BM x BN of C. Slices of 64 k of both operands go from memory straight into LDS, one slice ahead of the one that
// is multiplied (two buffers, one barrier a slice); 32x32x16 matrix instructions read their operands from there, eight
// values a lane, one step of 16 k ahead. A slice of an operand with k along its rows is [row][64 k], 128 bytes a row, the 16-byte pieces of row r at
// places piece ^ (r / 2 % 8): sixteen lanes that read sixteen rows touch all 256 bytes that LDS serves at a time. With k
// across, it is [64 k][row], and the pieces of line k stand at piece ^ 4 (k % 4), so that the four lines of a transposed read do, too.
// Places past either matrix's end read as zeros and add nothing.
//
// Measured in tiles of 256 x 256 by eight waves (50257 x 8192 x 4096, bfloat16, 32-bit result stored): 1200 TFLOP/s, the library's product 1390, this loop without
// loads 1530; the matrix units are busy 70 to 74 % of the time (60 % in the products for d_hidden) at a clock that stands at 1.64 to 1.84 GHz under them. Slices of
// 32 k in four buffers were 5 % slower, four waves of 128 x 128 each 11 %.
#pragma once
#include "lm_common.hpp"

namespace lm {

constexpr int SLICE = 64; // k per buffer

struct Operand {
    const void* data;
    int64_t stride; // values between rows (k along) or between lines of constant k (k across); a multiple of 8
    int64_t rows;   // extent of m or n
};

// ROWS x 64 k of one operand for one buffer; WAVES waves share the loads.
template <int ROWS, bool ACROSS, int WAVES>
struct Loader {
    static constexpr int LOADS = ROWS / 8 / WAVES; // instructions of a wave per slice
    static_assert(ROWS % (8 * WAVES) == 0, "every wave loads as much");
    static constexpr int PIECES = ACROSS ? ROWS / 8 : 8; // 16-byte pieces of a row or line
    static __device__ int turn(int row) { return !ACROSS ? row >> 1 & 7 : PIECES >= 16 ? (row & 3) * 4 : (row >> 1 & 1) * 4; }

    const char* base;
    int64_t line; // bytes between rows or lines
    int64_t first, rows, k;
    uint32_t offset[LOADS]; // of this lane, from base
    int piece[LOADS];

    __device__ void begin(const Operand& op, int64_t first_row, int64_t k_begin, int64_t k_end, int wave, int lane)
    {
        line = op.stride * 2;
        first = first_row;
        rows = op.rows;
        k = k_end;
        base = static_cast<const char*>(op.data) + (ACROSS ? k_begin * line + first_row * 2 : first_row * line + k_begin * 2);
        for (int j = 0; j < LOADS; ++j) {
            const int at = (wave * LOADS + j) * 64 + lane; // which 16-byte place of the buffer
            const int row = at / PIECES, place = at % PIECES;
            piece[j] = place ^ turn(row);
            offset[j] = static_cast<uint32_t>(row * line + piece[j] * 16);
        }
    }
    // k0: the slice's first k, whose place `base` is at
    __device__ void load(short* buffer, int64_t k0, int wave) const
    {
        int64_t bytes;
        if (ACROSS)
            bytes = (k - k0 < SLICE ? k - k0 : SLICE) * line - first * 2;
        else
            bytes = (rows - first < ROWS ? rows - first : ROWS) * line;
        const buffer_t w = window(base, bytes > 0 ? static_cast<uint32_t>(bytes) : 0);
        int64_t left = ACROSS ? rows - first : k - k0; // values of this slice along the memory's lines
        const int most = static_cast<int>(left < 1024 ? left : 1024);
#pragma unroll
        for (int j = 0; j < LOADS; ++j)
            load_to_lds(w, buffer + (wave * LOADS + j) * 512, piece[j] * 8 >= most ? OUTSIDE : offset[j]);
    }
    __device__ void advance() { base += ACROSS ? SLICE * line : SLICE * 2; }
};

// Fragments of 32 rows x 16 k from a buffer.
template <int ROWS, bool ACROSS, int TILES>
struct Reader {
    typedef Loader<ROWS, ACROSS, 1> Places;
    int at[ACROSS ? 2 * TILES : 4];

    __device__ void begin(int first_row, int lane)
    {
        if (ACROSS) {
            const int g = lane / 16, j = lane % 16;
            for (int u = 0; u < 2; ++u) {
                const int line = (g / 2) * 8 + u * 4 + j / 4;
                for (int t = 0; t < TILES; ++t) {
                    const int col = first_row + t * 32 + (g % 2) * 16 + 4 * (j % 4);
                    at[u * TILES + t] = line * ROWS + ((col / 8) ^ Places::turn(line)) * 8 + col % 8;
                }
            }
        } else {
            const int row = first_row + lane % 32;
            for (int s = 0; s < 4; ++s)
                at[s] = row * SLICE + (((s * 2 + lane / 32) ^ Places::turn(row)) * 8);
        }
    }
    __device__ s16x8 read(const short* buffer, int tile, int step) const
    {
        if (ACROSS)
            return join(read_turned(buffer + at[tile] + step * 16 * ROWS), read_turned(buffer + at[TILES + tile] + step * 16 * ROWS));
        return read16(buffer + at[step] + tile * 32 * SLICE);
    }
};

template <class Type, int BM_, int BN_, int WM_, int WN_, bool A_ACROSS, bool B_ACROSS>
struct Product {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;
    static constexpr int WAVES = WM * WN, THREADS = WAVES * 64;
    static constexpr int TM = BM / WM / 32, TN = BN / WN / 32; // 32x32 tiles of a wave
    typedef f32x16 Sums[TM][TN];

    // The wave's part of C: rows m0 + wave_m() + 32 i + 8 (r / 4) + 4 (lane / 32) + r % 4, columns n0 + wave_n() + 32 j + lane % 32
    // for register r of sums[i][j].
    static __device__ int wave_m() { return static_cast<int>(threadIdx.x / 64 / WN) * (BM / WM); }
    static __device__ int wave_n() { return static_cast<int>(threadIdx.x / 64 % WN) * (BN / WN); }

    struct Fragments {
        s16x8 a[TM], b[TN];
    };
    struct Place {
        Loader<BM, A_ACROSS, WAVES> la;
        Loader<BN, B_ACROSS, WAVES> lb;
        Reader<BM, A_ACROSS, TM> ra;
        Reader<BN, B_ACROSS, TN> rb;
        int wave;
        __device__ void load(short* a, short* b, int64_t k0) const
        {
            la.load(a, k0, wave);
            lb.load(b, k0, wave);
        }
        __device__ void read(const short* a, const short* b, int step, Fragments& f) const
        {
#pragma unroll
            for (int j = 0; j < TN; ++j)
                f.b[j] = rb.read(b, j, step);
#pragma unroll
            for (int i = 0; i < TM; ++i)
                f.a[i] = ra.read(a, i, step);
        }
    };
    static __device__ void multiply(const Fragments& f, Sums& sums)
    {
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j)
                sums[i][j] = Type::mfma32(f.a[i], f.b[j], sums[i][j]);
    }
    // One LDS read behind each of the first matrix instructions of a step, so that the reads of the next step's operands
    // run beside this one's products.
    static __device__ void interleave()
    {
        constexpr int reads = (A_ACROSS ? 2 : 1) * TM + (B_ACROSS ? 2 : 1) * TN, products = TM * TN;
        constexpr int each = (reads + products - 1) / products;
#pragma unroll
        for (int i = 0; i < products; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, each, 0);
        }
    }

    // One slice, its first fragments in f0 already: steps 0 to 2 read one step ahead in `a` and `b`; then the next slice has
    // to be in and everybody done with this one, whose place the slice after the next takes, and step 3 reads the next one's first.
    // Slices past the end are loaded as zeros, from an empty window, so that all slices run the same code.
    static __device__ void slice(Place& p, short* a, short* b, short* a_next, short* b_next, int64_t k0, Fragments& f0, Fragments& f1, Sums& sums)
    {
        p.read(a, b, 1, f1);
        multiply(f0, sums);
        interleave();
        __builtin_amdgcn_sched_barrier(0);
        p.read(a, b, 2, f0);
        multiply(f1, sums);
        interleave();
        __builtin_amdgcn_sched_barrier(0);
        p.read(a, b, 3, f1);
        multiply(f0, sums);
        interleave();
        __builtin_amdgcn_sched_barrier(0);
        wait_for_all();
        meet();
        p.la.advance();
        p.lb.advance();
        p.load(a, b, k0 + 2 * SLICE);
        p.read(a_next, b_next, 0, f0);
        multiply(f1, sums);
        interleave();
        __builtin_amdgcn_sched_barrier(0);
    }

    // sums = A B^T over k in [k_begin, k_end) for the tile at (m0, n0); a0, a1 and b0, b1: LDS for 64 BM and 64 BN values, arrays
    // of their own each, by which the compiler tells a read of one from a load in flight to another.
    static __device__ void run(const Operand& A, const Operand& B, int64_t m0, int64_t n0, int64_t k_begin, int64_t k_end, short* a0, short* a1,
                               short* b0, short* b1, Sums& sums)
    {
        const int lane = threadIdx.x % 64;
        Place p;
        p.wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
        p.la.begin(A, m0, k_begin, k_end, p.wave, lane);
        p.lb.begin(B, n0, k_begin, k_end, p.wave, lane);
        p.ra.begin(wave_m(), lane);
        p.rb.begin(wave_n(), lane);
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j)
                sums[i][j] = f32x16{};
        if (k_begin >= k_end)
            return;
        p.load(a0, b0, k_begin);
        p.la.advance();
        p.lb.advance();
        wait_for_all();
        meet();
        Fragments f0, f1;
        p.load(a1, b1, k_begin + SLICE);
        p.read(a0, b0, 0, f0);
        // Two slices a turn, one from each pair of buffers; an odd number of slices gets one of zeros. (Left in between, the loop
        // would be one whose turns may begin with either pair, and the compiler would wait for every load at its head.)
        for (int64_t k0 = k_begin; k0 < k_end; k0 += 2 * SLICE) {
            slice(p, a0, b0, a1, b1, k0, f0, f1, sums);
            slice(p, a1, b1, a0, b0, k0 + SLICE, f0, f1, sums);
        }
        wait_for_all(); // the last loads have written their zeros
    }

    // LDS for a wave's part of C in 16 bits, from the buffers of the operands.
    static __device__ short* wave_region(short* a0, short* a1, short* b0, short* b1)
    {
        constexpr int SIZE = (BM / WM) * (BN / WN), IN_A = BM * SLICE / SIZE, IN_B = BN * SLICE / SIZE;
        static_assert(2 * IN_A + 2 * IN_B >= WAVES, "the parts fit the buffers");
        const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
        return w < IN_A ? a0 + w * SIZE : w < 2 * IN_A ? a1 + (w - IN_A) * SIZE : w < 2 * IN_A + IN_B ? b0 + (w - 2 * IN_A) * SIZE : b1 + (w - 2 * IN_A - IN_B) * SIZE;
    }

    // out[n * stride + m] = round(value(j, m', x)) for x = C[m][n], where the lane's column is n0 + wave_n() + 32 j + lane % 32 and m' counts from the wave's
    // first row; rows m < rows, columns n < columns. Four neighbouring rows are a lane's own, so the wave turns its part in LDS, 8 bytes in
    // and 16 out a lane, and stores whole lines. `mine`: the wave_region, once all waves are done with what was there.
    // wide: 16-byte stores are allowed (out, stride).
    template <class Type16, class F>
    static __device__ void store_turned(Sums& sums, short* mine, int64_t m0, int64_t n0, int64_t rows, int64_t columns, short* out, int64_t stride, bool wide,
                                        F value)
    {
        constexpr int LINE = BM / WM, PIECES = LINE / 8, COLUMNS = BN / WN; // a line holds a column's rows; its pieces stand at places piece ^ column
        static_assert((PIECES & (PIECES - 1)) == 0 && 64 % PIECES == 0, "whole lines");
        const int lane = threadIdx.x % 64, half = lane / 32;
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const int column = 32 * j + lane % 32;
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    s16x4 y;
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        y[r] = to16<Type16>(value(j, 32 * i + 8 * g + 4 * half + r, sums[i][j][4 * g + r]));
                    *reinterpret_cast<s16x4*>(mine + column * LINE + ((4 * i + g) ^ column % PIECES) * 8 + 4 * half) = y;
                }
        }
        wait_for_lds();
        const int64_t mw = m0 + wave_m(), nw = n0 + wave_n();
        const int piece = lane % PIECES;
        const int64_t m = mw + piece * 8;
#pragma unroll
        for (int c = 0; c < COLUMNS; c += 64 / PIECES) {
            const int column = c + lane / PIECES;
            const s16x8 y = read16(mine + column * LINE + (piece ^ column % PIECES) * 8);
            if (nw + column >= columns || m >= rows)
                continue;
            short* to = out + (nw + column) * stride + m;
            if (wide && m + 8 <= rows) {
                *reinterpret_cast<s16x8*>(to) = y;
            } else {
                for (int r = 0; r < 8; ++r)
                    if (m + r < rows)
                        to[r] = y[r];
            }
        }
    }
};

} // namespace lm
