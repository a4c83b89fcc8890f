// Layer normalisation, forward and backward, and activations whose input is kept in 8 bits for the backward pass.
//
//   mean = sum x / C, var = sum (x - mean)^2 / C, rstd = 1 / sqrt(var + eps), x^ = (x - mean) rstd, y = x^ gamma + beta
//   G = dy gamma, dx = rstd (G - sum G / C - x^ sum (G x^) / C), dgamma = sum over rows of dy x^, dbeta = ... of dy
//
// Everything is bound by memory: a row is read once and stays in registers, a lane holding 8 or 16 of its values, and
// both passes over it (the sum, then the squares about the mean; the largest magnitude, then the codes) run there.
// Statistics and sums are 32 bits.
#include "amsim_rows.h"

#include <algorithm>

namespace amsim {

namespace {

// A row over LANES lanes of EACH values: 16 lanes for short ones (four rows a wavefront), a wavefront, four, eight or sixteen.
template <int LANES_, int EACH_> struct Shape {
    static constexpr int LANES = LANES_, EACH = EACH_, THREADS = LANES_ > 256 ? LANES_ : 256, ROWS = THREADS / LANES_;
    static constexpr int64_t HOLDS = (int64_t)LANES_ * EACH_;
};
constexpr int64_t MOST_HELD = 16384;
// fn(Shape) of the smallest that holds a row; rows beyond that are read again for every pass over them
template <typename Fn> int with_shape(int64_t cols, Fn &&fn)
{
    if (cols <= 128) return fn(Shape<16, 8>{});
    if (cols <= 512) return fn(Shape<64, 8>{});
    if (cols <= 1024) return fn(Shape<64, 16>{});
    if (cols <= 2048) return fn(Shape<256, 8>{});
    if (cols <= 4096) return fn(Shape<256, 16>{});
    if (cols <= 8192) return fn(Shape<512, 16>{});  // (1024 lanes of 8: 8192 x 8192 bf16 77 us, 53 so: two of them share a CU)
    return fn(Shape<1024, 16>{});
}
template <typename Fn> int with_type(int dtype, Fn &&fn)
{
    switch (dtype) {
    case AMSIM_DTYPE_F32: return fn(0.0f);
    case AMSIM_DTYPE_BF16: return fn((__bf16)0.0f);
    default: return fn((_Float16)0.0f);
    }
}

// what a thread has of its row
template <typename S> struct Place {
    int lane, group;  // within the row, the row within the workgroup
    float (*part)[RowLanes<S::LANES>::WAVES][2];
    __device__ __forceinline__ int64_t first_row() const { return (int64_t)blockIdx.x * S::ROWS + group; }
    __device__ __forceinline__ int64_t rows_apart() const { return (int64_t)gridDim.x * S::ROWS; }
    __device__ __forceinline__ RowLanes<S::LANES> lanes() const { return RowLanes<S::LANES>{part}; }
};
#define AMSIM_PLACE(S)                                                        \
    __shared__ float part_[2][RowLanes<S::LANES>::WAVES][2];                  \
    const Place<S> place{(int)threadIdx.x % S::LANES, (int)threadIdx.x / S::LANES, part_}

// ---- layer norm, forward ----------------------------------------------------------------------------------------------
// Moves each value twice, and a byte more where it is kept: 16384 x 4096 bf16 54 us (268 MB, 5.0 TB/s), kept 62 to 66 (335 MB); 256 x
// 512 f32 3.3, the latency of a load, two sums over the lanes and a store.

struct NormArgs {
    const void *x;
    int64_t rows, stride;
    int64_t cols;
    const void *gamma, *beta;  // null: ones, zeros
    int param_dtype;
    float eps;
    void *out;
    float *statistics;         // [rows][2], or null
    uint8_t *codes;            // [rows][pitch], or null
    float *scales;
    bool around;
};

template <typename T, typename S>
__global__ __launch_bounds__(S::THREADS) void norm_kernel(NormArgs g)
{
    constexpr int N = PIECE<T>, PIECES = S::EACH / N;
    AMSIM_PLACE(S);
    RowLanes<S::LANES> lanes = place.lanes();
    const int cols = (int)g.cols, pitch = (int)kept8_pitch(cols);
    float gamma[PIECES][N], beta[PIECES][N];
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        const int c = (p * S::LANES + place.lane) * N;
#pragma unroll
        for (int i = 0; i < N; ++i) gamma[p][i] = 1.0f, beta[p][i] = 0.0f;
        if (g.gamma) load_floats(g.gamma, g.param_dtype, c, cols - c, gamma[p]);
        if (g.beta) load_floats(g.beta, g.param_dtype, c, cols - c, beta[p]);
    }
    v4i raw[PIECES];
    auto load = [&](int64_t row) {
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int c = (p * S::LANES + place.lane) * N;
            raw[p] = load_piece((const T *)g.x + row * g.stride + c, row < g.rows ? cols - c : 0);
        }
    };
    load(place.first_row());
    for (int64_t row = place.first_row(); row < g.rows; row += place.rows_apart()) {
        float v[PIECES][N], sum = 0.0f, squares = 0.0f, largest = 0.0f;
#pragma unroll
        for (int p = 0; p < PIECES; ++p) piece_floats<T>(raw[p], v[p]);
        load(row + place.rows_apart());  // (the next row is under way while this one is worked on)
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                sum += v[p][i];
                largest = MaxOf::of(largest, __uint_as_float(magnitude_bits(v[p][i])));
            }
        }
        if (g.codes) lanes.template both<SumOf, MaxOf>(sum, largest);
        else sum = lanes.template one<SumOf>(sum);
        const float mean = sum / (float)cols;
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int c = (p * S::LANES + place.lane) * N;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float d = c + i < cols ? v[p][i] - mean : 0.0f;
                squares = __builtin_fmaf(d, d, squares);
            }
        }
        squares = lanes.template one<SumOf>(squares);
        const float rstd = 1.0f / sqrtf(squares / (float)cols + g.eps);
        T *out = (T *)g.out + row * cols;
        const float r = q8_multiplier(__float_as_uint(largest));
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int c = (p * S::LANES + place.lane) * N;
            if (g.codes && c < pitch) store_codes(g.codes + row * pitch + c, v[p], r);
#pragma unroll
            for (int i = 0; i < N; ++i) v[p][i] = __builtin_fmaf((v[p][i] - mean) * rstd, gamma[p][i], beta[p][i]);
            store_piece(out + c, cols - c, v[p], g.around);
        }
        if (place.lane == 0) {
            if (g.statistics) g.statistics[2 * row] = mean, g.statistics[2 * row + 1] = rstd;
            if (g.codes) g.scales[row] = q8_scale(__float_as_uint(largest));
        }
    }
}

// rows that no workgroup holds: read for the sum, for the squares, and for the results (2048 x 32768 bf16 101 us, kept 112; as many values in
// rows of 16384 that are held 60)
template <typename T>
__global__ __launch_bounds__(1024) void norm_long_kernel(NormArgs g)
{
    constexpr int N = PIECE<T>;
    using S = Shape<1024, N>;
    AMSIM_PLACE(S);
    RowLanes<S::LANES> lanes = place.lanes();
    const int64_t cols = g.cols, pitch = kept8_pitch(cols);
    for (int64_t row = blockIdx.x; row < g.rows; row += gridDim.x) {
        const T *x = (const T *)g.x + row * g.stride;
        float v[N], sum = 0.0f, squares = 0.0f, largest = 0.0f;
        for (int64_t c = place.lane * N; c < cols; c += 1024 * N) {
            piece_floats<T>(load_piece(x + c, cols - c), v);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                sum += v[i];
                largest = MaxOf::of(largest, __uint_as_float(magnitude_bits(v[i])));
            }
        }
        lanes.template both<SumOf, MaxOf>(sum, largest);
        const float mean = sum / (float)cols;
        for (int64_t c = place.lane * N; c < cols; c += 1024 * N) {
            piece_floats<T>(load_piece(x + c, cols - c), v);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float d = c + i < cols ? v[i] - mean : 0.0f;
                squares = __builtin_fmaf(d, d, squares);
            }
        }
        squares = lanes.template one<SumOf>(squares);
        const float rstd = 1.0f / sqrtf(squares / (float)cols + g.eps), r = q8_multiplier(__float_as_uint(largest));
        for (int64_t c = place.lane * N; c < pitch; c += 1024 * N) {
            float gamma[N], beta[N];
#pragma unroll
            for (int i = 0; i < N; ++i) gamma[i] = 1.0f, beta[i] = 0.0f;
            piece_floats<T>(load_piece(x + c, cols - c), v);
            if (g.codes) store_codes(g.codes + row * pitch + c, v, r);
            if (g.gamma) load_floats(g.gamma, g.param_dtype, c, cols - c, gamma);
            if (g.beta) load_floats(g.beta, g.param_dtype, c, cols - c, beta);
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = __builtin_fmaf((v[i] - mean) * rstd, gamma[i], beta[i]);
            store_piece((T *)g.out + row * cols + c, cols - c, v, g.around);
        }
        if (place.lane == 0) {
            if (g.statistics) g.statistics[2 * row] = mean, g.statistics[2 * row + 1] = rstd;
            if (g.codes) g.scales[row] = q8_scale(__float_as_uint(largest));
        }
    }
}

// ---- layer norm, backward ---------------------------------------------------------------------------------------------

struct NormGradArgs {
    const void *grad;
    int64_t rows, stride, cols;
    const void *x;             // or null: codes and scales
    int64_t x_stride;
    const uint8_t *codes;
    const float *scales, *statistics;
    const void *gamma;
    int param_dtype;
    void *grad_x;              // or null
    float *partial;            // [workgroups][2][cols]: of dgamma and dbeta, or null
    bool around;
};

// x as it was given, or as it was kept
template <typename T, bool KEPT> __device__ __forceinline__ auto load_input(const NormGradArgs &g, int64_t row, int64_t c, int64_t pitch)
{
    if constexpr (KEPT) {
        struct {
            uint32_t w[PIECE<T> / 4];
        } raw = {};
        if (c < pitch) __builtin_memcpy(&raw, __builtin_assume_aligned(g.codes + row * pitch + c, PIECE<T>), PIECE<T>);
        return raw;
    } else {
        return load_piece((const T *)g.x + row * g.x_stride + c, g.cols - c);
    }
}
template <typename T, bool KEPT, typename Raw> __device__ __forceinline__ void input_floats(const Raw &raw, float scale, float (&v)[PIECE<T>])
{
    if constexpr (KEPT) code_values(raw.w, scale, v);
    else piece_floats<T>(raw, v);
}

// dx needs two sums over the row, which meet in one pass over the lanes.  The gradients of gamma and beta: a lane adds up its
// columns over the rows that it sees; a workgroup's go to memory once, and column_sums_kernel adds those in their order.
// 16384 x 4096 bf16 with the sums' launch, 5 to 6 us of it: from x 87 us (403 MB and 25 of sums, 4.9 TB/s), from 8 bits 73 (335 and 25).
template <typename T, typename S, bool KEPT>
__global__ __launch_bounds__(S::THREADS) void norm_grad_kernel(NormGradArgs g)
{
    constexpr int N = PIECE<T>, PIECES = S::EACH / N;
    AMSIM_PLACE(S);
    RowLanes<S::LANES> lanes = place.lanes();
    const int cols = (int)g.cols, pitch = (int)kept8_pitch(cols);
    float gamma[PIECES][N], to_gamma[PIECES][N] = {}, to_beta[PIECES][N] = {};
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        const int c = (p * S::LANES + place.lane) * N;
#pragma unroll
        for (int i = 0; i < N; ++i) gamma[p][i] = 1.0f;
        if (g.gamma) load_floats(g.gamma, g.param_dtype, c, cols - c, gamma[p]);
    }
    v4i raw[PIECES];
    decltype(load_input<T, KEPT>(g, 0, 0, 0)) raw_x[PIECES];
    float next_mean, next_rstd, next_scale;
    auto load = [&](int64_t row) {
        const int64_t at = row < g.rows ? row : 0;
        next_mean = g.statistics[2 * at], next_rstd = g.statistics[2 * at + 1], next_scale = KEPT ? g.scales[at] : 0.0f;
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int c = (p * S::LANES + place.lane) * N;
            raw[p] = load_piece((const T *)g.grad + row * g.stride + c, row < g.rows ? cols - c : 0);
            raw_x[p] = load_input<T, KEPT>(g, at, c, pitch);
        }
    };
    constexpr bool AHEAD = S::LANES * S::EACH < 16384;  // (there are no registers for it in sixteen waves of 16 values)
    if constexpr (AHEAD) load(place.first_row());
    for (int64_t row = place.first_row(); row < g.rows; row += place.rows_apart()) {
        if constexpr (!AHEAD) load(row);
        const float mean = next_mean, rstd = next_rstd;
        float h[PIECES][N], d[PIECES][N], sum = 0.0f, dot = 0.0f;
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            piece_floats<T>(raw[p], d[p]);  // (zeros behind the row's end: nothing is added there)
            input_floats<T, KEPT>(raw_x[p], next_scale, h[p]);
        }
        if constexpr (AHEAD) load(row + place.rows_apart());  // (the next row is under way while this one is worked on)
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                h[p][i] = (h[p][i] - mean) * rstd;
                to_gamma[p][i] = __builtin_fmaf(d[p][i], h[p][i], to_gamma[p][i]);
                to_beta[p][i] += d[p][i];
                d[p][i] *= gamma[p][i];
                sum += d[p][i];
                dot = __builtin_fmaf(d[p][i], h[p][i], dot);
            }
        }
        if (!g.grad_x) continue;
        lanes.template both<SumOf, SumOf>(sum, dot);
        sum /= (float)cols, dot /= (float)cols;
        T *dx = (T *)g.grad_x + row * cols;
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int c = (p * S::LANES + place.lane) * N;
#pragma unroll
            for (int i = 0; i < N; ++i) d[p][i] = rstd * __builtin_fmaf(-dot, h[p][i], d[p][i] - sum);
            store_piece(dx + c, cols - c, d[p], g.around);
        }
    }
    if (!g.partial) return;
    float *out = g.partial + (int64_t)blockIdx.x * 2 * cols;
    if constexpr (S::ROWS == 1) {
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int c = (p * S::LANES + place.lane) * N;
            store_piece(out + c, cols - c < 4 ? cols - c : 4, *(const float (*)[4])&to_gamma[p][0]);
            store_piece(out + cols + c, cols - c < 4 ? cols - c : 4, *(const float (*)[4])&to_beta[p][0]);
            if constexpr (N == 8) {
                store_piece(out + c + 4, cols - c - 4 < 4 ? cols - c - 4 : 4, *(const float (*)[4])&to_gamma[p][4]);
                store_piece(out + cols + c + 4, cols - c - 4 < 4 ? cols - c - 4 : 4, *(const float (*)[4])&to_beta[p][4]);
            }
        }
    } else {  // the workgroup's rows meet in LDS
        __shared__ float sums[2][S::ROWS][S::HOLDS];
#pragma unroll
        for (int p = 0; p < PIECES; ++p)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int c = (p * S::LANES + place.lane) * N + i;
                sums[0][place.group][c] = to_gamma[p][i];
                sums[1][place.group][c] = to_beta[p][i];
            }
        __syncthreads();
        for (int c = threadIdx.x; c < cols; c += S::THREADS)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                float s = sums[k][0][c];
#pragma unroll
                for (int r = 1; r < S::ROWS; ++r) s += sums[k][r][c];
                out[k * cols + c] = s;
            }
    }
}

// rows that no workgroup holds: dx by rows, dgamma and dbeta by columns, a slab of rows to a workgroup (2048 x 32768 bf16 from x 171 us, from 8
// bits 143: gradient and input are read three times; as many values in rows of 16384 from x 90)
template <typename T, bool KEPT>
__global__ __launch_bounds__(1024) void norm_grad_long_kernel(NormGradArgs g)
{
    constexpr int N = PIECE<T>;
    using S = Shape<1024, N>;
    AMSIM_PLACE(S);
    RowLanes<S::LANES> lanes = place.lanes();
    const int64_t cols = g.cols, pitch = kept8_pitch(cols);
    for (int64_t row = blockIdx.x; row < g.rows; row += gridDim.x) {
        const T *dy = (const T *)g.grad + row * g.stride;
        const float mean = g.statistics[2 * row], rstd = g.statistics[2 * row + 1], scale = KEPT ? g.scales[row] : 0.0f;
        float h[N], d[N], gamma[N], sum = 0.0f, dot = 0.0f;
        auto load = [&](int64_t c) {
#pragma unroll
            for (int i = 0; i < N; ++i) gamma[i] = 1.0f;
            piece_floats<T>(load_piece(dy + c, cols - c), d);
            input_floats<T, KEPT>(load_input<T, KEPT>(g, row, c, pitch), scale, h);
            if (g.gamma) load_floats(g.gamma, g.param_dtype, c, cols - c, gamma);
#pragma unroll
            for (int i = 0; i < N; ++i) h[i] = (h[i] - mean) * rstd, d[i] *= gamma[i];
        };
        for (int64_t c = place.lane * N; c < cols; c += 1024 * N) {
            load(c);
#pragma unroll
            for (int i = 0; i < N; ++i) sum += d[i], dot = __builtin_fmaf(d[i], h[i], dot);
        }
        lanes.template both<SumOf, SumOf>(sum, dot);
        sum /= (float)cols, dot /= (float)cols;
        for (int64_t c = place.lane * N; c < cols; c += 1024 * N) {
            load(c);
#pragma unroll
            for (int i = 0; i < N; ++i) d[i] = rstd * __builtin_fmaf(-dot, h[i], d[i] - sum);
            store_piece((T *)g.grad_x + row * cols + c, cols - c, d, g.around);
        }
    }
}
template <typename T, bool KEPT>
__global__ __launch_bounds__(256) void norm_grad_columns_kernel(NormGradArgs g)
{
    constexpr int N = PIECE<T>;
    const int64_t cols = g.cols, pitch = kept8_pitch(cols), c = ((int64_t)blockIdx.x * 256 + threadIdx.x) * N;
    if (c >= cols) return;
    float to_gamma[N] = {}, to_beta[N] = {};
    for (int64_t row = blockIdx.y; row < g.rows; row += gridDim.y) {
        float h[N], d[N];
        const float mean = g.statistics[2 * row], rstd = g.statistics[2 * row + 1], scale = KEPT ? g.scales[row] : 0.0f;
        piece_floats<T>(load_piece((const T *)g.grad + row * g.stride + c, cols - c), d);
        input_floats<T, KEPT>(load_input<T, KEPT>(g, row, c, pitch), scale, h);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            to_gamma[i] = __builtin_fmaf(d[i], (h[i] - mean) * rstd, to_gamma[i]);
            to_beta[i] += d[i];
        }
    }
    float *out = g.partial + (int64_t)blockIdx.y * 2 * cols + c;
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (c + i < cols) out[i] = to_gamma[i], out[cols + i] = to_beta[i];
}

// [parts][2][cols] to the two gradients: 32 columns and 32 runs of parts to a workgroup, the runs joined in pairs
struct ColumnSums {
    const float *partial;
    int64_t parts, cols;
    void *grad[2];
    int dtype;
};
__global__ __launch_bounds__(1024) void column_sums_kernel(ColumnSums g)
{
    __shared__ float run[32][33];
    const int c = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int64_t col = (int64_t)blockIdx.x * 32 + c, width = 2 * g.cols, each = ceil_div64(g.parts, 32), end = min(g.parts, each * (w + 1));
    float s = 0.0f;
    if (col < width) {
#pragma unroll 8
        for (int64_t p = each * w; p < end; ++p) s += g.partial[p * width + col];
    }
    run[w][c] = s;
    for (int half = 16; half; half /= 2) {
        __syncthreads();
        if (w < half) run[w][c] += run[w + half][c];
    }
    if (w != 0 || col >= width) return;
    const int which = col >= g.cols;
    if (g.grad[which]) store_from_float(g.grad[which], g.dtype, col - which * g.cols, run[0][c]);
}

// ---- activations whose input is kept -------------------------------------------------------------------------------------

// Phi(-t) = exp(-t^2 / 2) R(t), t = |x|, and R(t) = 1/2 + w Q(w) in w = t / (1 + t / 4): what the reciprocal and Q are off by
// counts with w, so that next to zero little is left of it.  Q's coefficients: least largest relative error of R on t <= 14.5
// (least squares on the scaled complementary error function, the weights raised where the error was largest, one coefficient
// after the other rounded to 32 bits), 2.1e-8.  Below -13.2, where the gelu is less than 2^-126, it comes out as zero.
// Largest relative errors, of 2^20 values each: on -1 .. 0 3.0e-7, on -4 .. -1 1.1e-6, on -12 .. -4 8.8e-6 (the exponent's
// rounding), above zero 2.0e-7; in elementary 32-bit operations with the language's erfcf 2.8e-7, 1.1e-6, 1.1e-5 and 2.3e-7.
// Some 20 instructions, two of them at a quarter rate: with 16-bit tensors the vector units are about as busy as memory, and
// erfcf takes so many more that they would be the bound of 32-bit ones too.
struct Gelu {
    // R(t) and exp(-t^2 / 2)
    struct Parts {
        float r, e;
        __device__ __forceinline__ explicit Parts(float x)
        {
            const float t = fminf(fabsf(x), 15.0f), w = t * __builtin_amdgcn_rcpf(__builtin_fmaf(0.25f, t, 1.0f));
            float q = -1.278699954809781e-07f;
            q = __builtin_fmaf(q, w, 1.6464955479023047e-06f);
            q = __builtin_fmaf(q, w, -2.7883238544745836e-06f);
            q = __builtin_fmaf(q, w, -5.159039574209601e-05f);
            q = __builtin_fmaf(q, w, 0.00010789257066790015f);
            q = __builtin_fmaf(q, w, 0.003397819586098194f);
            q = __builtin_fmaf(q, w, -0.032908763736486435f);
            q = __builtin_fmaf(q, w, 0.15026246011257172f);
            q = __builtin_fmaf(q, w, -0.3989420533180237f);
            r = __builtin_fmaf(q, w, 0.5f);
            e = __builtin_amdgcn_exp2f(t * t * -0.72134752f);
        }
    };
    static __device__ __forceinline__ float value(float x)
    {
        const Parts p(x);
        const float tail = p.r * p.e;
        return x * (x < 0.0f ? tail : 1.0f - tail);
    }
    // Phi(x) + x phi(x) = 1 + e (|x| / sqrt(2 pi) - R) above zero, 1 less that below
    static __device__ __forceinline__ float slope(float x)
    {
        const Parts p(x);
        const float above = p.e * __builtin_fmaf(0.39894228f, fabsf(x), -p.r);
        return x < 0.0f ? -above : 1.0f + above;
    }
};
// With e = exp(-x) the swish is x / (1 + e), its slope s + x s (1 - s) of s = 1 / (1 + e); 1 - s is e s where s is near one.
// exp2's argument is rounded, which would cost as many last places as x is large: what was lost is put back by the first
// term of its series.  The reciprocal, a last place off by itself, is corrected by its residual.  Beyond 64 the one or the
// other of 1 and e is nothing beside the other, and exp(x) is held 2^64 times as large, or it would be zero from -88 on, where
// the swish itself is so only from -104 on.  In 32 bits the swish is within 2.2e-7 of itself from -87 on; without the
// corrections within 3.9e-6, and in 16 bits 5.9375 went to its farther neighbour.
struct Swish {
    static constexpr float LOG2E = 1.44269502f, LOG2E_REST = 1.92596299e-8f, LN2 = 0.693147182f;
    // exp2(x log2(e) + more)
    static __device__ __forceinline__ float exponential(float x, float more)
    {
        const float a = x * LOG2E, rest = __builtin_fmaf(x, LOG2E_REST, __builtin_fmaf(x, LOG2E, -a)), e = __builtin_amdgcn_exp2f(a + more);
        return __builtin_fmaf(e, rest * LN2, e);
    }
    static __device__ __forceinline__ bool far(float x) { return fabsf(x) > 64.0f; }
    static __device__ __forceinline__ float far_exponential(float x) { return exponential(fmaxf(x, -200.0f), 64.0f); }  // (2^64 exp(x))
    static __device__ __forceinline__ float value(float x)
    {
        if (far(x)) return x > 0.0f ? x : x * far_exponential(x) * 0x1p-64f;
        const float d = 1.0f + exponential(-x, 0.0f), r = __builtin_amdgcn_rcpf(d), q = x * r;
        return __builtin_fmaf(__builtin_fmaf(-d, q, x), r, q);
    }
    static __device__ __forceinline__ float slope(float x)
    {
        if (far(x)) return x > 0.0f ? 1.0f : (1.0f + x) * far_exponential(x) * 0x1p-64f;
        const float e = exponential(-x, 0.0f), d = 1.0f + e, r = __builtin_amdgcn_rcpf(d), s = __builtin_fmaf(__builtin_fmaf(-d, r, 1.0f), r, r);
        return __builtin_fmaf(x * s, x < 1.0f ? 1.0f - s : e * s, s);
    }
};
struct Linear {  // (nothing but the keeping)
    static __device__ __forceinline__ float value(float x) { return x; }
    static __device__ __forceinline__ float slope(float) { return 1.0f; }
};

// A row's values stay as they came between the search for the largest, the codes and the function.  16384 x 4096 bf16 gelu 61 to 64 us
// (335 MB, 5.2 to 5.5 TB/s) beside 34 vector instructions for 64 values, of two cycles each, or four with a literal: most of the
// SIMDs' time; swish 58.  8192 x 2048 f32 27 (151 MB, 5.5 TB/s), the vector units at most half of it.  Rows past 16384 are read
// twice: 2048 x 32768 bf16 88.
struct ActArgs {
    const void *x;
    int64_t rows, stride, cols;
    void *out;       // or null
    uint8_t *codes;  // or null
    float *scales;
    bool around;
};

template <typename T, typename S, typename F>
__global__ __launch_bounds__(S::THREADS) void activation_kernel(ActArgs g)
{
    constexpr int N = PIECE<T>, PIECES = S::EACH / N;
    AMSIM_PLACE(S);
    RowLanes<S::LANES> lanes = place.lanes();
    const int cols = (int)g.cols, pitch = (int)kept8_pitch(cols);
    for (int64_t row = place.first_row(); row < g.rows; row += place.rows_apart()) {
        v4i raw[PIECES];
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int c = (p * S::LANES + place.lane) * N;
            raw[p] = load_piece((const T *)g.x + row * g.stride + c, cols - c);
        }
        if (g.codes) {
            float largest = 0.0f;
#pragma unroll
            for (int p = 0; p < PIECES; ++p) {
                float v[N];
                piece_floats<T>(raw[p], v);
#pragma unroll
                for (int i = 0; i < N; ++i) largest = MaxOf::of(largest, __uint_as_float(magnitude_bits(v[i])));
            }
            largest = lanes.template one<MaxOf>(largest);
            const float r = q8_multiplier(__float_as_uint(largest));
#pragma unroll
            for (int p = 0; p < PIECES; ++p) {
                const int c = (p * S::LANES + place.lane) * N;
                float v[N];
                piece_floats<T>(raw[p], v);
                if (c < pitch) store_codes(g.codes + row * pitch + c, v, r);
            }
            if (place.lane == 0) g.scales[row] = q8_scale(__float_as_uint(largest));
        }
        if (!g.out) continue;
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int c = (p * S::LANES + place.lane) * N;
            float v[N];
            piece_floats<T>(raw[p], v);
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = F::value(v[i]);
            store_piece((T *)g.out + row * cols + c, cols - c, v, g.around);
        }
    }
}
template <typename T, typename F>
__global__ __launch_bounds__(1024) void activation_long_kernel(ActArgs g)
{
    constexpr int N = PIECE<T>;
    using S = Shape<1024, N>;
    AMSIM_PLACE(S);
    RowLanes<S::LANES> lanes = place.lanes();
    const int64_t cols = g.cols, pitch = kept8_pitch(cols);
    for (int64_t row = blockIdx.x; row < g.rows; row += gridDim.x) {
        const T *x = (const T *)g.x + row * g.stride;
        float v[N], largest = 0.0f;
        if (g.codes) {
            for (int64_t c = place.lane * N; c < cols; c += 1024 * N) {
                piece_floats<T>(load_piece(x + c, cols - c), v);
#pragma unroll
                for (int i = 0; i < N; ++i) largest = MaxOf::of(largest, __uint_as_float(magnitude_bits(v[i])));
            }
            largest = lanes.template one<MaxOf>(largest);
        }
        const float r = q8_multiplier(__float_as_uint(largest));
        for (int64_t c = place.lane * N; c < pitch; c += 1024 * N) {
            piece_floats<T>(load_piece(x + c, cols - c), v);
            if (g.codes) store_codes(g.codes + row * pitch + c, v, r);
            if (!g.out) continue;
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = F::value(v[i]);
            store_piece((T *)g.out + row * cols + c, cols - c, v, g.around);
        }
        if (g.codes && place.lane == 0) g.scales[row] = q8_scale(__float_as_uint(largest));
    }
}

// dx = dy f'(what was kept); without dy: what was kept.  16384 x 4096 bf16 gelu 64 us (335 MB), 33 instructions a value; it took 69 where
// the slope had one more.  8192 x 2048 f32 29, bound by memory (151 MB, 5.2 TB/s).
struct ActGradArgs {
    const void *grad;  // or null
    int64_t rows, stride, cols;
    const uint8_t *codes;
    const float *scales;
    void *grad_x;
    bool around;
};
template <typename T, typename F, int LANES>
__global__ __launch_bounds__(256) void activation_grad_kernel(ActGradArgs g)
{
    constexpr int N = PIECE<T>;
    const int64_t cols = g.cols, pitch = kept8_pitch(cols);
    for (int64_t row = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES; row < g.rows; row += (int64_t)gridDim.x * (256 / LANES)) {
        const T *dy = g.grad ? (const T *)g.grad + row * g.stride : nullptr;
        const float scale = g.scales[row];
#pragma unroll 4
        for (int64_t c = (int64_t)(threadIdx.x % LANES) * N; c < cols; c += LANES * N) {
            uint32_t w[N / 4];
            float v[N], d[N];
            __builtin_memcpy(w, __builtin_assume_aligned(g.codes + row * pitch + c, N), N);
            code_values(w, scale, v);
            if (dy) {
                piece_floats<T>(load_piece(dy + c, cols - c), d);
#pragma unroll
                for (int i = 0; i < N; ++i) v[i] = d[i] * F::slope(v[i]);
            }
            store_piece((T *)g.grad_x + row * cols + c, cols - c, v, g.around);
        }
    }
}

// ---- launches ---------------------------------------------------------------------------------------------------------------

// Workgroups of a normalisation, which go over the rows in turn with gamma and beta in registers: as many as the card holds at
// once, so that none waits for a second round (16384 x 2048 bf16: 31 us with 1792, 34 with 1024; 8192 x 8192: 53 with 512, 59 with 1024),
// but two rounds of them where four waves hold a row of 16 values a lane (16384 x 4096 bf16, forward and backward: 131 us with 2048, 138
// with 1024; 8192 x 4096 75 and 74).  An activation's rows, which have nothing in common, are a workgroup each (16384 x 4096 bf16: 58
// us, 69 by 2048 workgroups).
template <typename S> unsigned workgroups(int64_t rows)
{
    const int to_a_cu = S::LANES > 256 ? 1024 / S::LANES : S::EACH == 8 ? 7 : S::LANES == 64 ? 4 : 8;
    return (unsigned)std::min<int64_t>(ceil_div64(rows, S::ROWS), 256 * to_a_cu);
}
unsigned long_workgroups(int64_t rows) { return (unsigned)std::min<int64_t>(rows, 512); }
// ... of the backward pass, each of which leaves 2 x cols sums to be added up: as many as the card holds, from 1024 rows (or groups of
// rows) on at least four to each, below that up to 256 workgroups, of one row each up to 256 rows (65536 x 512 bf16: 45 us with 1280,
// 57 with 512; 16384 x 4096 bf16: 72 with 768, 89 with 1024; 8192 x 512 f32: 13.8 with 512, 15.3 with 1280).  Few wide rows so write
// more sums than they have values: 256 x 16384 bf16 21 us, 34 MB of sums written and read beside 25 MB of tensors; 512 x 16384 25, 256 x 8192
// 13, 512 x 8192 15, 1024 x 8192 19.
constexpr int64_t GRAD_SLABS = 64;
int64_t grad_parts(int64_t rows, int64_t cols)
{
    if (cols > MOST_HELD) return std::min(rows, GRAD_SLABS);
    int64_t parts = 0;
    with_shape(cols, [&](auto shape) {
        using S = decltype(shape);
        const int64_t groups = ceil_div64(rows, S::ROWS), held = 256 * (S::LANES > 256 ? 1 : S::EACH == 8 ? 5 : 3);
        parts = std::min({groups, held, std::max<int64_t>(256, groups / 4)});
        return 0;
    });
    return parts;
}

template <typename T, bool KEPT> int launch_norm_grad(const NormGradArgs &g, hipStream_t stream)
{
    if (g.cols > MOST_HELD) {
        if (g.grad_x) norm_grad_long_kernel<T, KEPT><<<long_workgroups(g.rows), 1024, 0, stream>>>(g);
        if (g.partial)
            norm_grad_columns_kernel<T, KEPT><<<dim3((unsigned)ceil_div64(g.cols, 256 * PIECE<T>), (unsigned)grad_parts(g.rows, g.cols)), 256, 0, stream>>>(g);
    } else {
        with_shape(g.cols, [&](auto shape) {
            using S = decltype(shape);
            norm_grad_kernel<T, S, KEPT><<<(unsigned)grad_parts(g.rows, g.cols), S::THREADS, 0, stream>>>(g);
            return 0;
        });
    }
    AMSIM_HIP_CHECK(hipGetLastError());
    return AMSIM_OK;
}

template <typename F> int launch_activation(const ActArgs &g, int dtype, hipStream_t stream)
{
    return with_type(dtype, [&](auto zero) {
        using T = decltype(zero);
        if (g.cols > MOST_HELD) {
            activation_long_kernel<T, F><<<long_workgroups(g.rows), 1024, 0, stream>>>(g);
        } else {
            with_shape(g.cols, [&](auto shape) {
                using S = decltype(shape);
                activation_kernel<T, S, F><<<(unsigned)std::min<int64_t>(ceil_div64(g.rows, S::ROWS), 1 << 20), S::THREADS, 0, stream>>>(g);
                return 0;
            });
        }
        AMSIM_HIP_CHECK(hipGetLastError());
        return (int)AMSIM_OK;
    });
}
template <typename F> int launch_activation_grad(const ActGradArgs &g, int dtype, hipStream_t stream)
{
    return with_type(dtype, [&](auto zero) {
        using T = decltype(zero);
        const int64_t pieces = ceil_div64(g.cols, PIECE<T>);
        const int lanes = pieces <= 16 ? 16 : pieces <= 64 ? 64 : 256;
        const unsigned blocks = (unsigned)std::min<int64_t>(ceil_div64(g.rows, 256 / lanes), 1 << 20);
        const auto kernel = lanes == 16 ? activation_grad_kernel<T, F, 16> : lanes == 64 ? activation_grad_kernel<T, F, 64> : activation_grad_kernel<T, F, 256>;
        kernel<<<blocks, 256, 0, stream>>>(g);
        AMSIM_HIP_CHECK(hipGetLastError());
        return (int)AMSIM_OK;
    });
}

int check_rows(const char *what, const void *x, int dtype, int64_t rows, int64_t cols, int64_t stride)
{
    const std::string w(what);
    if (!known_dtype(dtype)) return fail(AMSIM_ERR_INVALID, w + ": unknown element type");
    if (!mx_extents_fit(rows, cols)) return fail(AMSIM_ERR_UNSUPPORTED, w + ": extents out of range");
    if (rows == 0 || cols == 0) return fail(AMSIM_ERR_INVALID, w + ": empty tensor");
    if (!x) return fail(AMSIM_ERR_INVALID, w + ": null pointer");
    if (stride < cols && rows > 1) return fail(AMSIM_ERR_INVALID, w + ": rows overlap");
    if ((uintptr_t)x & (element_bytes(dtype) - 1)) return fail(AMSIM_ERR_INVALID, w + ": misaligned pointer");
    return AMSIM_OK;
}
bool around(int64_t rows, int64_t cols, int dtype) { return mx_goes_around((double)rows * (double)cols * element_bytes(dtype)); }
bool off(const void *p, uintptr_t bytes) { return (uintptr_t)p & (bytes - 1); }
uint8_t *codes_of(void *kept) { return (uint8_t *)kept; }
float *scales_of(void *kept, int64_t rows, int64_t cols) { return kept ? (float *)((uint8_t *)kept + rows * kept8_pitch(cols)) : nullptr; }

}  // namespace

}  // namespace amsim

using namespace amsim;

extern "C" {

size_t amsim_kept8_workspace_bytes(int64_t rows, int64_t cols)
{
    return mx_extents_fit(rows, cols) && rows && cols ? (size_t)kept8_bytes(rows, cols) : 0;
}

int amsim_kept8_values(const void *kept, int64_t rows, int64_t cols, int dtype, void *out, void *stream)
{
    if (int rc = check_rows("kept8", out, dtype, rows, cols, cols)) return rc;
    if (!kept) return fail(AMSIM_ERR_INVALID, "kept8: null pointer");
    if (off(kept, 16)) return fail(AMSIM_ERR_INVALID, "kept8: misaligned pointer");
    return launch_activation_grad<Linear>({nullptr, rows, cols, cols, codes_of((void *)kept), scales_of((void *)kept, rows, cols), out, around(rows, cols, dtype)}, dtype, (hipStream_t)stream);
}

int amsim_layer_norm(const void *x, int dtype, int64_t rows, int64_t cols, int64_t row_stride, const void *gamma, const void *beta, int param_dtype,
                     float epsilon, void *out, float *statistics, void *kept, void *stream)
{
    if (int rc = check_rows("layer_norm", x, dtype, rows, cols, row_stride)) return rc;
    if ((gamma || beta) && !known_dtype(param_dtype)) return fail(AMSIM_ERR_INVALID, "layer_norm: unknown element type");
    if (!out) return fail(AMSIM_ERR_INVALID, "layer_norm: null pointer");
    if (!(epsilon >= 0)) return fail(AMSIM_ERR_INVALID, "layer_norm: epsilon must not be negative");
    const uintptr_t element = element_bytes(dtype), param = element_bytes(param_dtype);
    if (off(out, element) || off(statistics, 4) || off(kept, 16) || (gamma && off(gamma, param)) || (beta && off(beta, param)))
        return fail(AMSIM_ERR_INVALID, "layer_norm: misaligned pointer");
    const NormArgs g{x, rows, row_stride, cols, gamma, beta, param_dtype, epsilon, out, statistics, codes_of(kept), scales_of(kept, rows, cols), around(rows, cols, dtype)};
    return with_type(dtype, [&](auto zero) {
        using T = decltype(zero);
        if (cols > MOST_HELD) {
            norm_long_kernel<T><<<long_workgroups(rows), 1024, 0, (hipStream_t)stream>>>(g);
        } else {
            with_shape(cols, [&](auto shape) {
                using S = decltype(shape);
                norm_kernel<T, S><<<workgroups<S>(rows), S::THREADS, 0, (hipStream_t)stream>>>(g);
                return 0;
            });
        }
        AMSIM_HIP_CHECK(hipGetLastError());
        return (int)AMSIM_OK;
    });
}

size_t amsim_layer_norm_grad_workspace_bytes(int64_t rows, int64_t cols)
{
    return mx_extents_fit(rows, cols) && rows && cols ? (size_t)grad_parts(rows, cols) * 2 * cols * 4 : 0;
}

int amsim_layer_norm_grad(const void *grad, int dtype, int64_t rows, int64_t cols, int64_t row_stride, const void *x, int64_t x_row_stride,
                          const void *kept, const float *statistics, const void *gamma, int param_dtype, void *grad_x, void *grad_gamma,
                          void *grad_beta, void *workspace, size_t workspace_bytes, void *stream)
{
    if (int rc = check_rows("layer_norm", grad, dtype, rows, cols, row_stride)) return rc;
    if (!x == !kept) return fail(AMSIM_ERR_INVALID, "layer_norm: either x or what was kept of it is needed");
    if (x)
        if (int rc = check_rows("layer_norm", x, dtype, rows, cols, x_row_stride)) return rc;
    if ((gamma || grad_gamma || grad_beta) && !known_dtype(param_dtype)) return fail(AMSIM_ERR_INVALID, "layer_norm: unknown element type");
    if (!statistics) return fail(AMSIM_ERR_INVALID, "layer_norm: null pointer");
    const uintptr_t element = element_bytes(dtype), param = element_bytes(param_dtype);
    if (off(kept, 16) || off(statistics, 4) || off(grad_x, element) || (gamma && off(gamma, param)) || (grad_gamma && off(grad_gamma, param))
        || (grad_beta && off(grad_beta, param)))
        return fail(AMSIM_ERR_INVALID, "layer_norm: misaligned pointer");
    const bool sums = grad_gamma || grad_beta;
    if (sums && cols >= 1 << 25) return fail(AMSIM_ERR_UNSUPPORTED, "layer_norm: more columns than one launch sums");
    if (sums && (!workspace || workspace_bytes < amsim_layer_norm_grad_workspace_bytes(rows, cols) || off(workspace, 256)))
        return fail(AMSIM_ERR_WORKSPACE, "layer_norm: workspace missing, misaligned or too small");
    if (!grad_x && !sums) return AMSIM_OK;
    const NormGradArgs g{grad, rows, row_stride, cols, x, x_row_stride, codes_of((void *)kept), scales_of((void *)kept, rows, cols), statistics, gamma,
                         param_dtype, grad_x, sums ? (float *)workspace : nullptr, around(rows, cols, dtype)};
    const int rc = with_type(dtype, [&](auto zero) {
        using T = decltype(zero);
        return kept ? launch_norm_grad<T, true>(g, (hipStream_t)stream) : launch_norm_grad<T, false>(g, (hipStream_t)stream);
    });
    if (rc || !sums) return rc;
    column_sums_kernel<<<(unsigned)ceil_div64(2 * cols, 32), 1024, 0, (hipStream_t)stream>>>(
        ColumnSums{(const float *)workspace, grad_parts(rows, cols), cols, {grad_gamma, grad_beta}, param_dtype});
    AMSIM_HIP_CHECK(hipGetLastError());
    return AMSIM_OK;
}

int amsim_activation(const void *x, int dtype, int64_t rows, int64_t cols, int64_t row_stride, int kind, void *out, void *kept, void *stream)
{
    if (int rc = check_rows("activation", x, dtype, rows, cols, row_stride)) return rc;
    if (!out && !kept) return fail(AMSIM_ERR_INVALID, "activation: null pointer");
    if (off(out, element_bytes(dtype)) || off(kept, 16)) return fail(AMSIM_ERR_INVALID, "activation: misaligned pointer");
    const ActArgs g{x, rows, row_stride, cols, out, codes_of(kept), scales_of(kept, rows, cols), around(rows, cols, dtype)};
    switch (kind) {
    case AMSIM_ACT_NONE: return launch_activation<Linear>(g, dtype, (hipStream_t)stream);
    case AMSIM_ACT_GELU: return launch_activation<Gelu>(g, dtype, (hipStream_t)stream);
    case AMSIM_ACT_SWISH: return launch_activation<Swish>(g, dtype, (hipStream_t)stream);
    default: return fail(AMSIM_ERR_INVALID, "activation: unknown activation");
    }
}

int amsim_activation_grad(const void *grad, int dtype, int64_t rows, int64_t cols, int64_t row_stride, const void *kept, int kind, void *grad_x, void *stream)
{
    if (int rc = check_rows("activation", grad, dtype, rows, cols, row_stride)) return rc;
    if (!kept || !grad_x) return fail(AMSIM_ERR_INVALID, "activation: null pointer");
    if (off(kept, 16) || off(grad_x, element_bytes(dtype))) return fail(AMSIM_ERR_INVALID, "activation: misaligned pointer");
    const ActGradArgs g{grad, rows, row_stride, cols, codes_of((void *)kept), scales_of((void *)kept, rows, cols), grad_x, around(rows, cols, dtype)};
    switch (kind) {
    case AMSIM_ACT_GELU: return launch_activation_grad<Gelu>(g, dtype, (hipStream_t)stream);
    case AMSIM_ACT_SWISH: return launch_activation_grad<Swish>(g, dtype, (hipStream_t)stream);
    default: return fail(AMSIM_ERR_INVALID, "activation: unknown activation");
    }
}

}  // extern "C"
