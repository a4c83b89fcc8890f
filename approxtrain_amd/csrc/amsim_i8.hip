// Conversions to 8-bit integers with a scale for each row or column (amsim_i8.h), and back.
//
// Bound by memory, and below some hundred thousand values by the launches: a scale has to be known before the first code is
// written.  Along rows one workgroup sees 16 rows whole and holds them in registers between the two; along columns the
// largest magnitudes are gathered first (by the conversion along rows, where there is one of the same tensor), and the
// tensor is read again.
//
// A wavefront's unit is 16 rows x 64 columns, a step of one fragment: loads of 16 bytes a lane, whole lines of 128 bytes and
// more; codes of rows go out as 1 KB in a piece.  For an operand of the columns the unit's bytes are transposed in
// a wavefront's own corner of LDS, four by four in registers.
#include "amsim_i8.h"

#include <algorithm>

namespace amsim {

namespace {

constexpr int WAVES = 8, WG = 64 * WAVES;

template <typename T> struct Unit {
    static constexpr int N = PIECE<T>;          // values of a lane's piece, and rows that a load covers
    static constexpr int LANES = 64 / N;        // lanes to a row
    static constexpr int LOADS = 16 / N;
};
__device__ __forceinline__ int lane_id() { return threadIdx.x & 63; }
template <typename T> __device__ __forceinline__ int unit_row(int i) { return i * Unit<T>::N + lane_id() / Unit<T>::LANES; }
template <typename T> __device__ __forceinline__ int unit_col() { return lane_id() % Unit<T>::LANES * Unit<T>::N; }

// rows row0 .. row0 + 15, columns col0 .. col0 + 63, zeros outside; `positive` applied
template <typename T>
__device__ __forceinline__ void load_unit(const T *x, const T *positive, int64_t rows, int64_t cols, int64_t stride, int64_t row0, int64_t col0,
                                          v4i (&raw)[Unit<T>::LOADS])
{
    using U = Unit<T>;
    const int64_t c = col0 + unit_col<T>();
    v4i keep[U::LOADS];
#pragma unroll
    for (int i = 0; i < U::LOADS; ++i) {
        const int64_t r = row0 + unit_row<T>(i);
        raw[i] = load_piece(x + r * stride + c, r < rows ? cols - c : 0);
        if (positive) keep[i] = load_piece(positive + r * cols + c, r < rows ? cols - c : 0);
    }
    if (!positive) return;
#pragma unroll
    for (int i = 0; i < U::LOADS; ++i) {
        T v[U::N], y[U::N];
        __builtin_memcpy(v, &raw[i], 16);
        __builtin_memcpy(y, &keep[i], 16);
#pragma unroll
        for (int e = 0; e < U::N; ++e) v[e] = to_float(y[e]) > 0.0f ? v[e] : (T)0.0f;
        __builtin_memcpy(&raw[i], v, 16);
    }
}

// The codes of a unit, PIECE bytes for each load, to the operands that are wanted.  `corner`: 320 dwords of LDS for this
// wavefront alone.
constexpr int CORNER = 320;
template <int N> struct Codes {
    uint32_t w[16 / N][N / 4];
};
template <typename T>
__device__ __forceinline__ void store_unit(const Codes<Unit<T>::N> &codes, uint32_t *corner, int64_t rows, int64_t cols, int64_t row0, int64_t col0,
                                           uint8_t *by_rows, uint8_t *by_columns)
{
    using U = Unit<T>;
    const int lane = lane_id(), c = unit_col<T>();
    if (by_rows) {
        uint8_t *to = by_rows + (row0 / 16 * i8_steps(cols) + col0 / 64) * 1024;
#pragma unroll
        for (int i = 0; i < U::LOADS; ++i)
            __builtin_memcpy(__builtin_assume_aligned(to + (c / 16 * 16 + unit_row<T>(i)) * 16 + c % 16, U::N), codes.w[i], U::N);
    }
    if (!by_columns) return;
    // rows 20 dwords apart: the 64 lanes' reads below meet every bank twice, which is the least
#pragma unroll
    for (int i = 0; i < U::LOADS; ++i)
#pragma unroll
        for (int d = 0; d < U::N / 4; ++d) corner[unit_row<T>(i) * 20 + c / 4 + d] = codes.w[i][d];
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    const int quad = lane / 4, high = lane % 4;  // four columns, four rows
    uint32_t in[4], out[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) in[i] = corner[(4 * high + i) * 20 + quad];
    const uint32_t a = __builtin_amdgcn_perm(in[1], in[0], 0x05010400u), b = __builtin_amdgcn_perm(in[3], in[2], 0x05010400u);
    const uint32_t e = __builtin_amdgcn_perm(in[1], in[0], 0x07030602u), f = __builtin_amdgcn_perm(in[3], in[2], 0x07030602u);
    out[0] = __builtin_amdgcn_perm(b, a, 0x05040100u), out[1] = __builtin_amdgcn_perm(b, a, 0x07060302u);
    out[2] = __builtin_amdgcn_perm(f, e, 0x05040100u), out[3] = __builtin_amdgcn_perm(f, e, 0x07060302u);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < 4; ++i) corner[quad * 20 + 4 * i + high] = out[i];
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    const v4i column = *(const v4i *)&corner[quad * 20 + 4 * high];
    const int64_t col = col0 + lane, steps = i8_steps(rows);
    if (col < ceil_div64(cols, 16) * 16) {
        uint8_t *to = by_columns + (col / 16 * steps + row0 / 64) * 1024 + col % 16 * 16;
        *(v4i *)(to + row0 % 64 / 16 * 256) = column;
        if (row0 + 16 >= rows)  // (what is left of the last step)
            for (int64_t r = row0 % 64 / 16 + 1; r < 4; ++r) *(v4i *)(to + r * 256) = v4i{0, 0, 0, 0};
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
}

// ---- along rows -----------------------------------------------------------------------------------------------------

// maxima or sums over the lanes that hold the same columns of a unit, in every one of them
template <typename Op, typename T> __device__ __forceinline__ float down_unit(float v)
{
    if constexpr (Unit<T>::LANES == 8) v = with_dpp<Op, 0x128>(v);  // the other eight of sixteen
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = Op::of(__uint_as_float(r[0]), __uint_as_float(r[1]));
    const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return Op::of(__uint_as_float(h[0]), __uint_as_float(h[1]));
}

// HELD units of a wave stay in registers; 0: rows are read again.
template <typename T, int HELD>
__global__ __launch_bounds__(WG) void rows_kernel(I8Rows g)
{
    using U = Unit<T>;
    __shared__ uint32_t largest_of[WAVES][16];
    __shared__ __attribute__((aligned(16))) uint32_t corners[WAVES][CORNER];
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row0 = (int64_t)blockIdx.x * 16, units = i8_steps(g.cols);
    const T *x = (const T *)g.x, *positive = (const T *)g.positive;
    v4i held[HELD ? HELD : 1][U::LOADS];
    uint32_t largest[U::LOADS] = {};
    float factor[U::LOADS];
#pragma unroll
    for (int i = 0; i < U::LOADS; ++i) {
        const int64_t r = row0 + unit_row<T>(i);
        factor[i] = g.row_factor && r < g.rows ? g.row_factor[r] : 1.0f;
    }
    // what the unit's values are as codes are made of them
    auto floats = [&](const v4i &raw, int64_t col0, float (&v)[U::N]) {
        piece_floats<T>(raw, v);
        if (g.col_factor) {
            float f[U::N];
            const int64_t c = col0 + unit_col<T>();
            load_floats(g.col_factor, AMSIM_DTYPE_F32, c, g.cols - c, f);
#pragma unroll
            for (int e = 0; e < U::N; ++e) v[e] *= f[e];
        }
    };
    auto look = [&](const v4i (&raw)[U::LOADS], int64_t col0) {
#pragma unroll
        for (int i = 0; i < U::LOADS; ++i) {
            float v[U::N];
            floats(raw[i], col0, v);
#pragma unroll
            for (int e = 0; e < U::N; ++e) largest[i] = max(largest[i], magnitude_bits(v[e]));
        }
        if (!g.partial) return;
        float most[U::N] = {}, sum[U::N] = {};
#pragma unroll
        for (int i = 0; i < U::LOADS; ++i) {
            float v[U::N];
            piece_floats<T>(raw[i], v);
#pragma unroll
            for (int e = 0; e < U::N; ++e) {
                sum[e] += v[e];
                most[e] = MaxOf::of(most[e], __uint_as_float(magnitude_bits(v[e] * factor[i])));
            }
        }
#pragma unroll
        for (int e = 0; e < U::N; ++e) most[e] = down_unit<MaxOf, T>(most[e]), sum[e] = down_unit<SumOf, T>(sum[e]);
        if (lane >= U::LANES) return;
        float *to = g.partial + (int64_t)blockIdx.x * 2 * g.cols;
        const int64_t c = col0 + unit_col<T>();
#pragma unroll
        for (int e = 0; e < U::N; ++e)
            if (c + e < g.cols) to[c + e] = most[e], to[g.cols + c + e] = sum[e];
    };
    if constexpr (HELD > 0) {
#pragma unroll
        for (int h = 0; h < HELD; ++h) load_unit(x, positive, g.rows, g.cols, g.row_stride, row0, (wave + h * WAVES) * 64, held[h]);
#pragma unroll
        for (int h = 0; h < HELD; ++h)
            if (wave + h * WAVES < units) look(held[h], (wave + h * WAVES) * 64);
    } else {
        for (int64_t u = wave; u < units; u += 2 * WAVES) {
            v4i two[2][U::LOADS];
            load_unit(x, positive, g.rows, g.cols, g.row_stride, row0, u * 64, two[0]);
            load_unit(x, positive, g.rows, g.cols, g.row_stride, row0, (u + WAVES) * 64, two[1]);
            look(two[0], u * 64);
            if (u + WAVES < units) look(two[1], (u + WAVES) * 64);
        }
    }
    if (!g.by_rows && !g.by_columns) return;
#pragma unroll
    for (int i = 0; i < U::LOADS; ++i) {
        float m = __uint_as_float(largest[i]);
        m = with_dpp<MaxOf, 0xb1>(m);
        m = with_dpp<MaxOf, 0x4e>(m);
        m = with_dpp<MaxOf, 0x141>(m);
        if constexpr (U::LANES == 16) m = with_dpp<MaxOf, 0x140>(m);
        if (lane % U::LANES == 0) largest_of[wave][unit_row<T>(i)] = __float_as_uint(m);
    }
    __syncthreads();
    float multiplier[U::LOADS];
#pragma unroll
    for (int i = 0; i < U::LOADS; ++i) {
        uint32_t m = 0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) m = max(m, largest_of[w][unit_row<T>(i)]);
        multiplier[i] = q8_multiplier(m);
        const int64_t r = row0 + unit_row<T>(i);
        if (wave == 0 && lane % U::LANES == 0 && r < g.rows) g.scales[r] = q8_scale(m);
    }
    auto encode = [&](const v4i (&raw)[U::LOADS], int64_t col0) {
        Codes<U::N> codes;
#pragma unroll
        for (int i = 0; i < U::LOADS; ++i) {
            float v[U::N];
            floats(raw[i], col0, v);
#pragma unroll
            for (int d = 0; d < U::N / 4; ++d) codes.w[i][d] = q8_codes4(v[4 * d], v[4 * d + 1], v[4 * d + 2], v[4 * d + 3], multiplier[i]);
        }
        store_unit<T>(codes, corners[wave], g.rows, g.cols, row0, col0, g.by_rows, g.by_columns);
    };
    if constexpr (HELD > 0) {
#pragma unroll
        for (int h = 0; h < HELD; ++h)
            if (wave + h * WAVES < units) encode(held[h], (wave + h * WAVES) * 64);
    } else {
        for (int64_t u = wave; u < units; u += 2 * WAVES) {
            v4i two[2][U::LOADS];
            load_unit(x, positive, g.rows, g.cols, g.row_stride, row0, u * 64, two[0]);
            load_unit(x, positive, g.rows, g.cols, g.row_stride, row0, (u + WAVES) * 64, two[1]);
            encode(two[0], u * 64);
            if (u + WAVES < units) encode(two[1], (u + WAVES) * 64);
        }
    }
}

// ---- along columns --------------------------------------------------------------------------------------------------

// the largest magnitudes (and sums) of a slab of rows: [slabs][2][cols]
struct Look {
    const void *x, *positive;
    int64_t rows, cols, stride;
    const float *row_factor;
    int64_t slab;
    float *partial;
};
template <typename T>
__global__ __launch_bounds__(256) void columns_look_kernel(Look g)
{
    constexpr int N = PIECE<T>, AHEAD = 4;
    __shared__ float most_of[4][64 * N], sum_of[4][64 * N];
    const int lane = lane_id(), wave = threadIdx.x >> 6;
    const int64_t c = (int64_t)blockIdx.x * 64 * N + lane * N, from = (int64_t)blockIdx.y * g.slab, end = min(g.rows, from + g.slab);
    const T *x = (const T *)g.x, *positive = (const T *)g.positive;
    float most[N] = {}, sum[N] = {};
    for (int64_t r = from + wave; r < end; r += 4 * AHEAD) {
        v4i raw[AHEAD], keep[AHEAD];
#pragma unroll
        for (int h = 0; h < AHEAD; ++h) {
            const int64_t at = r + 4 * h;
            raw[h] = load_piece(x + at * g.stride + c, at < end ? g.cols - c : 0);
            if (positive) keep[h] = load_piece(positive + at * g.cols + c, at < end ? g.cols - c : 0);
        }
#pragma unroll
        for (int h = 0; h < AHEAD; ++h) {
            const int64_t at = r + 4 * h;
            const float f = g.row_factor && at < end ? g.row_factor[at] : 1.0f;
            float v[N], y[N];
            piece_floats<T>(raw[h], v);
            if (positive) piece_floats<T>(keep[h], y);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                if (positive && !(y[e] > 0.0f)) v[e] = 0.0f;
                sum[e] += v[e];
                most[e] = MaxOf::of(most[e], __uint_as_float(magnitude_bits(v[e] * f)));
            }
        }
    }
#pragma unroll
    for (int e = 0; e < N; ++e) most_of[wave][lane * N + e] = most[e], sum_of[wave][lane * N + e] = sum[e];
    __syncthreads();
    float *to = g.partial + (int64_t)blockIdx.y * 2 * g.cols;
    for (int i = threadIdx.x; i < 64 * N; i += 256) {
        const int64_t col = (int64_t)blockIdx.x * 64 * N + i;
        if (col >= g.cols) break;
        float m = most_of[0][i], s = sum_of[0][i];
#pragma unroll
        for (int w = 1; w < 4; ++w) m = MaxOf::of(m, most_of[w][i]), s += sum_of[w][i];
        to[col] = m, to[g.cols + col] = s;
    }
}

// of [parts][2][cols]: multipliers, scales and sums.  32 columns and 32 runs of parts to a workgroup, the runs joined in pairs.
struct Join {
    const float *partial;
    int64_t parts, cols;
    float *multipliers, *scales;
    void *sums;
    int sums_dtype;
};
__global__ __launch_bounds__(1024) void columns_join_kernel(Join g)
{
    __shared__ float most_of[32][33], sum_of[32][33];
    const int c = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int64_t col = (int64_t)blockIdx.x * 32 + c, each = ceil_div64(g.parts, 32), end = min(g.parts, each * (w + 1));
    float m = 0.0f, s = 0.0f;
    if (col < g.cols) {
#pragma unroll 4
        for (int64_t p = each * w; p < end; ++p) {
            m = MaxOf::of(m, g.partial[p * 2 * g.cols + col]);
            if (g.sums) s += g.partial[(p * 2 + 1) * g.cols + col];
        }
    }
    most_of[w][c] = m, sum_of[w][c] = s;
    for (int half = 16; half; half /= 2) {
        __syncthreads();
        if (w < half) most_of[w][c] = MaxOf::of(most_of[w][c], most_of[w + half][c]), sum_of[w][c] += sum_of[w + half][c];
    }
    if (w != 0 || col >= g.cols) return;
    if (g.multipliers) {
        const uint32_t largest = __float_as_uint(most_of[0][c]);
        g.multipliers[col] = q8_multiplier(largest);
        g.scales[col] = q8_scale(largest);
    }
    if (g.sums) store_from_float(g.sums, g.sums_dtype, col, sum_of[0][c]);
}

// A workgroup of four waves takes 64 rows (a step of the columns' operand), four units in turn to a wave.
template <typename T>
__global__ __launch_bounds__(256) void columns_kernel(I8Columns g, const float *multipliers)
{
    using U = Unit<T>;
    __shared__ __attribute__((aligned(16))) uint32_t corners[4][CORNER];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t units = i8_steps(g.cols), across = ceil_div64(units, 4), u = (int64_t)blockIdx.x % across * 4 + wave, step = (int64_t)blockIdx.x / across;
    if (u >= units) return;
    const int64_t col0 = u * 64, c = col0 + unit_col<T>();
    float multiplier[U::N];
    load_floats(multipliers, AMSIM_DTYPE_F32, c, g.cols - c, multiplier);
    v4i raw[4][U::LOADS];
#pragma unroll
    for (int q = 0; q < 4; ++q) load_unit((const T *)g.x, (const T *)g.positive, g.rows, g.cols, g.row_stride, step * 64 + 16 * q, col0, raw[q]);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int64_t row0 = step * 64 + 16 * q;
        if (row0 >= g.rows) break;
        Codes<U::N> codes;
#pragma unroll
        for (int i = 0; i < U::LOADS; ++i) {
            const int64_t r = row0 + unit_row<T>(i);
            const float f = g.row_factor && r < g.rows ? g.row_factor[r] : 1.0f;
            float v[U::N];
            piece_floats<T>(raw[q][i], v);
#pragma unroll
            for (int d = 0; d < U::N / 4; ++d) {
                uint32_t b[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) b[e] = q8_code(g.row_factor ? v[4 * d + e] * f : v[4 * d + e], multiplier[4 * d + e]) & 255u;
                codes.w[i][d] = b[0] | b[1] << 8 | b[2] << 16 | b[3] << 24;
            }
        }
        store_unit<T>(codes, corners[wave], g.rows, g.cols, row0, col0, g.by_rows, g.by_columns);
    }
}

template <typename T>
__global__ __launch_bounds__(256) void dequantize_kernel(const uint8_t *q, int64_t rows, int64_t length, T *out)
{
    constexpr int N = PIECE<T>;
    const int64_t steps = i8_steps(length), f = (int64_t)blockIdx.x / steps, step = (int64_t)blockIdx.x % steps;
    const float *scales = (const float *)(q + i8_code_bytes(rows, length));
#pragma unroll
    for (int at = threadIdx.x; at < 1024 / N; at += 256) {
        const int r = at / (64 / N), c = at % (64 / N) * N;
        const int64_t row = 16 * f + r, col = 64 * step + c;
        if (row >= rows || col >= length) continue;
        uint32_t w[N / 4];
        __builtin_memcpy(w, __builtin_assume_aligned(q + ((f * steps + step) * 64 + c / 16 * 16 + r) * 16 + c % 16, N), N);
        float v[N];
        code_values(w, scales[row], v);
        store_piece(out + row * length + col, length - col, v);
    }
}

template <typename Fn> int with_type(int dtype, Fn &&fn)
{
    switch (dtype) {
    case AMSIM_DTYPE_F32: return fn(0.0f);
    case AMSIM_DTYPE_BF16: return fn((__bf16)0.0f);
    default: return fn((_Float16)0.0f);
    }
}

int64_t slab_rows(int64_t rows, int64_t cols)
{
    const int64_t across = ceil_div64(cols, 256), slabs = std::max<int64_t>(1, std::min<int64_t>(ceil_div64(rows, 32), 2048 / across));
    return ceil_div64(ceil_div64(rows, slabs), 16) * 16;
}

constexpr int64_t MOST_BLOCKS = 1 << 22;  // (of up to 1024 threads: a launch has less than 2^32)

}  // namespace

int i8_convert_rows(const I8Rows &j, hipStream_t stream)
{
    const int64_t blocks = ceil_div64(j.rows, 16), each = ceil_div64(i8_steps(j.cols), WAVES);
    if (blocks >= MOST_BLOCKS) return fail(AMSIM_ERR_UNSUPPORTED, "int8: more rows than one launch takes");
    return with_type(j.dtype, [&](auto zero) {
        using T = decltype(zero);
        const auto kernel = each == 1 ? rows_kernel<T, 1> : each == 2 ? rows_kernel<T, 2> : each <= 4 ? rows_kernel<T, 4> : each <= 8 ? rows_kernel<T, 8> : rows_kernel<T, 0>;
        kernel<<<(unsigned)blocks, WG, 0, stream>>>(j);
        AMSIM_HIP_CHECK(hipGetLastError());
        return (int)AMSIM_OK;
    });
}

int64_t i8_columns_workspace(int64_t rows, int64_t cols) { return ceil_div64(rows, slab_rows(rows, cols)) * 2 * cols + cols; }

int i8_convert_columns(const I8Columns &j, float *workspace, hipStream_t stream)
{
    const int64_t slab = slab_rows(j.rows, j.cols), slabs = ceil_div64(j.rows, slab);
    const int64_t blocks = ceil_div64(i8_steps(j.cols), 4) * ceil_div64(j.rows, 64);
    if (blocks >= MOST_BLOCKS || ceil_div64(j.cols, 32) >= MOST_BLOCKS) return fail(AMSIM_ERR_UNSUPPORTED, "int8: more columns than one launch takes");
    float *multipliers = workspace, *partial = workspace + j.cols;
    return with_type(j.dtype, [&](auto zero) {
        using T = decltype(zero);
        if (!j.partial) {
            const Look look{j.x, j.positive, j.rows, j.cols, j.row_stride, j.row_factor, slab, partial};
            columns_look_kernel<T><<<dim3((unsigned)ceil_div64(j.cols, 64 * PIECE<T>), (unsigned)slabs), 256, 0, stream>>>(look);
            AMSIM_HIP_CHECK(hipGetLastError());
        }
        const bool codes = j.by_rows || j.by_columns;
        const Join join{j.partial ? j.partial : partial, j.partial ? ceil_div64(j.rows, 16) : slabs, j.cols, codes ? multipliers : nullptr, j.scales, j.sums, j.sums_dtype};
        columns_join_kernel<<<(unsigned)ceil_div64(j.cols, 32), 1024, 0, stream>>>(join);
        AMSIM_HIP_CHECK(hipGetLastError());
        if (codes) {
            columns_kernel<T><<<(unsigned)blocks, 256, 0, stream>>>(j, multipliers);
            AMSIM_HIP_CHECK(hipGetLastError());
        }
        return (int)AMSIM_OK;
    });
}

}  // namespace amsim

using namespace amsim;

extern "C" {

size_t amsim_i8_operand_bytes(int64_t rows, int64_t length)
{
    return i8_extents_fit(rows, length) && rows && length ? (size_t)i8_bytes(rows, length) : 0;
}

size_t amsim_i8_quantize_workspace_bytes(int64_t rows, int64_t cols) { return i8_extents_fit(cols, rows) && rows && cols ? (size_t)i8_columns_workspace(rows, cols) * 4 : 0; }

int amsim_i8_quantize(const void *x, int dtype, int64_t rows, int64_t cols, int64_t row_stride, void *by_rows, void *by_columns, void *workspace,
                      size_t workspace_bytes, void *stream)
{
    if (!known_dtype(dtype)) return fail(AMSIM_ERR_INVALID, "int8: unknown element type");
    if ((by_rows && !i8_extents_fit(rows, cols)) || (by_columns && !i8_extents_fit(cols, rows)) || rows < 0 || cols < 0)
        return fail(AMSIM_ERR_UNSUPPORTED, "int8: extents out of range");
    if (rows == 0 || cols == 0) return fail(AMSIM_ERR_INVALID, "int8: empty tensor");
    if (!x || (!by_rows && !by_columns)) return fail(AMSIM_ERR_INVALID, "int8: null pointer");
    if (row_stride < cols && rows > 1) return fail(AMSIM_ERR_INVALID, "int8: rows overlap");
    if (((uintptr_t)x & (element_bytes(dtype) - 1)) || ((uintptr_t)by_rows & 15) || ((uintptr_t)by_columns & 15)) return fail(AMSIM_ERR_INVALID, "int8: misaligned pointer");
    if (by_columns && (!workspace || workspace_bytes < amsim_i8_quantize_workspace_bytes(rows, cols) || ((uintptr_t)workspace & 255)))
        return fail(AMSIM_ERR_WORKSPACE, "int8: workspace missing, misaligned or too small");
    if (by_rows) {
        const I8Rows j{x, nullptr, dtype, rows, cols, row_stride, nullptr, (uint8_t *)by_rows, nullptr, (float *)((uint8_t *)by_rows + i8_code_bytes(rows, cols)), nullptr, nullptr};
        if (int rc = i8_convert_rows(j, (hipStream_t)stream)) return rc;
    }
    if (!by_columns) return AMSIM_OK;
    const I8Columns j{x, nullptr, dtype, rows, cols, row_stride, nullptr, nullptr, (uint8_t *)by_columns, (float *)((uint8_t *)by_columns + i8_code_bytes(cols, rows)),
                      nullptr, 0, nullptr};
    return i8_convert_columns(j, (float *)workspace, (hipStream_t)stream);
}

int amsim_i8_dequantize(const void *q, int64_t rows, int64_t length, int dtype, void *out, void *stream)
{
    if (!known_dtype(dtype)) return fail(AMSIM_ERR_INVALID, "int8: unknown element type");
    if (!i8_extents_fit(rows, length)) return fail(AMSIM_ERR_UNSUPPORTED, "int8: extents out of range");
    if (rows == 0 || length == 0) return fail(AMSIM_ERR_INVALID, "int8: empty tensor");
    if (!q || !out) return fail(AMSIM_ERR_INVALID, "int8: null pointer");
    if (((uintptr_t)q & 15) || ((uintptr_t)out & 15)) return fail(AMSIM_ERR_INVALID, "int8: misaligned pointer");
    const int64_t blocks = ceil_div64(rows, 16) * i8_steps(length);
    if (blocks >= 4 * MOST_BLOCKS) return fail(AMSIM_ERR_UNSUPPORTED, "int8: more values than one launch takes");
    return with_type(dtype, [&](auto zero) {
        using T = decltype(zero);
        dequantize_kernel<T><<<(unsigned)blocks, 256, 0, (hipStream_t)stream>>>((const uint8_t *)q, rows, length, (T *)out);
        AMSIM_HIP_CHECK(hipGetLastError());
        return (int)AMSIM_OK;
    });
}

}  // extern "C"
