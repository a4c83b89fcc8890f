// What the conversions to 8-bit operands share (amsim_i8.hip, amsim_i8_small.hip): units of 16 rows x 64 columns from memory to
// codes, and rows.
//
// A wavefront's unit is a step of one fragment: loads of 16 bytes a lane, whole lines of 128 bytes and more; codes of rows go
// out as 1 KB in a piece.  For an operand of the columns the unit's bytes are transposed in a wavefront's own corner of
// LDS, four by four in registers.
#ifndef AMSIM_I8_CONVERT_H_
#define AMSIM_I8_CONVERT_H_

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
template <bool MASK, typename T>
__device__ __forceinline__ void load_unit(const T *x, const T *positive, int64_t rows, int64_t cols, int64_t stride, int64_t row0, int64_t col0,
                                          v4i (&raw)[Unit<T>::LOADS])
{
    using U = Unit<T>;
    const int64_t c = col0 + unit_col<T>();
    v4i keep[MASK ? U::LOADS : 1];
#pragma unroll
    for (int i = 0; i < U::LOADS; ++i) {
        const int64_t r = row0 + unit_row<T>(i);
        raw[i] = load_piece(x + r * stride + c, r < rows ? cols - c : 0);
        if constexpr (MASK) keep[i] = load_piece(positive + r * cols + c, r < rows ? cols - c : 0);
    }
    if constexpr (MASK)
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

// HELD units of a wave stay in registers; 0: rows are read again.  4096 x 4096 bf16 12.4 us (50 MB): all loads are under way at
// once, and the codes go out when a row's largest is known.
template <typename T, int HELD, bool MASK> __device__ __forceinline__ void convert_rows(const I8Rows &g, uint32_t *lds)
{
    using U = Unit<T>;
    uint32_t (*corners)[CORNER] = (uint32_t (*)[CORNER])lds, (*largest_of)[16] = (uint32_t (*)[16])(lds + WAVES * CORNER);
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row0 = (int64_t)blockIdx.x * 16, units = i8_steps(g.cols);
    const T *x = (const T *)g.x, *positive = (const T *)g.positive;
    v4i held[HELD ? HELD : 1][U::LOADS];
    uint32_t largest[U::LOADS] = {};
    // What the unit's values are as codes are made of them.  The columns' factors come by way of LDS where rows are held (from
    // memory, twice for every unit, they took 10 us of 4096 x 4096's 22).
    float *factors = (float *)(lds + WAVES * (CORNER + 16));
    auto floats = [&](const v4i &raw, int64_t col0, float (&v)[U::N]) {
        piece_floats<T>(raw, v);
        if (g.col_factor) {
            float f[U::N];
            const int64_t c = col0 + unit_col<T>();
            if constexpr (HELD > 0) {
#pragma unroll
                for (int e = 0; e < U::N; e += 4) __builtin_memcpy(f + e, __builtin_assume_aligned(factors + c + e, 16), 16);
            } else {
                load_floats(g.col_factor, AMSIM_DTYPE_F32, c, g.cols - c, f);
            }
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
    };
    if constexpr (HELD > 0) {
#pragma unroll
        for (int h = 0; h < HELD; ++h) load_unit<MASK>(x, positive, g.rows, g.cols, g.row_stride, row0, (wave + h * WAVES) * 64, held[h]);
        if (g.col_factor) {
            for (int64_t c = threadIdx.x * 4; c < units * 64; c += WG * 4) {
                const v4i f = load_piece(g.col_factor + c, g.cols - c);
                __builtin_memcpy(__builtin_assume_aligned(factors + c, 16), &f, 16);
            }
            __syncthreads();
        }
#pragma unroll
        for (int h = 0; h < HELD; ++h)
            if (wave + h * WAVES < units) look(held[h], (wave + h * WAVES) * 64);
    } else {
        for (int64_t u = wave; u < units; u += 2 * WAVES) {
            v4i two[2][U::LOADS];
            load_unit<MASK>(x, positive, g.rows, g.cols, g.row_stride, row0, u * 64, two[0]);
            load_unit<MASK>(x, positive, g.rows, g.cols, g.row_stride, row0, (u + WAVES) * 64, two[1]);
            look(two[0], u * 64);
            if (u + WAVES < units) look(two[1], (u + WAVES) * 64);
        }
    }
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
            load_unit<MASK>(x, positive, g.rows, g.cols, g.row_stride, row0, u * 64, two[0]);
            load_unit<MASK>(x, positive, g.rows, g.cols, g.row_stride, row0, (u + WAVES) * 64, two[1]);
            encode(two[0], u * 64);
            if (u + WAVES < units) encode(two[1], (u + WAVES) * 64);
        }
    }
}

// Rows by themselves, for few of them: sixteen to a workgroup would leave most of the card idle.  LANES lanes hold a row, EACH
// values each (0: the row is read again), and write its 16-byte pieces of the fragments' lines.
template <typename T, int LANES, int EACH, bool MASK> __device__ __forceinline__ void convert_single_rows(const I8Rows &g, float *lds)
{
    constexpr int N = PIECE<T>, PIECES = EACH ? EACH / N : 1;
    const int in_row = threadIdx.x % LANES;
    const int64_t row = (int64_t)blockIdx.x * (WG / LANES) + threadIdx.x / LANES, steps = i8_steps(g.cols);
    const T *x = (const T *)g.x, *positive = (const T *)g.positive;
    RowLanes<LANES> lanes{(float (*)[RowLanes<LANES>::WAVES][2])lds};
    auto load = [&](int64_t c) {
        const int64_t count = row < g.rows ? g.cols - c : 0;
        v4i raw = load_piece(x + row * g.row_stride + c, count);
        if constexpr (MASK) {
            const v4i keep = load_piece(positive + row * g.cols + c, count);
            T v[N], y[N];
            __builtin_memcpy(v, &raw, 16);
            __builtin_memcpy(y, &keep, 16);
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = to_float(y[e]) > 0.0f ? v[e] : (T)0.0f;
            __builtin_memcpy(&raw, v, 16);
        }
        return raw;
    };
    auto floats = [&](v4i raw, int64_t c, float (&v)[N]) {
        piece_floats<T>(raw, v);
        if (!g.col_factor) return;
        float f[N];
        load_floats(g.col_factor, AMSIM_DTYPE_F32, c, g.cols - c, f);
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] *= f[e];
    };
    float largest = 0.0f;
    auto look = [&](v4i raw, int64_t c) {
        float v[N];
        floats(raw, c, v);
#pragma unroll
        for (int e = 0; e < N; ++e) largest = MaxOf::of(largest, __uint_as_float(magnitude_bits(v[e])));
    };
    auto store = [&](v4i raw, int64_t c, float multiplier) {
        if (c >= steps * I8_STEP || row >= ceil_div64(g.rows, 16) * 16) return;
        float v[N];
        floats(raw, c, v);
        store_codes(g.by_rows + (row / 16 * steps + c / 64) * 1024 + (c % 64 / 16 * 16 + row % 16) * 16 + c % 16, v, multiplier);
    };
    v4i raw[PIECES];
    if constexpr (EACH > 0) {
#pragma unroll
        for (int p = 0; p < PIECES; ++p) raw[p] = load((int64_t)(p * LANES + in_row) * N);
#pragma unroll
        for (int p = 0; p < PIECES; ++p) look(raw[p], (int64_t)(p * LANES + in_row) * N);
    } else {
#pragma unroll 4
        for (int64_t c = in_row * N; c < g.cols; c += LANES * N) look(load(c), c);
    }
    largest = lanes.template one<MaxOf>(largest);
    const float multiplier = q8_multiplier(__float_as_uint(largest));
    if (in_row == 0 && row < g.rows) g.scales[row] = q8_scale(__float_as_uint(largest));
    if constexpr (EACH > 0) {
#pragma unroll
        for (int p = 0; p < PIECES; ++p) store(raw[p], (int64_t)(p * LANES + in_row) * N, multiplier);
    } else {
#pragma unroll 4
        for (int64_t c = in_row * N; c < steps * I8_STEP; c += LANES * N) store(load(c), c, multiplier);
    }
}

// a piece's codes with its columns' multipliers; `scaled`: of factor times the values
template <typename T>
__device__ __forceinline__ void column_codes(v4i raw, bool scaled, float factor, const float (&multiplier)[PIECE<T>], uint32_t (&w)[PIECE<T> / 4])
{
    float v[PIECE<T>];
    piece_floats<T>(raw, v);
#pragma unroll
    for (int d = 0; d < PIECE<T> / 4; ++d) {
        uint32_t b[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) b[e] = q8_code(scaled ? v[4 * d + e] * factor : v[4 * d + e], multiplier[4 * d + e]);
        w[d] = q8_pack(b[0], b[1], b[2], b[3]);
    }
}

// How rows are converted: by sixteen with 0 to 8 units of a wave held, or by themselves.  Eight units by themselves have a CU's
// registers (4096 x 4096 bf16: a serving call 72.0 us, 73.8 in half of them); beside a look they leave half to it (a training
// step of 4096^3 274 us, 285 else, and 290 in launches of their own).
constexpr int EIGHT_ALONE = 9, LANES_64 = -1, LANES_512 = -2, LANES_512_TWICE = -3, LANES_512_AGAIN = -4;

// Whether rows are converted by themselves: us so, and by sixteen, of bf16 rows of 4096: 16 rows 4.9 and 7.7, 512 rows 4.5 and 8.2,
// 1024 rows 6.8 and 8.8, 2048 rows 10.0 and 10.3, 4096 rows 17.6 and 12.9 (pieces of 16 bytes from different workgroups fill a
// line); 2048 rows of 10000 24.9 and 21.9.
bool single_rows(const I8Rows &j) { return !j.by_columns && j.rows <= 1024; }

constexpr int64_t MOST_BLOCKS = 1 << 22;  // (of up to 512 threads: a launch has less than 2^32)

template <typename Fn> int with_type(int dtype, Fn &&fn)
{
    switch (dtype) {
    case AMSIM_DTYPE_F32: return fn(0.0f);
    case AMSIM_DTYPE_BF16: return fn((__bf16)0.0f);
    default: return fn((_Float16)0.0f);
    }
}

}  // namespace

// Rows and columns in one launch, or columns alone, where the columns are short enough to be converted whole.
bool i8_small(const I8Rows *rows, const I8Columns &columns);
int i8_convert_small(const I8Rows *rows, const I8Columns &columns, hipStream_t stream);

}  // namespace amsim
#endif  // AMSIM_I8_CONVERT_H_
