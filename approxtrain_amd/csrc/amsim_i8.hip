// Conversions to 8-bit integers with a scale for each row or column (amsim_i8.h), and back.
//
// Bound by memory, and below some hundred thousand values by the launches: a scale has to be known before the first code is
// written.  Along rows one workgroup sees 16 rows whole and holds them in registers between the two; along columns slabs of
// rows are looked through first, beside a conversion along rows where there is one, and the tensor is read again.
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

// ---- along columns --------------------------------------------------------------------------------------------------

// The largest magnitudes (and sums) in every column of a slab of rows: [slabs][2][cols].  A workgroup's waves take its rows in
// turn, four of them under way at once.
struct Look {
    const void *x, *positive;
    int dtype;
    int64_t rows, cols, stride;
    const float *row_factor;
    bool sums;
    int64_t slab, across;    // rows of a slab, workgroups across
    float *partial;
};
template <typename T, bool MASK> __device__ __forceinline__ void look_through(const Look &g, int64_t id, float *lds)
{
    constexpr int N = PIECE<T>, AHEAD = 4;
    float (*most_of)[64 * N] = (float (*)[64 * N])lds, (*sum_of)[64 * N] = most_of + WAVES;
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t slab = id / g.across, col0 = id % g.across * 64 * N, c = col0 + lane * N, from = slab * g.slab, end = min(g.rows, from + g.slab);
    const T *x = (const T *)g.x, *positive = (const T *)g.positive;
    float most[N] = {}, sum[N] = {};
    for (int64_t r = from + wave; r < end; r += WAVES * AHEAD) {
        v4i raw[AHEAD], keep[MASK ? AHEAD : 1];
#pragma unroll
        for (int h = 0; h < AHEAD; ++h) {
            const int64_t at = r + WAVES * h;
            raw[h] = load_piece(x + at * g.stride + c, at < end ? g.cols - c : 0);
            if constexpr (MASK) keep[h] = load_piece(positive + at * g.cols + c, at < end ? g.cols - c : 0);
        }
#pragma unroll
        for (int h = 0; h < AHEAD; ++h) {
            const int64_t at = r + WAVES * h;
            const float f = g.row_factor && at < end ? g.row_factor[at] : 1.0f;
            float v[N], y[N];
            piece_floats<T>(raw[h], v);
            if constexpr (MASK) piece_floats<T>(keep[h], y);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                if (MASK && !(y[e] > 0.0f)) v[e] = 0.0f;
                sum[e] += v[e];
                most[e] = MaxOf::of(most[e], __uint_as_float(magnitude_bits(v[e] * f)));
            }
        }
    }
#pragma unroll
    for (int e = 0; e < N; ++e) most_of[wave][lane * N + e] = most[e], sum_of[wave][lane * N + e] = sum[e];
    __syncthreads();
    float *to = g.partial + slab * 2 * g.cols;
    for (int i = threadIdx.x; i < 64 * N; i += WG) {
        if (col0 + i >= g.cols) break;
        float m = most_of[0][i], s = sum_of[0][i];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) m = MaxOf::of(m, most_of[w][i]), s += sum_of[w][i];
        to[col0 + i] = m;
        if (g.sums) to[g.cols + col0 + i] = s;
    }
}

// How rows are converted: by sixteen with 0 to 8 units of a wave held, or by themselves.  Eight units by themselves have a CU's
// registers (4096 x 4096 bf16: a serving call 72.0 us, 73.8 in half of them); beside a look they leave half to it (a training
// step of 4096^3 274 us, 285 else, and 290 in launches of their own).
constexpr int EIGHT_ALONE = 9, LANES_64 = -1, LANES_512 = -2, LANES_512_TWICE = -3, LANES_512_AGAIN = -4;

// A conversion along rows, a look through columns, or both beside each other (the two do not wait for each other).
constexpr int LDS_FLOATS = 2 * WAVES * 64 * PIECE<__bf16>;
template <typename T, int HOW, bool MASK> __global__ __launch_bounds__(WG, HOW == EIGHT_ALONE || (HOW == 8 && sizeof(T) == 4) ? 2 : 4) void rows_and_look_kernel(I8Rows rows, unsigned row_blocks, Look look)
{
    __shared__ __attribute__((aligned(16))) float lds[LDS_FLOATS];
    static_assert(LDS_FLOATS >= WAVES * (CORNER + 16) + WAVES * 8 * 64, "");
    if (blockIdx.x < row_blocks) {
        if constexpr (HOW >= 0) convert_rows<T, (HOW == EIGHT_ALONE ? 8 : HOW), MASK>(rows, (uint32_t *)lds);
        else if constexpr (HOW == LANES_64) convert_single_rows<T, 64, 16, MASK>(rows, lds);
        else if constexpr (HOW == LANES_512) convert_single_rows<T, 512, 8, MASK>(rows, lds);
        else if constexpr (HOW == LANES_512_TWICE) convert_single_rows<T, 512, 16, MASK>(rows, lds);
        else convert_single_rows<T, 512, 0, MASK>(rows, lds);
        return;
    }
    const int64_t id = blockIdx.x - row_blocks;
    if (look.dtype == AMSIM_DTYPE_F32) look_through<float, MASK>(look, id, lds);
    else if (look.dtype == AMSIM_DTYPE_BF16) look_through<__bf16, MASK>(look, id, lds);
    else look_through<_Float16, MASK>(look, id, lds);
}

// A wavefront's 64 columns over the slabs, joined by maximum or sum: 16 lanes' loads are 64 columns of a slab, four slabs
// to a load, eight loads under way.  In every lane: those of columns 4 (lane % 16) and the three that follow.
template <typename Op> __device__ __forceinline__ v4f over_slabs(const float *partial, int64_t slabs, int64_t cols, int64_t col0)
{
    constexpr int AHEAD = 8;
    const int lane = lane_id();
    const int64_t c = col0 + lane % 16 * 4;
    v4f all = {0, 0, 0, 0};
    for (int64_t p = lane / 16; p < ceil_div64(slabs, 4) * 4; p += 4 * AHEAD) {
        v4f v[AHEAD];
#pragma unroll
        for (int h = 0; h < AHEAD; ++h) v[h] = __builtin_bit_cast(v4f, load_piece(partial + (p + 4 * h) * 2 * cols + c, p + 4 * h < slabs ? cols - c : 0));
#pragma unroll
        for (int h = 0; h < AHEAD; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) all[e] = Op::of(all[e], v[h][e]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(all[e]), __float_as_uint(all[e]), false, false);
        all[e] = Op::of(__uint_as_float(r[0]), __uint_as_float(r[1]));
        const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(all[e]), __float_as_uint(all[e]), false, false);
        all[e] = Op::of(__uint_as_float(h[0]), __uint_as_float(h[1]));
    }
    return all;
}

// A workgroup of four waves takes 64 rows (a step of the columns' operand), four units in turn to a wave, whose loads are under
// way while the slabs are joined.  Look and conversion of 4096 x 4096 to columns: f32 31 us (150 MB), bf16 23; 784 x 300 f32 9.4.
template <typename T, bool MASK>
__global__ __launch_bounds__(256) void columns_kernel(I8Columns g, const float *partial, int64_t slabs)
{
    using U = Unit<T>;
    __shared__ __attribute__((aligned(16))) uint32_t corners[4][CORNER];
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t units = i8_steps(g.cols), across = ceil_div64(units, 4), u = (int64_t)blockIdx.x % across * 4 + wave, step = (int64_t)blockIdx.x / across;
    if (u >= units) return;
    const int64_t col0 = u * 64, first = col0 + lane * 4;
    const bool codes = g.by_rows || g.by_columns;
    v4i raw[4][U::LOADS];
    if (codes)
#pragma unroll
        for (int q = 0; q < 4; ++q) load_unit<MASK>((const T *)g.x, (const T *)g.positive, g.rows, g.cols, g.row_stride, step * 64 + 16 * q, col0, raw[q]);
    float factor[4][U::LOADS];
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int i = 0; i < U::LOADS; ++i) {
            const int64_t r = step * 64 + 16 * q + unit_row<T>(i);
            factor[q][i] = g.row_factor && r < g.rows ? g.row_factor[r] : 1.0f;
        }
    if (step == 0 && g.sums) {
        const v4f s = over_slabs<SumOf>(partial + g.cols, slabs, g.cols, col0);
        if (lane < 16)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (first + e < g.cols) store_from_float(g.sums, g.sums_dtype, first + e, s[e]);
    }
    if (!codes) return;
    const v4f most = over_slabs<MaxOf>(partial, slabs, g.cols, col0);
    if (lane < 16) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t largest = __float_as_uint(most[e]);
            corners[wave][4 * lane + e] = __float_as_uint(q8_multiplier(largest));
            if (step == 0 && first + e < g.cols) g.scales[first + e] = q8_scale(largest);
        }
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    float multiplier[U::N];
#pragma unroll
    for (int e = 0; e < U::N; ++e) multiplier[e] = __uint_as_float(corners[wave][unit_col<T>() + e]);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int64_t row0 = step * 64 + 16 * q;
        if (row0 >= g.rows) break;
        Codes<U::N> unit;
#pragma unroll
        for (int i = 0; i < U::LOADS; ++i) {
            const float f = factor[q][i];
            float v[U::N];
            piece_floats<T>(raw[q][i], v);
#pragma unroll
            for (int d = 0; d < U::N / 4; ++d) {
                uint32_t b[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) b[e] = q8_code(g.row_factor ? v[4 * d + e] * f : v[4 * d + e], multiplier[4 * d + e]);
                unit.w[i][d] = q8_pack(b[0], b[1], b[2], b[3]);
            }
        }
        store_unit<T>(unit, corners[wave], g.rows, g.cols, row0, col0, g.by_rows, g.by_columns);
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

// Slabs of rows that are looked through: enough workgroups for the card beside those that convert rows, few enough for
// every wavefront that converts columns to join them by itself (to quantise the columns of 16384 x 1000 bf16 takes 24.1 us
// with 64 slabs, 28.9 with 32, 29.8 with 256; a training step of 8192 x 512 x 512 62 with 64, 64 with 128).
int64_t slab_rows(int64_t rows, int64_t cols)
{
    const int64_t slabs = std::min(ceil_div64(rows, 64), std::max<int64_t>(16, std::min<int64_t>(64, 128 / ceil_div64(cols, 512))));
    return ceil_div64(rows, slabs);
}

constexpr int64_t MOST_BLOCKS = 1 << 22;  // (of up to 512 threads: a launch has less than 2^32)

// Whether rows are converted by themselves: us so, and by sixteen, of bf16 rows of 4096: 16 rows 4.9 and 7.7, 512 rows 4.5 and 8.2,
// 1024 rows 6.8 and 8.8, 2048 rows 10.0 and 10.3, 4096 rows 17.6 and 12.9 (pieces of 16 bytes from different workgroups fill a
// line); 2048 rows of 10000 24.9 and 21.9.
bool single_rows(const I8Rows &j) { return !j.by_columns && j.rows <= 1024; }

template <typename T, int HOW> void launch_rows_and_look(const I8Rows &rows, unsigned row_blocks, const Look &look, unsigned look_blocks, hipStream_t stream)
{
    const auto kernel = rows.positive || look.positive ? rows_and_look_kernel<T, HOW, true> : rows_and_look_kernel<T, HOW, false>;
    kernel<<<row_blocks + look_blocks, WG, 0, stream>>>(rows, row_blocks, look);
}

}  // namespace

int64_t i8_partial_floats(int64_t rows, int64_t cols) { return ceil_div64(rows, slab_rows(rows, cols)) * 2 * cols; }

int i8_convert(const I8Rows *rows, const I8Columns *columns, float *partial, hipStream_t stream)
{
    Look look{};
    int64_t row_blocks = 0, look_blocks = 0, blocks = 0, slabs = 0;
    if (rows) row_blocks = ceil_div64(rows->rows, 16) * (!single_rows(*rows) ? 1 : rows->cols <= 1024 ? 2 : 16);
    if (columns) {
        const I8Columns &c = *columns;
        look = Look{c.x, c.positive, c.dtype, c.rows, c.cols, c.row_stride, c.row_factor, c.sums != nullptr, slab_rows(c.rows, c.cols),
                    ceil_div64(c.cols, c.dtype == AMSIM_DTYPE_F32 ? 64 * PIECE<float> : 64 * PIECE<__bf16>), partial};
        slabs = ceil_div64(c.rows, look.slab);
        look_blocks = slabs * look.across;
        blocks = ceil_div64(i8_steps(c.cols), 4) * (c.by_rows || c.by_columns ? ceil_div64(c.rows, 64) : 1);
    }
    if (row_blocks + look_blocks >= MOST_BLOCKS || blocks >= MOST_BLOCKS) return fail(AMSIM_ERR_UNSUPPORTED, "int8: more values than one launch takes");
    if (const int rc = with_type(rows ? rows->dtype : AMSIM_DTYPE_F32, [&](auto zero) {
            using T = decltype(zero);
            const I8Rows j = rows ? *rows : I8Rows{};
            const int64_t each = ceil_div64(i8_steps(j.cols), WAVES);  // units of a wave
            const auto launch = rows && single_rows(j) ? j.cols <= 1024 ? launch_rows_and_look<T, LANES_64> : j.cols <= 4096 ? launch_rows_and_look<T, LANES_512>
                                  : j.cols <= 8192 ? launch_rows_and_look<T, LANES_512_TWICE> : launch_rows_and_look<T, LANES_512_AGAIN>
                              : each <= 1 ? launch_rows_and_look<T, 1> : each == 2 ? launch_rows_and_look<T, 2> : each <= 4 ? launch_rows_and_look<T, 4>
                              : each <= 8 ? columns ? launch_rows_and_look<T, 8> : launch_rows_and_look<T, EIGHT_ALONE> : launch_rows_and_look<T, 0>;
            launch(j, (unsigned)row_blocks, look, (unsigned)look_blocks, stream);
            AMSIM_HIP_CHECK(hipGetLastError());
            return (int)AMSIM_OK;
        }))
        return rc;
    if (!columns) return AMSIM_OK;
    return with_type(columns->dtype, [&](auto zero) {
        const auto kernel = columns->positive ? columns_kernel<decltype(zero), true> : columns_kernel<decltype(zero), false>;
        kernel<<<(unsigned)blocks, 256, 0, stream>>>(*columns, partial, slabs);
        AMSIM_HIP_CHECK(hipGetLastError());
        return (int)AMSIM_OK;
    });
}

}  // namespace amsim

using namespace amsim;

extern "C" {

size_t amsim_i8_operand_workspace_bytes(int64_t rows, int64_t length)
{
    return i8_extents_fit(rows, length) && rows && length ? (size_t)i8_bytes(rows, length) : 0;
}

size_t amsim_i8_quantize_workspace_bytes(int64_t rows, int64_t cols) { return i8_extents_fit(cols, rows) && rows && cols ? (size_t)i8_partial_floats(rows, cols) * 4 : 0; }

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
    const I8Rows r{x, nullptr, dtype, rows, cols, row_stride, nullptr, (uint8_t *)by_rows, nullptr, (float *)((uint8_t *)by_rows + i8_code_bytes(rows, cols))};
    const I8Columns c{x, nullptr, dtype, rows, cols, row_stride, nullptr, nullptr, (uint8_t *)by_columns, (float *)((uint8_t *)by_columns + i8_code_bytes(cols, rows)),
                      nullptr, 0};
    return i8_convert(by_rows ? &r : nullptr, by_columns ? &c : nullptr, (float *)workspace, (hipStream_t)stream);
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
