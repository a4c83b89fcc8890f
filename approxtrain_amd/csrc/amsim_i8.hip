// Conversions to 8-bit integers with a scale for each row or column (amsim_i8.h), and back.
//
// Bound by memory, and below some hundred thousand values by the launches: a scale has to be known before the first code is
// written.  Along rows one workgroup sees 16 rows whole and holds them in registers between the two; along columns slabs of
// rows are looked through first, beside a conversion along rows where there is one, and the tensor is read again.
#include "amsim_i8_convert.h"

namespace amsim {

namespace {

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
// way while the slabs are joined.  Look and conversion of 4096 x 4096 to columns: f32 32 us (150 MB), bf16 23; 784 x 300 f32 9.7.
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
        for (int i = 0; i < U::LOADS; ++i) column_codes<T>(raw[q][i], g.row_factor != nullptr, factor[q][i], multiplier, unit.w[i]);
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

// Slabs of rows that are looked through: enough workgroups for the card beside those that convert rows, few enough for
// every wavefront that converts columns to join them by itself (to quantise the columns of 16384 x 1000 bf16 takes 24.1 us
// with 64 slabs, 28.9 with 32, 29.8 with 256; a training step of 8192 x 512 x 512 62 with 64, 64 with 128).
int64_t slab_rows(int64_t rows, int64_t cols)
{
    const int64_t slabs = std::min(ceil_div64(rows, 64), std::max<int64_t>(16, std::min<int64_t>(64, 128 / ceil_div64(cols, 512))));
    return ceil_div64(rows, slabs);
}

template <typename T, int HOW> void launch_rows_and_look(const I8Rows &rows, unsigned row_blocks, const Look &look, unsigned look_blocks, hipStream_t stream)
{
    const auto kernel = rows.positive || look.positive ? rows_and_look_kernel<T, HOW, true> : rows_and_look_kernel<T, HOW, false>;
    kernel<<<row_blocks + look_blocks, WG, 0, stream>>>(rows, row_blocks, look);
}

}  // namespace

int64_t i8_partial_floats(int64_t rows, int64_t cols) { return ceil_div64(rows, slab_rows(rows, cols)) * 2 * cols; }

int i8_convert(const I8Rows *rows, const I8Columns *columns, float *partial, hipStream_t stream)
{
    if (columns && i8_small(rows, *columns)) return i8_convert_small(rows, *columns, stream);
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
