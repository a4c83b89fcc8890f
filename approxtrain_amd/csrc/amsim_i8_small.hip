// Conversions to 8-bit operands in one launch, where columns are so short that a workgroup takes 64 of them from top to
// bottom: small training steps are bound by their launches, the host's half of one more than the device's.
#include "amsim_i8_convert.h"

namespace amsim {

namespace {

// maxima or sums over the lanes that hold the same columns of a unit, in every one of them
template <typename Op, typename T> __device__ __forceinline__ float down_unit(float v)
{
    if constexpr (Unit<T>::LANES == 8) v = with_dpp<Op, 0x128>(v);  // the other eight of sixteen
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = Op::of(__uint_as_float(r[0]), __uint_as_float(r[1]));
    const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return Op::of(__uint_as_float(h[0]), __uint_as_float(h[1]));
}

// Its waves' units, two at a time, once for the largest magnitudes and the sums and, beyond 256 rows, again for the codes.
template <typename T, bool MASK> __device__ __forceinline__ void convert_whole_columns(const I8Columns &g, int64_t id, uint32_t *lds)
{
    using U = Unit<T>;
    constexpr int AT_ONCE = 2;
    uint32_t (*corners)[CORNER] = (uint32_t (*)[CORNER])lds;
    float (*most_of)[64] = (float (*)[64])(lds + WAVES * CORNER), (*sum_of)[64] = most_of + WAVES;
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = unit_col<T>();
    const int col0 = (int)id * 64, groups = (int)ceil_div64(g.rows, 16);
    v4i raw[AT_ONCE][U::LOADS];
    float factor[AT_ONCE][U::LOADS];
    auto load = [&](int group) {
#pragma unroll
        for (int h = 0; h < AT_ONCE; ++h) {
            const int row0 = (group + h * WAVES) * 16;
            load_unit<MASK>((const T *)g.x, (const T *)g.positive, g.rows, g.cols, g.row_stride, row0, col0, raw[h]);
#pragma unroll
            for (int i = 0; i < U::LOADS; ++i) {
                const int r = row0 + unit_row<T>(i);
                factor[h][i] = g.row_factor && r < g.rows ? g.row_factor[r] : 1.0f;
            }
        }
    };
    float most[U::N] = {}, sum[U::N] = {};
    int group = wave;
    do {
        load(group);
#pragma unroll
        for (int h = 0; h < AT_ONCE; ++h)
#pragma unroll
            for (int i = 0; i < U::LOADS; ++i) {
                float v[U::N];
                piece_floats<T>(raw[h][i], v);
#pragma unroll
                for (int e = 0; e < U::N; ++e) {
                    sum[e] += v[e];
                    most[e] = MaxOf::of(most[e], __uint_as_float(magnitude_bits(v[e] * factor[h][i])));
                }
            }
        group += AT_ONCE * WAVES;
    } while (group < groups);
#pragma unroll
    for (int e = 0; e < U::N; ++e) most[e] = down_unit<MaxOf, T>(most[e]), sum[e] = down_unit<SumOf, T>(sum[e]);
    if (lane < U::LANES)
#pragma unroll
        for (int e = 0; e < U::N; ++e) most_of[wave][c + e] = most[e], sum_of[wave][c + e] = sum[e];
    __syncthreads();
    if (g.sums && wave == 0 && col0 + lane < g.cols) {
        float s = sum_of[0][lane];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) s += sum_of[w][lane];
        store_from_float(g.sums, g.sums_dtype, col0 + lane, s);
    }
    if (!g.by_rows && !g.by_columns) return;
    float multiplier[U::N];
#pragma unroll
    for (int e = 0; e < U::N; ++e) {
        float m = most_of[0][c + e];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) m = MaxOf::of(m, most_of[w][c + e]);
        multiplier[e] = q8_multiplier(__float_as_uint(m));
        if (wave == 0 && lane < U::LANES && col0 + c + e < g.cols) g.scales[col0 + c + e] = q8_scale(__float_as_uint(m));
    }
    const bool again = groups > AT_ONCE * WAVES;
    for (group = wave; group < groups; group += AT_ONCE * WAVES) {
        if (again) load(group);
#pragma unroll
        for (int h = 0; h < AT_ONCE; ++h) {
            if (group + h * WAVES >= groups) break;
            Codes<U::N> unit;
#pragma unroll
            for (int i = 0; i < U::LOADS; ++i) column_codes<T>(raw[h][i], g.row_factor != nullptr, factor[h][i], multiplier, unit.w[i]);
            store_unit<T>(unit, corners[wave], g.rows, g.cols, (group + h * WAVES) * 16, col0, g.by_rows, g.by_columns);
        }
    }
}

// Rows' type T, converted as HOW says (NO_ROWS: not at all), beside columns of type C.
constexpr int NO_ROWS = 100;
template <typename T, int HOW, bool MASK, typename C> __global__ __launch_bounds__(WG, 4) void small_kernel(I8Rows rows, unsigned row_blocks, I8Columns columns)
{
    __shared__ __attribute__((aligned(16))) uint32_t lds[WAVES * (CORNER + 16) + WAVES * 4 * 64];
    static_assert(sizeof(lds) >= 4 * WAVES * (CORNER + 128), "");
    if (blockIdx.x >= row_blocks) return convert_whole_columns<C, MASK>(columns, blockIdx.x - row_blocks, lds);
    if constexpr (HOW == LANES_64) convert_single_rows<T, 64, 16, MASK>(rows, (float *)lds);
    else if constexpr (HOW == LANES_512) convert_single_rows<T, 512, 8, MASK>(rows, (float *)lds);
    else if constexpr (HOW != NO_ROWS) convert_rows<T, HOW, MASK>(rows, lds);
}

template <typename T, typename C> int launch(const I8Rows *rows, const I8Columns &columns, hipStream_t stream)
{
    const I8Rows j = rows ? *rows : I8Rows{};
    const unsigned column_blocks = (unsigned)i8_steps(columns.cols);
    unsigned row_blocks = rows ? (unsigned)ceil_div64(j.rows, 16) : 0;
    auto start = [&](auto how) {
        constexpr int HOW = decltype(how)::value;
        const auto kernel = columns.positive ? small_kernel<T, HOW, true, C> : small_kernel<T, HOW, false, C>;
        kernel<<<row_blocks + column_blocks, WG, 0, stream>>>(j, row_blocks, columns);
    };
    const int64_t each = ceil_div64(i8_steps(j.cols), WAVES);
    if (!rows) {
        start(std::integral_constant<int, NO_ROWS>{});
    } else if (single_rows(j)) {
        row_blocks *= j.cols <= 1024 ? 2 : 16;
        if (j.cols <= 1024) start(std::integral_constant<int, LANES_64>{});
        else start(std::integral_constant<int, LANES_512>{});
    } else if (each <= 1) {
        start(std::integral_constant<int, 1>{});
    } else if (each == 2) {
        start(std::integral_constant<int, 2>{});
    } else {
        start(std::integral_constant<int, 4>{});
    }
    AMSIM_HIP_CHECK(hipGetLastError());
    return AMSIM_OK;
}

}  // namespace

// us of a call so, and in two launches, calls in a row: gradients of a 128 x 784 x 300 layer 10.2 and 15.7, a training step of 64 x 100 x
// 100 21 and 32, of 256 x 512 x 512 24 and 32, columns of 512 x 512 bf16 8.1 and 9.5, of 250 x 8000 f32 6.2 and 10.0; but of 784 x 300
// 11.7 and 9.7, the forward pass of 128 x 784 x 300 18.2 and 16.5, columns of 1000 x 250 15.7 and 11.0: few workgroups read long columns
// twice.  Up to 2^18 values they take one launch all the same: a training step of such layers waits for the host, which saves
// 2.5 us with it.  (A captured step does not wait so, and is 2 to 5 us slower for it.)
bool i8_small(const I8Rows *rows, const I8Columns &columns)
{
    if (columns.rows > 512 && (columns.rows > 1024 || columns.rows * columns.cols > 1 << 18)) return false;
    if (!rows) return i8_steps(columns.cols) < MOST_BLOCKS;
    // (either type beside 32 bits, or one type; rows of either kind that the kernels above hold)
    if (columns.dtype != AMSIM_DTYPE_F32 && columns.dtype != rows->dtype) return false;
    return rows->cols <= (single_rows(*rows) ? 4096 : 2048) && ceil_div64(rows->rows, 16) * 16 + i8_steps(columns.cols) < MOST_BLOCKS;
}

int i8_convert_small(const I8Rows *rows, const I8Columns &columns, hipStream_t stream)
{
    return with_type(rows ? rows->dtype : columns.dtype, [&](auto zero) {
        using T = decltype(zero);
        return columns.dtype == AMSIM_DTYPE_F32 ? launch<T, float>(rows, columns, stream) : launch<T, T>(rows, columns, stream);
    });
}

}  // namespace amsim
