// Conversion of tensors to MXFP4 operands (amsim_mx.h) and back.
//
// Rows may start on any element: pieces of 16 bytes that cross two lines cost less than elements one by one (3616 x
// 3762 in 16 bits, both directions and back: 29 us against 50).
// Bound by memory: an element is read once, 4 or 2 bytes, and written as 17/32 of a byte for each direction
// asked for.  A training step multiplies the same tensor along either axis, so one pass makes both operands, and
// of a gradient also the sums of its columns.
#include "amsim_mx.h"

namespace amsim {

namespace {

constexpr int WG = 256;

// (AROUND: see mx_goes_around)
template <bool AROUND> __device__ __forceinline__ v4i load_piece(const void *p)
{
    return AROUND ? __builtin_nontemporal_load((const v4i_anywhere *)p) : load16(p);
}

// ---- rows alone: four lanes share a block, and nothing has to be exchanged but its largest magnitude --------

template <typename T> struct Eighth;  // 8 values of a block
template <> struct Eighth<float> { float v[8]; };
template <> struct Eighth<__bf16> { __bf16 v[8]; };
template <> struct Eighth<_Float16> { _Float16 v[8]; };

// A workgroup: 64 rows of a step of 128.  A wavefront's 64 lanes read four rows, 128 values of each; the scales of
// the four fragments meet in LDS, as the bytes of one dword.
template <typename T, bool AROUND>
__global__ __launch_bounds__(WG) void rows_kernel(const T *x, int64_t rows, int64_t cols, int64_t row_stride, uint8_t *out)
{
    __shared__ uint8_t scales[4][64];
    const int64_t steps = mx_steps(cols), step = (int64_t)blockIdx.x % steps, row0 = (int64_t)blockIdx.x / steps * 64;
    const int r = threadIdx.x / 16, c = threadIdx.x % 16 * 8, lane = c / 32 * 16 + r;  // of a fragment
    const int64_t col = 128 * step + c;
    Eighth<T> e[4];
#pragma unroll
    for (int f = 0; f < 4; ++f) {
        const int64_t row = row0 + 16 * f + r;
        const T *p = x + row * row_stride + col;
        if (row < rows && col + 8 <= cols) {
            v4i piece[sizeof(e[f]) / 16];
#pragma unroll
            for (int i = 0; i < (int)(sizeof(e[f]) / 16); ++i) piece[i] = load_piece<AROUND>((const char *)p + 16 * i);
            __builtin_memcpy(&e[f], piece, sizeof(e[f]));
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) e[f].v[i] = row < rows && col + i < cols ? p[i] : (T)0.0f;
        }
    }
#pragma unroll
    for (int f = 0; f < 4; ++f) {
        uint32_t largest = mx_exponent_field(e[f].v);
        largest = max(largest, (uint32_t)__shfl_xor((int)largest, 1, 64));
        largest = max(largest, (uint32_t)__shfl_xor((int)largest, 2, 64));
        const uint32_t code = mx_scale_code(largest);
        if (threadIdx.x % 4 == 0) scales[f][lane] = (uint8_t)code;
        if (row0 + 16 * f < rows)
            *(uint32_t *)(out + (((row0 / 16 + f) * steps + step) * 64 + lane) * 16 + c % 32 / 2) = mx_encode8(e[f].v, code);
    }
    __syncthreads();
    if (threadIdx.x >= 64) return;
    const int l = threadIdx.x;
    const uint32_t w = scales[0][l] | scales[1][l] << 8 | scales[2][l] << 16 | (uint32_t)scales[3][l] << 24;
    *(uint32_t *)(out + mx_code_bytes(rows, cols) + ((row0 / 64 * steps + step) * 64 + l) * 4) = w;
}

// ---- columns, or rows and columns ---------------------------------------------------------------------------
// A workgroup owns 32 x 128 values, in LDS: of the 256 blocks of 32 along the rows and down the columns each
// thread takes one, so that the largest magnitude, the scale and the 16 bytes of codes are its own affair.  LDS
// rows are padded by 16 bytes: sixteen rows' 16-byte reads meet all banks.

constexpr int HIGH = 32, WIDE = 128;

struct TileJobs {
    MxConversion job[2];
    int64_t tiles[2], column_tiles[2];
};

template <typename T> struct Tile {
    static constexpr int PER_VEC = 16 / sizeof(T);
    static constexpr int STRIDE = WIDE + PER_VEC;  // elements of an LDS row
    T v[HIGH][STRIDE];
};

template <typename T> __device__ __forceinline__ T masked(T v, T y) { return to_float(y) > 0.0f ? v : (T)0.0f; }

template <bool AROUND, typename T>
__device__ __forceinline__ void load_tile(Tile<T> &t, const MxConversion &j, int64_t row0, int64_t col0)
{
    constexpr int PER_VEC = Tile<T>::PER_VEC, VECS = WIDE / PER_VEC;  // 16-byte pieces of a row of the tile
    constexpr int LOADS = HIGH * VECS / WG;
    const T *x = (const T *)j.x, *y = (const T *)j.positive;
    v4i piece[LOADS], keep[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int at = threadIdx.x + WG * i, r = at / VECS, c = at % VECS * PER_VEC;
        piece[i] = v4i{0, 0, 0, 0};
        if (row0 + r >= j.rows) continue;
        const T *p = x + (row0 + r) * j.row_stride + col0 + c, *q = y + (row0 + r) * j.cols + col0 + c;
        if (col0 + c + PER_VEC <= j.cols) {
            piece[i] = load_piece<AROUND>(p);
            if (y) keep[i] = load16(q);
        } else {
            T last[PER_VEC], also[PER_VEC];
#pragma unroll
            for (int e = 0; e < PER_VEC; ++e) {
                last[e] = col0 + c + e < j.cols ? p[e] : (T)0.0f;
                also[e] = y && col0 + c + e < j.cols ? q[e] : (T)0.0f;
            }
            __builtin_memcpy(&piece[i], last, 16);
            __builtin_memcpy(&keep[i], also, 16);
        }
    }
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int at = threadIdx.x + WG * i, r = at / VECS, c = at % VECS * PER_VEC;
        if (y) {
            T a[PER_VEC], b[PER_VEC];
            __builtin_memcpy(a, &piece[i], 16);
            __builtin_memcpy(b, &keep[i], 16);
#pragma unroll
            for (int e = 0; e < PER_VEC; ++e) a[e] = masked(a[e], b[e]);
            __builtin_memcpy(&piece[i], a, 16);
        }
        *(v4i *)&t.v[r][c] = piece[i];
    }
}

// The scale of a block of fragment `f`, a byte of its group's dword; behind the last fragment the group's other bytes are zeros.
__device__ __forceinline__ void store_scale(uint8_t *scales, int64_t rows, int64_t f, int64_t steps, int64_t step, int lane, uint32_t code)
{
    uint8_t *to = scales + ((f / 4 * steps + step) * 64 + lane) * 4;
    to[f % 4] = (uint8_t)code;
    if (16 * (f + 1) >= rows)
        for (int i = (int)(f % 4) + 1; i < 4; ++i) to[i] = 0;
}

// block `kb` of row `r` of the tile
template <typename T> __device__ __forceinline__ MxBlock<T> row_block(const Tile<T> &t, int r, int kb)
{
    MxBlock<T> b;
    constexpr int PIECES = 32 * sizeof(T) / 16;
    v4i piece[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) piece[i] = *(const v4i *)&t.v[r][32 * kb + i * Tile<T>::PER_VEC];
    __builtin_memcpy(&b, piece, sizeof(b));
    return b;
}

template <typename T, bool AROUND> __device__ __forceinline__ void convert_tile(const MxConversion &j, int64_t row_tile, int64_t column_tile, uint8_t *lds)
{
    Tile<T> &t = *(Tile<T> *)lds;
    const int64_t row0 = row_tile * HIGH, col0 = column_tile * WIDE;
    load_tile<AROUND>(t, j, row0, col0);
    __syncthreads();
    if (threadIdx.x < 128) {  // two fragments of 16 rows
        const int lane = threadIdx.x & 63;
        const int64_t f = row0 / 16 + threadIdx.x / 64, steps = mx_steps(j.cols), step = column_tile;
        if (!j.by_rows || 16 * f >= j.rows) return;
        const MxBlock<T> b = row_block(t, threadIdx.x / 64 * 16 + lane % 16, lane / 16);
        const uint32_t code = mx_scale_code(b.exponent_field());
        *(v4i *)(j.by_rows + ((f * steps + step) * 64 + lane) * 16) = b.encode(code);
        store_scale(j.by_rows + mx_code_bytes(j.rows, j.cols), j.rows, f, steps, step, lane, code);
    } else {  // eight fragments of 16 columns, a quarter of a step of each
        const int c = threadIdx.x - 128;
        const int64_t f = col0 / 16 + c / 16, steps = mx_steps(j.rows), step = row0 / 128;
        const int lane = (int)(row0 / 32 % 4) * 16 + c % 16;
        if (16 * f >= j.cols) return;
        T v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = t.v[i][c];
        if (j.by_columns) {
            MxBlock<T> b;
            __builtin_memcpy(&b, v, sizeof(b));
            const uint32_t code = mx_scale_code(b.exponent_field());
            *(v4i *)(j.by_columns + ((f * steps + step) * 64 + lane) * 16) = b.encode(code);
            store_scale(j.by_columns + mx_code_bytes(j.cols, j.rows), j.cols, f, steps, step, lane, code);
        }
        if (j.sums && row0 < j.rows && col0 + c < j.cols) {
            float s[4] = {};  // (four chains: fewer roundings in each)
#pragma unroll
            for (int i = 0; i < 32; ++i) s[i % 4] += to_float(v[i]);
            j.sums[row_tile * j.cols + col0 + c] = (s[0] + s[1]) + (s[2] + s[3]);
        }
    }
}

// (types are branched on here: the two tensors of a forward pass may differ in theirs, and share a launch)
template <bool AROUND>
__global__ __launch_bounds__(WG) void tiles_kernel(TileJobs jobs)
{
    __shared__ __attribute__((aligned(16))) uint8_t lds[sizeof(Tile<float>)];
    const int which = (int64_t)blockIdx.x >= jobs.tiles[0];
    const MxConversion &j = jobs.job[which];
    const int64_t tile = (int64_t)blockIdx.x - (which ? jobs.tiles[0] : 0), columns = jobs.column_tiles[which];
    if (j.dtype == AMSIM_DTYPE_F32) convert_tile<float, AROUND>(j, tile / columns, tile % columns, lds);
    else if (j.dtype == AMSIM_DTYPE_BF16) convert_tile<__bf16, AROUND>(j, tile / columns, tile % columns, lds);
    else convert_tile<_Float16, AROUND>(j, tile / columns, tile % columns, lds);
}

inline bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

// A workgroup reads the 1 KB of a fragment's step and writes 16 rows of 128 values, eight per thread.
template <typename T, bool AROUND>
__global__ __launch_bounds__(WG) void dequantize_kernel(const uint8_t *q, int64_t rows, int64_t length, T *out)
{
    const int64_t steps = mx_steps(length), f = (int64_t)blockIdx.x / steps, step = (int64_t)blockIdx.x % steps;
    const int r = threadIdx.x / 16, c = threadIdx.x % 16 * 8, lane = c / 32 * 16 + r;
    const int64_t row = 16 * f + r, col = 128 * step + c;
    if (row >= rows || col >= length) return;
    const uint32_t w = *(const uint32_t *)(q + ((f * steps + step) * 64 + lane) * 16 + c % 32 / 2);
    const float s = mx_scale_value(q[mx_code_bytes(rows, length) + ((f / 4 * steps + step) * 64 + lane) * 4 + f % 4]);
    T v[8];
    v2f p;
    p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0); v[0] = from_float<T>(p.x * s); v[1] = from_float<T>(p.y * s);
    p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1); v[2] = from_float<T>(p.x * s); v[3] = from_float<T>(p.y * s);
    p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2); v[4] = from_float<T>(p.x * s); v[5] = from_float<T>(p.y * s);
    p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3); v[6] = from_float<T>(p.x * s); v[7] = from_float<T>(p.y * s);
    T *o = out + row * length + col;
    if (col + 8 <= length) {
        v4i piece[sizeof(v) / 16];
        __builtin_memcpy(piece, v, sizeof(v));
#pragma unroll
        for (int i = 0; i < (int)(sizeof(v) / 16); ++i) {
            v4i_anywhere *to = (v4i_anywhere *)((char *)o + 16 * i);
            if (AROUND) __builtin_nontemporal_store(piece[i], to);
            else *to = piece[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (col + i < length) o[i] = v[i];
    }
}

template <typename T> void launch_rows(const MxConversion &j, unsigned blocks, hipStream_t stream)
{
    const auto kernel = mx_goes_around((double)j.rows * (double)j.cols * sizeof(T)) ? rows_kernel<T, true> : rows_kernel<T, false>;
    kernel<<<blocks, WG, 0, stream>>>((const T *)j.x, j.rows, j.cols, j.row_stride, j.by_rows);
}
template <typename T> void launch_dequantize(const uint8_t *q, int64_t rows, int64_t length, void *out, unsigned blocks, hipStream_t stream)
{
    const auto kernel = mx_goes_around((double)rows * (double)length * sizeof(T)) ? dequantize_kernel<T, true> : dequantize_kernel<T, false>;
    kernel<<<blocks, WG, 0, stream>>>(q, rows, length, (T *)out);
}

}  // namespace

int mx_convert(const MxConversion *jobs, int count, hipStream_t stream)
{
    if (count == 1 && jobs[0].by_rows && !jobs[0].by_columns && !jobs[0].positive && !jobs[0].sums) {
        const MxConversion &j = jobs[0];
        const int64_t blocks = mx_steps(j.cols) * ceil_div64(j.rows, 64);
        if (blocks >= (1ll << 24)) return fail(AMSIM_ERR_UNSUPPORTED, "mxfp4: more tiles than one launch takes");
        switch (j.dtype) {
        case AMSIM_DTYPE_F32: launch_rows<float>(j, (unsigned)blocks, stream); break;
        case AMSIM_DTYPE_BF16: launch_rows<__bf16>(j, (unsigned)blocks, stream); break;
        default: launch_rows<_Float16>(j, (unsigned)blocks, stream); break;
        }
        AMSIM_HIP_CHECK(hipGetLastError());
        return AMSIM_OK;
    }
    TileJobs t{};
    int64_t tiles = 0;
    double bytes = 0;
    for (int i = 0; i < count; ++i) {
        const MxConversion &j = jobs[i];
        t.job[i] = j;
        t.column_tiles[i] = ceil_div64(j.cols, WIDE);
        // (down the columns the last step is filled up with zeros)
        const int64_t row_tiles = j.by_columns ? mx_steps(j.rows) * (128 / HIGH) : ceil_div64(j.rows, HIGH);
        tiles += t.tiles[i] = row_tiles * t.column_tiles[i];
        bytes += (double)j.rows * (double)j.cols * element_bytes(j.dtype);
    }
    if (tiles >= (1ll << 24)) return fail(AMSIM_ERR_UNSUPPORTED, "mxfp4: more tiles than one launch takes");
    const auto kernel = mx_goes_around(bytes) ? tiles_kernel<true> : tiles_kernel<false>;
    kernel<<<(unsigned)tiles, WG, 0, stream>>>(t);
    AMSIM_HIP_CHECK(hipGetLastError());
    return AMSIM_OK;
}

}  // namespace amsim

using namespace amsim;

extern "C" {

size_t amsim_mxfp4_operand_workspace_bytes(int64_t rows, int64_t length)
{
    return mx_extents_fit(rows, length) ? (size_t)(mx_code_bytes(rows, length) + mx_scale_bytes(rows, length)) : 0;
}

int amsim_mxfp4_quantize(const void *x, int dtype, int64_t rows, int64_t cols, int64_t row_stride, void *by_rows,
                         void *by_columns, void *stream)
{
    if (!known_dtype(dtype)) return fail(AMSIM_ERR_INVALID, "mxfp4: unknown element type");
    if (!mx_extents_fit(rows, cols)) return fail(AMSIM_ERR_UNSUPPORTED, "mxfp4: extents out of range");
    if (rows == 0 || cols == 0) return fail(AMSIM_ERR_INVALID, "mxfp4: empty tensor");
    if (row_stride < cols && rows > 1) return fail(AMSIM_ERR_INVALID, "mxfp4: rows overlap");
    if (!by_rows && !by_columns) return fail(AMSIM_ERR_INVALID, "mxfp4: no direction asked for");
    if (!x) return fail(AMSIM_ERR_INVALID, "mxfp4: null pointer");
    if (!aligned16(by_rows) || !aligned16(by_columns) || ((uintptr_t)x & (element_bytes(dtype) - 1)))
        return fail(AMSIM_ERR_INVALID, "mxfp4: misaligned pointer");
    const MxConversion job{x, nullptr, dtype, rows, cols, row_stride, (uint8_t *)by_rows, (uint8_t *)by_columns, nullptr};
    return mx_convert(&job, 1, (hipStream_t)stream);
}

int amsim_mxfp4_dequantize(const void *q, int64_t rows, int64_t length, int dtype, void *out, void *stream)
{
    if (!known_dtype(dtype)) return fail(AMSIM_ERR_INVALID, "mxfp4: unknown element type");
    if (!mx_extents_fit(rows, length)) return fail(AMSIM_ERR_UNSUPPORTED, "mxfp4: extents out of range");
    if (rows == 0 || length == 0) return fail(AMSIM_ERR_INVALID, "mxfp4: empty tensor");
    if (!q || !out) return fail(AMSIM_ERR_INVALID, "mxfp4: null pointer");
    if (!aligned16(q) || !aligned16(out)) return fail(AMSIM_ERR_INVALID, "mxfp4: misaligned pointer");
    const int64_t blocks = ceil_div64(rows, 16) * mx_steps(length);
    if (blocks >= (1ll << 24)) return fail(AMSIM_ERR_UNSUPPORTED, "mxfp4: more tiles than one launch takes");
    hipStream_t s = (hipStream_t)stream;
    const uint8_t *p = (const uint8_t *)q;
    switch (dtype) {
    case AMSIM_DTYPE_F32: launch_dequantize<float>(p, rows, length, out, (unsigned)blocks, s); break;
    case AMSIM_DTYPE_BF16: launch_dequantize<__bf16>(p, rows, length, out, (unsigned)blocks, s); break;
    default: launch_dequantize<_Float16>(p, rows, length, out, (unsigned)blocks, s); break;
    }
    AMSIM_HIP_CHECK(hipGetLastError());
    return AMSIM_OK;
}

}  // extern "C"
