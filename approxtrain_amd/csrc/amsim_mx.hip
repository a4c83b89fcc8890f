// Conversion of tensors to MXFP4 operands (amsim_mx.h) and back.
//
// Bound by memory: an element is read once, 4 or 2 bytes, and written as 17/32 of a byte for each direction
// asked for.  A training step multiplies the same tensor along either axis, so one pass makes both operands.
// A workgroup owns 128 x 128 values: coalesced loads, LDS, and then each thread takes whole blocks of 32 out
// of it, along a row or down a column, so that the largest magnitude, the scale and the 16 bytes of codes
// are one lane's own affair.  LDS rows are padded by 16 bytes: sixteen rows' 16-byte reads meet all banks.
#include "amsim_mx.h"

namespace amsim {

namespace {

constexpr int WG = 256;
constexpr int TILE = 128;

struct QuantizeArgs {
    const void *x;
    int64_t rows, cols, row_stride;  // row_stride in elements
    uint8_t *by_rows, *by_columns;   // null where that direction is not asked for
    int64_t column_tiles;
    bool vectors;                    // rows start on 16-byte boundaries
};

template <typename T> struct Tile {
    static constexpr int PER_VEC = 16 / sizeof(T);
    static constexpr int STRIDE = TILE + PER_VEC;  // elements of an LDS row
    T v[TILE][STRIDE];
};

template <typename T>
__device__ __forceinline__ void load_tile(Tile<T> &t, const QuantizeArgs &a, int64_t row0, int64_t col0)
{
    constexpr int PER_VEC = Tile<T>::PER_VEC, VECS = TILE / PER_VEC;  // 16-byte pieces of a row of the tile
    constexpr int LOADS = TILE * VECS / WG;
    const T *x = (const T *)a.x;
    if (a.vectors) {
        v4i piece[LOADS];
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int at = threadIdx.x + WG * i, r = at / VECS, c = at % VECS * PER_VEC;
            piece[i] = v4i{0, 0, 0, 0};
            if (row0 + r >= a.rows) continue;
            const T *p = x + (row0 + r) * a.row_stride + col0 + c;
            if (col0 + c + PER_VEC <= a.cols) {
                piece[i] = *(const v4i *)p;
            } else {
                T last[PER_VEC];
#pragma unroll
                for (int e = 0; e < PER_VEC; ++e) last[e] = col0 + c + e < a.cols ? p[e] : (T)0.0f;
                __builtin_memcpy(&piece[i], last, 16);
            }
        }
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int at = threadIdx.x + WG * i, r = at / VECS, c = at % VECS * PER_VEC;
            *(v4i *)&t.v[r][c] = piece[i];
        }
    } else {
        const int c = threadIdx.x % TILE;
#pragma unroll 16
        for (int r = threadIdx.x / TILE; r < TILE; r += WG / TILE)
            t.v[r][c] = row0 + r < a.rows && col0 + c < a.cols ? x[(row0 + r) * a.row_stride + col0 + c] : (T)0.0f;
    }
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
// block `kb` down column `c`
template <typename T> __device__ __forceinline__ MxBlock<T> column_block(const Tile<T> &t, int c, int kb)
{
    MxBlock<T> b;
    T v[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = t.v[32 * kb + i][c];
    __builtin_memcpy(&b, v, sizeof(b));
    return b;
}

// Codes of the tile's 128 rows (or columns), 8 fragments of 16, to the operand; the scales to LDS.
template <typename T, bool COLUMNS>
__device__ __forceinline__ void encode_tile(const Tile<T> &t, uint8_t (&scales)[8][64], uint8_t *codes, int64_t rows,
                                            int64_t row0, int64_t steps, int64_t step)
{
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int f = (threadIdx.x >> 6) + 4 * i, lane = threadIdx.x & 63;
        if (row0 + 16 * f >= rows) continue;
        const MxBlock<T> b = COLUMNS ? column_block(t, 16 * f + lane % 16, lane / 16) : row_block(t, 16 * f + lane % 16, lane / 16);
        const uint32_t code = mx_scale_code(b.exponent_field());
        scales[f][lane] = (uint8_t)code;
        *(v4i *)(codes + (((row0 / 16 + f) * steps + step) * 64 + lane) * 16) = b.encode(code);
    }
}
__device__ __forceinline__ void store_scales(const uint8_t (&scales)[8][64], int i, uint8_t *out, int64_t rows, int64_t row0,
                                             int64_t steps, int64_t step)
{
    const int g = i >> 6, lane = i & 63;
    if (row0 + 64 * g >= rows) return;
    const uint32_t w = scales[4 * g][lane] | scales[4 * g + 1][lane] << 8 | scales[4 * g + 2][lane] << 16 | (uint32_t)scales[4 * g + 3][lane] << 24;
    *(uint32_t *)(out + (((row0 / 64 + g) * steps + step) * 64 + lane) * 4) = w;
}

template <typename T, bool ROWS, bool COLUMNS>
__global__ __launch_bounds__(WG) void quantize_kernel(QuantizeArgs a)
{
    __shared__ Tile<T> t;
    __shared__ uint8_t scales[2][8][64];
    const int64_t row0 = (int64_t)blockIdx.x / a.column_tiles * TILE, col0 = (int64_t)blockIdx.x % a.column_tiles * TILE;
    load_tile(t, a, row0, col0);
    // (scales of fragments that do not exist are not written below; their bytes of a dword that is are zeros)
    for (int i = threadIdx.x; i < (int)sizeof(scales) / 4; i += WG) ((uint32_t *)scales)[i] = 0;
    __syncthreads();
    const int64_t row_steps = mx_steps(a.cols), column_steps = mx_steps(a.rows);
    if (ROWS) encode_tile<T, false>(t, scales[0], a.by_rows, a.rows, row0, row_steps, col0 / TILE);
    if (COLUMNS) encode_tile<T, true>(t, scales[1], a.by_columns, a.cols, col0, column_steps, row0 / TILE);
    __syncthreads();
    const int i = threadIdx.x & 127;
    if (ROWS && threadIdx.x < 128)
        store_scales(scales[0], i, a.by_rows + mx_code_bytes(a.rows, a.cols), a.rows, row0, row_steps, col0 / TILE);
    if (COLUMNS && threadIdx.x >= 128)
        store_scales(scales[1], i, a.by_columns + mx_code_bytes(a.cols, a.rows), a.cols, col0, column_steps, row0 / TILE);
}

template <typename T> void launch_quantize(const QuantizeArgs &a, unsigned tiles, hipStream_t stream)
{
    if (a.by_rows && a.by_columns) quantize_kernel<T, true, true><<<tiles, WG, 0, stream>>>(a);
    else if (a.by_rows) quantize_kernel<T, true, false><<<tiles, WG, 0, stream>>>(a);
    else quantize_kernel<T, false, true><<<tiles, WG, 0, stream>>>(a);
}

// A workgroup reads the 1 KB of a fragment's step and writes 16 rows of 128 values, eight per thread.
template <typename T>
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
    if (col + 8 <= length && length % 8 == 0) {  // (out starts on a 16-byte boundary)
#pragma unroll
        for (int i = 0; i < (int)(8 * sizeof(T) / 16); ++i) ((v4i *)o)[i] = ((const v4i *)v)[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (col + i < length) o[i] = v[i];
    }
}

inline bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

int mx_quantize(const void *x, int dtype, int64_t rows, int64_t cols, int64_t row_stride, void *by_rows, void *by_columns,
                hipStream_t stream)
{
    const int64_t column_tiles = ceil_div64(cols, TILE), tiles = ceil_div64(rows, TILE) * column_tiles;
    if (tiles >= (1ll << 24)) return fail(AMSIM_ERR_UNSUPPORTED, "mxfp4: more tiles than one launch takes");
    QuantizeArgs a{x, rows, cols, row_stride, (uint8_t *)by_rows, (uint8_t *)by_columns, column_tiles,
                   aligned16(x) && (rows == 1 || row_stride * element_bytes(dtype) % 16 == 0)};
    switch (dtype) {
    case AMSIM_DTYPE_F32: launch_quantize<float>(a, (unsigned)tiles, stream); break;
    case AMSIM_DTYPE_BF16: launch_quantize<__bf16>(a, (unsigned)tiles, stream); break;
    default: launch_quantize<_Float16>(a, (unsigned)tiles, stream); break;
    }
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
    return mx_quantize(x, dtype, rows, cols, row_stride, by_rows, by_columns, (hipStream_t)stream);
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
    case AMSIM_DTYPE_F32: dequantize_kernel<float><<<(unsigned)blocks, WG, 0, s>>>(p, rows, length, (float *)out); break;
    case AMSIM_DTYPE_BF16: dequantize_kernel<__bf16><<<(unsigned)blocks, WG, 0, s>>>(p, rows, length, (__bf16 *)out); break;
    default: dequantize_kernel<_Float16><<<(unsigned)blocks, WG, 0, s>>>(p, rows, length, (_Float16 *)out); break;
    }
    AMSIM_HIP_CHECK(hipGetLastError());
    return AMSIM_OK;
}

}  // extern "C"
