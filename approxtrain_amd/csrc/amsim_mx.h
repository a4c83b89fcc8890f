// MXFP4 operands: storage, element codes and the conversions that the kernels of the 4-bit products share.
//
// A tensor of `rows` x `length` values has one scale for every 32 consecutive values of a row (the length is
// the reduction axis of a product).  With E the exponent field of the block's largest magnitude the scale's
// code is max(E - 2, 0) and stands for 2^(code - 127); the elements are x / scale, rounded to the nearest of
// +-{0, 0.5, 1, 1.5, 2, 3, 4, 6}, ties to the even code, saturated at 6.  A block that holds an infinity or
// a NaN has the scale code 255 and reads back as NaN.
//
// Storage follows the operands of the 16x16x128 matrix instruction, so that a wavefront's loads are whole
// lines wherever they come from, and no kernel has an edge in its loads but for the last fragment of rows:
//   codes   [rows / 16][length / 128][64 lanes][16 bytes]   lane = 16 * (block of 32 within the 128) + row % 16
//   scales  [rows / 64][length / 128][64 lanes][4 bytes]    byte = (row / 16) % 4
// with extents rounded up, the scales right behind the codes.  Values beyond the length are zeros, and so are rows
// beyond the last one and their scales: equal values are equal bytes.
#ifndef AMSIM_MX_H_
#define AMSIM_MX_H_

#include "amsim_internal.h"

namespace amsim {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v2i __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef unsigned short v2us __attribute__((ext_vector_type(2)));

// 16 bytes at any element's address: rows need not start on 16-byte boundaries, the hardware takes such pieces too
typedef int v4i_anywhere __attribute__((ext_vector_type(4), aligned(2)));
__device__ __forceinline__ v4i load16(const void *p) { return *(const v4i_anywhere *)p; }
__device__ __forceinline__ void store16(void *p, v4i v) { *(v4i_anywhere *)p = v; }

__host__ __device__ inline int64_t ceil_div64(int64_t a, int64_t b) { return (a + b - 1) / b; }
// steps of 128 along the reduction
__host__ __device__ inline int64_t mx_steps(int64_t length) { return ceil_div64(length, 128); }
__host__ __device__ inline int64_t mx_code_bytes(int64_t rows, int64_t length) { return ceil_div64(rows, 16) * mx_steps(length) * 1024; }
__host__ __device__ inline int64_t mx_scale_bytes(int64_t rows, int64_t length) { return ceil_div64(rows, 64) * mx_steps(length) * 256; }

// extents for which every byte offset and launch extent used by the kernels fits
inline bool mx_extents_fit(int64_t rows, int64_t length)
{
    return rows >= 0 && length >= 0 && rows < (1ll << 31) && length < (1ll << 31) && (double)rows * (double)length <= 35184372088832.0;
}

// Whether a tensor of so many bytes is read for conversion, or written, past the last-level cache: it would not be there when
// it is read next, and keeps out what is.  In 16 bits, past the cache and through it, us:
//   16384 x 8192 (256 MB)  by rows 57 and 61, both ways 67 and 74; back 47 and 74, and converted again 104 and 147
//                          product of a reduction of 8192 483 and 530, of 1024 97 and 98, and converted 153 and 191
//   14336 x 8192 (224 MB)  product 82 and 87, and converted 134 and 133, and copied 175 and 190
//   208 MB                 product 78 and 81, and converted 126 and 122
//   160 MB                 back 30 and 32, and converted 67 and 62
//   64 MB                  product 30 and 29, and converted 47 and 43
inline bool mx_goes_around(double bytes) { return bytes >= 224 << 20; }

inline int element_bytes(int dtype) { return dtype == AMSIM_DTYPE_F32 ? 4 : 2; }
inline bool known_dtype(int dtype) { return dtype == AMSIM_DTYPE_F32 || dtype == AMSIM_DTYPE_BF16 || dtype == AMSIM_DTYPE_F16; }

__device__ __forceinline__ uint32_t mx_scale_code(uint32_t exponent_field)
{
    return exponent_field >= 255u ? 255u : exponent_field > 2u ? exponent_field - 2u : 0u;
}
// the scale as a float: 2^(code - 127), NaN for 255
__device__ __forceinline__ float mx_scale_value(uint32_t code)
{
    return __uint_as_float(code == 255u ? 0x7fc00000u : code ? code << 23 : 0x00400000u);
}

// 32 values of one block in registers, as they lie in memory
template <typename T> struct MxBlock;

template <> struct MxBlock<float> {
    float v[32];
    __device__ __forceinline__ uint32_t exponent_field() const
    {
        uint32_t m[4] = {0, 0, 0, 0};  // (as whole numbers: a NaN's bits are above all others')
#pragma unroll
        for (int i = 0; i < 32; ++i) m[i % 4] = max(m[i % 4], __float_as_uint(v[i]) & 0x7fffffffu);
        return max(max(m[0], m[1]), max(m[2], m[3])) >> 23;
    }
    __device__ __forceinline__ v4i encode(uint32_t code) const
    {
        const float s = mx_scale_value(code == 255u ? 127u : code);
        v4i r;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            uint32_t w = 0;
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[8 * d], v[8 * d + 1], s, 0);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[8 * d + 2], v[8 * d + 3], s, 1);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[8 * d + 4], v[8 * d + 5], s, 2);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[8 * d + 6], v[8 * d + 7], s, 3);
            r[d] = code == 255u ? 0 : (int)w;
        }
        return r;
    }
};

template <typename T> struct MxBlock16 {
    uint32_t v[16];  // pairs, the lower index in the lower half
    __device__ __forceinline__ uint32_t largest_bits() const
    {
        v2us m = {0, 0};
#pragma unroll
        for (int i = 0; i < 16; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(v2us, v[i] & 0x7fff7fffu));
        return max((uint32_t)m.x, (uint32_t)m.y);
    }
};
template <> struct MxBlock<__bf16> : MxBlock16<__bf16> {
    __device__ __forceinline__ uint32_t exponent_field() const { return largest_bits() >> 7; }
    __device__ __forceinline__ v4i encode(uint32_t code) const
    {
        const float s = mx_scale_value(code == 255u ? 127u : code);
        v4i r;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            uint32_t w = 0;
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(v2bf, v[4 * d]), s, 0);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(v2bf, v[4 * d + 1]), s, 1);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(v2bf, v[4 * d + 2]), s, 2);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(v2bf, v[4 * d + 3]), s, 3);
            r[d] = code == 255u ? 0 : (int)w;
        }
        return r;
    }
};
template <> struct MxBlock<_Float16> : MxBlock16<_Float16> {
    __device__ __forceinline__ uint32_t exponent_field() const
    {
        return __float_as_uint((float)__builtin_bit_cast(_Float16, (unsigned short)largest_bits())) >> 23;
    }
    __device__ __forceinline__ v4i encode(uint32_t code) const
    {
        const float s = mx_scale_value(code == 255u ? 127u : code);
        v4i r;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            uint32_t w = 0;
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(v2h, v[4 * d]), s, 0);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(v2h, v[4 * d + 1]), s, 1);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(v2h, v[4 * d + 2]), s, 2);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(v2h, v[4 * d + 3]), s, 3);
            r[d] = code == 255u ? 0 : (int)w;
        }
        return r;
    }
};

// the same for 8 values: the exponent field of their largest magnitude, and their codes
__device__ __forceinline__ uint32_t mx_exponent_field(const float (&v)[8])
{
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    return m >> 23;
}
template <typename T> __device__ __forceinline__ uint32_t mx_largest16(const T (&v)[8])
{
    uint32_t p[4];
    __builtin_memcpy(p, v, 16);
    v2us m = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(v2us, p[i] & 0x7fff7fffu));
    return max((uint32_t)m.x, (uint32_t)m.y);
}
__device__ __forceinline__ uint32_t mx_exponent_field(const __bf16 (&v)[8]) { return mx_largest16(v) >> 7; }
__device__ __forceinline__ uint32_t mx_exponent_field(const _Float16 (&v)[8])
{
    return __float_as_uint((float)__builtin_bit_cast(_Float16, (unsigned short)mx_largest16(v))) >> 23;
}
__device__ __forceinline__ uint32_t mx_encode8(const float (&v)[8], uint32_t code)
{
    const float s = mx_scale_value(code == 255u ? 127u : code);
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], s, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], s, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], s, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], s, 3);
    return code == 255u ? 0 : w;
}
__device__ __forceinline__ uint32_t mx_encode8(const __bf16 (&v)[8], uint32_t code)
{
    const float s = mx_scale_value(code == 255u ? 127u : code);
    v2bf p[4];
    __builtin_memcpy(p, v, 16);
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, p[0], s, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, p[1], s, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, p[2], s, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, p[3], s, 3);
    return code == 255u ? 0 : w;
}
__device__ __forceinline__ uint32_t mx_encode8(const _Float16 (&v)[8], uint32_t code)
{
    const float s = mx_scale_value(code == 255u ? 127u : code);
    v2h p[4];
    __builtin_memcpy(p, v, 16);
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, p[0], s, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, p[1], s, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, p[2], s, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, p[3], s, 3);
    return code == 255u ? 0 : w;
}

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__bf16 v) { return (float)v; }
__device__ __forceinline__ float to_float(_Float16 v) { return (float)v; }
template <typename T> __device__ __forceinline__ T from_float(float v) { return (T)v; }

// an element of a vector whose type is known at run time only (biases)
__device__ __forceinline__ float load_as_float(const void *p, int dtype, int64_t i)
{
    if (dtype == AMSIM_DTYPE_F32) return ((const float *)p)[i];
    if (dtype == AMSIM_DTYPE_BF16) return (float)((const __bf16 *)p)[i];
    return (float)((const _Float16 *)p)[i];
}

// (a NaN stays one)
__device__ __forceinline__ float activate(float v, int act) { return act == AMSIM_ACT_RELU && v < 0.0f ? 0.0f : v; }

// A tensor to be converted: the operand of its rows, of its columns, or both.
struct MxConversion {
    const void *x;
    const void *positive;            // [rows][cols] of x's type, or null: where it is not above zero x counts as zero
    int dtype;
    int64_t rows, cols, row_stride;  // row_stride in elements
    uint8_t *by_rows, *by_columns;   // null where that direction is not asked for
    float *sums;                     // [ceil(rows / 32)][cols], or null: sums of every 32 rows
};
// One launch for one or two tensors.
int mx_convert(const MxConversion *jobs, int count, hipStream_t stream);

}  // namespace amsim

// For tests: how the products of one call would run, one (m, n, k) or the two of a backward pass, (m, k, n) and (k, n, m).
// info = {rows and columns of the tiles, splits of either's reduction: 0 where one workgroup's waves share it}.
extern "C" int amsim_mxfp4_plan(int count, const int64_t *extents, int64_t *info);
#endif  // AMSIM_MX_H_
