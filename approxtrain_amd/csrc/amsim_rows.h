// What the kernels that go over rows share: pieces of 16 bytes as 32-bit floats, sums and maxima over the lanes that
// hold a row, and rows as 8-bit integers with a scale each.
//
// Eight bits (Q): with a = max(|v|, 2^-119) over the row, r = 127 / a and the scale s = a / 127, either rounded to 32 bits
// once, a value's code is the integer nearest to the exact product v r, ties to even; it stands for code * s.  The largest
// magnitude has the code 127: a r lies within 127 (1 +- 2^-24).  (2^-119: 127 / a stays finite, and a / 127 normal.)  A row
// that holds an infinity or a NaN has the scale NaN.
#ifndef AMSIM_ROWS_H_
#define AMSIM_ROWS_H_

#include "amsim_mx.h"

namespace amsim {

constexpr uint32_t Q8_SMALLEST = (uint32_t)(127 - 119) << 23;  // 2^-119

// of the largest magnitude's bits: what values are multiplied by, and the scale
__device__ __forceinline__ float q8_multiplier(uint32_t largest)
{
    return largest >= 0x7f800000u ? 0.0f : 127.0f / __uint_as_float(max(largest, Q8_SMALLEST));
}
__device__ __forceinline__ float q8_scale(uint32_t largest)
{
    return largest >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : __uint_as_float(max(largest, Q8_SMALLEST)) / 127.0f;
}
__device__ __forceinline__ uint32_t magnitude_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// The code of one value in the lowest byte: within 1.5 * 2^23 +- 2^22 a float's last place is 1, so that the sum's one
// rounding, behind the exact product, is the rounding to an integer.
__device__ __forceinline__ uint32_t q8_code(float v, float r) { return __float_as_uint(__builtin_fmaf(v, r, 12582912.0f)); }
// the lowest bytes of four
__device__ __forceinline__ uint32_t q8_pack(uint32_t a, uint32_t b, uint32_t c, uint32_t d)
{
    return __builtin_amdgcn_perm(b, a, 0x0c0c0400u) | __builtin_amdgcn_perm(d, c, 0x04000c0cu);
}
__device__ __forceinline__ uint32_t q8_codes4(float a, float b, float c, float d, float r)
{
    return q8_pack(q8_code(a, r), q8_code(b, r), q8_code(c, r), q8_code(d, r));
}
__device__ __forceinline__ float q8_value(uint32_t codes, int i, float s) { return (float)(int8_t)(codes >> 8 * i) * s; }

// ---- rows kept in 8 bits: codes [rows][pitch], then a scale for each row ------------------------------------------
__host__ __device__ inline int64_t kept8_pitch(int64_t cols) { return ceil_div64(cols, 16) * 16; }
inline int64_t kept8_bytes(int64_t rows, int64_t cols) { return rows * (kept8_pitch(cols) + 4); }

// ---- pieces of 16 bytes ---------------------------------------------------------------------------------------------
template <typename T> constexpr int PIECE = 16 / sizeof(T);

// `count` elements of a piece (all of it from PIECE on), the others zeros
template <typename T> __device__ __forceinline__ v4i load_piece(const T *p, int64_t count)
{
    v4i raw = {0, 0, 0, 0};
    if (count >= PIECE<T>) {
        raw = load16(p);
    } else if (count > 0) {
        T e[PIECE<T>];
#pragma unroll
        for (int i = 0; i < PIECE<T>; ++i) e[i] = i < count ? p[i] : (T)0.0f;
        __builtin_memcpy(&raw, e, 16);
    }
    return raw;
}
template <typename T> __device__ __forceinline__ void piece_floats(v4i raw, float (&v)[PIECE<T>])
{
    T e[PIECE<T>];
    __builtin_memcpy(e, &raw, 16);
#pragma unroll
    for (int i = 0; i < PIECE<T>; ++i) v[i] = to_float(e[i]);
}
// (around: past the last-level cache, where it would not be when it is read next; mx_goes_around)
template <typename T> __device__ __forceinline__ void store_piece(T *p, int64_t count, const float (&v)[PIECE<T>], bool around = false)
{
    T e[PIECE<T>];
#pragma unroll
    for (int i = 0; i < PIECE<T>; ++i) e[i] = from_float<T>(v[i]);
    if (count >= PIECE<T>) {
        v4i raw;
        __builtin_memcpy(&raw, e, 16);
        if (around) __builtin_nontemporal_store(raw, (v4i_anywhere *)p);
        else store16(p, raw);
    } else {
#pragma unroll
        for (int i = 0; i < PIECE<T>; ++i)
            if (i < count) p[i] = e[i];
    }
}
// N values of a vector whose type is known at run time only, zeros behind its end
template <int N> __device__ __forceinline__ void load_floats(const void *p, int dtype, int64_t at, int64_t count, float (&v)[N])
{
    if (dtype == AMSIM_DTYPE_F32 && count >= N) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const v4f f = __builtin_bit_cast(v4f, load16((const float *)p + at + i));
#pragma unroll
            for (int e = 0; e < 4; ++e) v[i + e] = f[e];
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = i < count ? load_as_float(p, dtype, at + i) : 0.0f;
}
__device__ __forceinline__ void store_from_float(void *p, int dtype, int64_t i, float v)
{
    if (dtype == AMSIM_DTYPE_F32) ((float *)p)[i] = v;
    else if (dtype == AMSIM_DTYPE_BF16) ((__bf16 *)p)[i] = (__bf16)v;
    else ((_Float16 *)p)[i] = (_Float16)v;
}
// a piece's codes: PIECE bytes
template <int N> __device__ __forceinline__ void store_codes(uint8_t *to, const float (&v)[N], float r)
{
    uint32_t w[N / 4];
#pragma unroll
    for (int i = 0; i < N / 4; ++i) w[i] = q8_codes4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3], r);
    __builtin_memcpy(__builtin_assume_aligned(to, N), w, N);
}
template <int N> __device__ __forceinline__ void code_values(const uint32_t (&w)[N / 4], float s, float (&v)[N])
{
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = q8_value(w[i / 4], i % 4, s);
}

// ---- over the lanes that hold a row ---------------------------------------------------------------------------------
// combine(a, b) over groups of LANES lanes, the same in each; above 64 by way of LDS, one meeting a call (two halves of
// `part` in turn: who writes one has met everybody since it was read).
struct SumOf {
    static __device__ __forceinline__ float of(float a, float b) { return a + b; }
};
struct MaxOf {
    static __device__ __forceinline__ float of(float a, float b) { return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b))); }
};
template <typename Op, int CTRL> __device__ __forceinline__ float with_dpp(float v)
{
    const int other = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true);
    return Op::of(v, __builtin_bit_cast(float, other));
}
template <typename Op, int LANES> __device__ __forceinline__ float over_lanes(float v)
{
    static_assert(LANES == 16 || LANES == 64, "");
    v = with_dpp<Op, 0xb1>(v);   // the neighbour in a pair
    v = with_dpp<Op, 0x4e>(v);   // the other pair of four
    v = with_dpp<Op, 0x141>(v);  // the other four of eight (mirrored: all four hold the same)
    v = with_dpp<Op, 0x140>(v);  // the other eight of sixteen
    if constexpr (LANES == 64) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = Op::of(__uint_as_float(r[0]), __uint_as_float(r[1]));
        const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = Op::of(__uint_as_float(h[0]), __uint_as_float(h[1]));
    }
    return v;
}

template <int LANES> struct RowLanes {
    static constexpr int WAVES = LANES > 64 ? LANES / 64 : 1, WITHIN = LANES < 64 ? LANES : 64;
    float (*part)[WAVES][2];  // [2][WAVES][2], in LDS
    int turn = 0;
    template <typename A, typename B> __device__ __forceinline__ void both(float &a, float &b)
    {
        a = over_lanes<A, WITHIN>(a);
        b = over_lanes<B, WITHIN>(b);
        if constexpr (LANES > 64) {
            float (*p)[2] = part[turn];
            turn ^= 1;
            if ((threadIdx.x & 63) == 0) p[threadIdx.x >> 6][0] = a, p[threadIdx.x >> 6][1] = b;
            __syncthreads();
            a = p[0][0], b = p[0][1];
#pragma unroll
            for (int w = 1; w < WAVES; ++w) a = A::of(a, p[w][0]), b = B::of(b, p[w][1]);
        }
    }
    template <typename A> __device__ __forceinline__ float one(float a)
    {
        a = over_lanes<A, WITHIN>(a);
        if constexpr (LANES > 64) {
            float (*p)[2] = part[turn];
            turn ^= 1;
            if ((threadIdx.x & 63) == 0) p[threadIdx.x >> 6][0] = a;
            __syncthreads();
            a = p[0][0];
#pragma unroll
            for (int w = 1; w < WAVES; ++w) a = A::of(a, p[w][0]);
        }
        return a;
    }
};

}  // namespace amsim
#endif  // AMSIM_ROWS_H_
