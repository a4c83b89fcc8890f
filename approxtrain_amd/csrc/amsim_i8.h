// Operands of the products in 8-bit integers: storage, and the conversions that write it.
//
// A tensor of `rows` x `length` values has a scale for every row (the length is the reduction axis of a product); codes and
// scale are those of amsim_rows.h (Q).  Storage follows the operands of the 16x16x64 matrix instruction, so that a
// wavefront's loads are whole lines wherever they come from:
//   codes   [rows / 16][length / 64][64 lanes][16 bytes]   lane = 16 * (16 values within the 64) + row % 16
//   scales  [rows] floats, right behind them
// with extents rounded up.  Codes beyond the length and beyond the last row are zeros: equal values are equal bytes.
#ifndef AMSIM_I8_H_
#define AMSIM_I8_H_

#include "amsim_rows.h"

namespace amsim {

constexpr int I8_STEP = 64;
constexpr int64_t I8_MOST_STEPS = 131072 / I8_STEP;  // of one sum: 127^2 * 131072 < 2^31
__host__ __device__ inline int64_t i8_steps(int64_t length) { return ceil_div64(length, I8_STEP); }
__host__ __device__ inline int64_t i8_code_bytes(int64_t rows, int64_t length) { return ceil_div64(rows, 16) * i8_steps(length) * 1024; }
inline int64_t i8_bytes(int64_t rows, int64_t length) { return i8_code_bytes(rows, length) + 4 * rows; }

// Converts x[rows][cols].  By rows: scales over a row (of x col_factor where that is given), codes to an operand of the
// rows, of the columns, or both.  By columns: scales over a column (of row_factor x), the same, and the columns' sums.
struct I8Rows {
    const void *x, *positive;        // positive: [rows][cols] of x's type, or null: where it is not above zero x counts as zero
    int dtype;
    int64_t rows, cols, row_stride;  // row_stride in elements
    const float *col_factor;         // or null
    uint8_t *by_rows, *by_columns;   // codes, or null
    float *scales;                   // [rows]
};
struct I8Columns {
    const void *x, *positive;
    int dtype;
    int64_t rows, cols, row_stride;
    const float *row_factor;         // or null: ones
    uint8_t *by_rows, *by_columns;   // both null: sums alone
    float *scales;                   // [cols]
    void *sums;                      // [cols] of sums_dtype, or null: of x
    int sums_dtype;
};
// Either or both (of one tensor or two), null where there is none: a launch that converts the rows and looks through the
// columns, and one that converts the columns.  partial: i8_partial_floats of the columns' extents.
int64_t i8_partial_floats(int64_t rows, int64_t cols);
int i8_convert(const I8Rows *rows, const I8Columns *columns, float *partial, hipStream_t stream);

inline bool i8_extents_fit(int64_t rows, int64_t length) { return mx_extents_fit(rows, length) && length <= 16 * I8_MOST_STEPS * I8_STEP; }

}  // namespace amsim

// For tests: how the products of one call would run, as amsim_mxfp4_plan (amsim_mx.h).
extern "C" int amsim_i8_plan(int count, const int64_t *extents, int64_t *info);
#endif  // AMSIM_I8_H_
