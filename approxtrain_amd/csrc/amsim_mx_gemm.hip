// Products of MXFP4 operands (amsim_mx.h) on the matrix cores: out[m][n] = act(sum_k a[m][k] b[n][k] + bias[n]).
//
// A 16x16x128 instruction takes 16 bytes of codes and one scale from each lane: a lane's operand is one block of
// 32 values, which is what the storage hands out.  The product of two elements is exact, and so are the sums
// within an instruction but for bits far below the largest term; steps add up in 32 bits.  The operands are
// swapped in the instruction (b's rows are its rows) so that a lane ends up with four neighbouring columns.
#include "amsim_mx.h"

#include <algorithm>

namespace amsim {

namespace {

constexpr int WG = 256;

struct Operand {
    const uint8_t *codes, *scales;
    int64_t rows, fragments, groups;  // of 16 and of 64 rows
};
inline Operand operand(const void *q, int64_t rows, int64_t length)
{
    const uint8_t *p = (const uint8_t *)q;
    return Operand{p, p + mx_code_bytes(rows, length), rows, ceil_div64(rows, 16), ceil_div64(rows, 64)};
}

struct GemmArgs {
    Operand a, b;
    int64_t steps, steps_per_split;
    const void *bias;
    int bias_dtype, act, out_dtype;
    void *out;
    float *partial;  // [splits][m][n] where the reduction is split, else null
    int64_t tiles_n;
};

template <typename T>
__device__ __forceinline__ void store4(T *o, const float (&v)[4], int count, bool vector)
{
    T t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = from_float<T>(v[i]);
    if (count == 4 && vector) {
        __builtin_memcpy(__builtin_assume_aligned(o, 4 * sizeof(T)), t, sizeof(t));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < count) o[i] = t[i];
    }
}

// columns n .. n + 3 of row m, bias and activation included
__device__ __forceinline__ void finish4(const GemmArgs &g, int64_t m, int64_t n, float (&v)[4])
{
    const int64_t N = g.b.rows;
    const int count = (int)(N - n < 4 ? N - n : 4);
    const bool vector = N % 4 == 0;
    if (g.partial) {
        store4(g.partial + ((int64_t)blockIdx.y * g.a.rows + m) * N + n, v, count, vector);
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (g.bias && i < count) v[i] += load_as_float(g.bias, g.bias_dtype, n + i);
        v[i] = activate(v[i], g.act);
    }
    if (g.out_dtype == AMSIM_DTYPE_F32) store4((float *)g.out + m * N + n, v, count, vector);
    else if (g.out_dtype == AMSIM_DTYPE_BF16) store4((__bf16 *)g.out + m * N + n, v, count, vector);
    else store4((_Float16 *)g.out + m * N + n, v, count, vector);
}

template <int SA, int SB> __device__ __forceinline__ v4f mfma(v4i a, v4i b, v4f c, int sa, int sb)
{
    const v8i wa = {a[0], a[1], a[2], a[3], 0, 0, 0, 0}, wb = {b[0], b[1], b[2], b[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wa, wb, c, 4, 4, SA, sa, SB, sb);
}

// Fragments straight from memory to registers: 2 x 2 waves of F x F fragments each.
template <int F>
__global__ __launch_bounds__(WG) void gemm_kernel(GemmArgs g)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t tm = (int64_t)blockIdx.x / g.tiles_n, tn = (int64_t)blockIdx.x % g.tiles_n;
    const int64_t fa = (tm * 2 + wave / 2) * F, fb = (tn * 2 + wave % 2) * F;
    const int64_t beg = blockIdx.y * g.steps_per_split, end = min(beg + g.steps_per_split, g.steps);
    const uint8_t *pa[F], *pb[F], *sa[F], *sb[F];
#pragma unroll
    for (int i = 0; i < F; ++i) {
        const int64_t f = min(fa + i, g.a.fragments - 1), h = min(fb + i, g.b.fragments - 1);
        pa[i] = g.a.codes + (f * g.steps * 64 + lane) * 16;
        pb[i] = g.b.codes + (h * g.steps * 64 + lane) * 16;
        sa[i] = g.a.scales + (f / 4 * g.steps * 64 + lane) * 4 + f % 4;
        sb[i] = g.b.scales + (h / 4 * g.steps * 64 + lane) * 4 + h % 4;
    }
    v4f acc[F][F] = {};
    for (int64_t s = beg; s < end; ++s) {
        v4i a[F], b[F];
        int ca[F], cb[F];
#pragma unroll
        for (int i = 0; i < F; ++i) {
            a[i] = *(const v4i *)(pa[i] + s * 1024);
            b[i] = *(const v4i *)(pb[i] + s * 1024);
            ca[i] = sa[i][s * 256];
            cb[i] = sb[i][s * 256];
        }
#pragma unroll
        for (int i = 0; i < F; ++i)
#pragma unroll
            for (int j = 0; j < F; ++j) acc[i][j] = mfma<0, 0>(b[j], a[i], acc[i][j], cb[j], ca[i]);
    }
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
        for (int j = 0; j < F; ++j) {
            const int64_t m = (fa + i) * 16 + lane % 16, n = (fb + j) * 16 + lane / 16 * 4;
            if (m >= g.a.rows || n >= g.b.rows) continue;
            float v[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
            finish4(g, m, n, v);
        }
}

// The partial sums of a split reduction, added in the order of the splits.
__global__ __launch_bounds__(WG) void gemm_reduce_kernel(GemmArgs g, int splits)
{
    const int64_t N = g.b.rows, quads = ceil_div64(N, 4), at = (int64_t)blockIdx.x * WG + threadIdx.x;
    if (at >= g.a.rows * quads) return;
    const int64_t m = at / quads, n = at % quads * 4;
    const int count = (int)(N - n < 4 ? N - n : 4);
    float v[4] = {0, 0, 0, 0};
    for (int s = 0; s < splits; ++s) {
        const float *p = g.partial + ((int64_t)s * g.a.rows + m) * N + n;
        if (N % 4 == 0) {
            const v4f q = *(const v4f *)p;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] += q[i];
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i < count) v[i] += p[i];
        }
    }
    GemmArgs h = g;
    h.partial = nullptr;
    finish4(h, m, n, v);
}

struct Plan {
    int fragments;  // per wave and direction
    int64_t tiles_m, tiles_n, splits, steps_per_split;
};

Plan plan(int64_t m, int64_t n, int64_t k)
{
    Plan p{};
    const int64_t steps = mx_steps(k);
    for (int f = 4; f >= 1; f /= 2) {
        p.fragments = f;
        p.tiles_m = ceil_div64(m, 32 * f);
        p.tiles_n = ceil_div64(n, 32 * f);
        if (p.tiles_m * p.tiles_n >= 256) break;
    }
    const int64_t tiles = p.tiles_m * p.tiles_n;
    p.splits = std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(512 / tiles, steps / 8), 16));
    p.steps_per_split = ceil_div64(steps, p.splits);
    p.splits = ceil_div64(steps, p.steps_per_split);
    return p;
}

size_t product_workspace(int64_t m, int64_t n, int64_t k)
{
    const Plan p = plan(m, n, k);
    return p.splits > 1 ? (size_t)p.splits * m * n * 4 : 0;
}

int product(const Operand &a, const Operand &b, int64_t k, const void *bias, int bias_dtype, int act, void *out, int out_dtype,
            void *workspace, hipStream_t stream)
{
    const Plan p = plan(a.rows, b.rows, k);
    const int64_t tiles = p.tiles_m * p.tiles_n, quads = a.rows * ceil_div64(b.rows, 4);
    if (tiles >= (1ll << 24)) return fail(AMSIM_ERR_UNSUPPORTED, "mxfp4: more tiles than one launch takes");
    GemmArgs g{a, b, mx_steps(k), p.steps_per_split, bias, bias_dtype, act, out_dtype, out,
               p.splits > 1 ? (float *)workspace : nullptr, p.tiles_n};
    const dim3 grid((unsigned)tiles, (unsigned)p.splits);
    switch (p.fragments) {
    case 4: gemm_kernel<4><<<grid, WG, 0, stream>>>(g); break;
    case 2: gemm_kernel<2><<<grid, WG, 0, stream>>>(g); break;
    default: gemm_kernel<1><<<grid, WG, 0, stream>>>(g); break;
    }
    AMSIM_HIP_CHECK(hipGetLastError());
    if (p.splits > 1) {
        gemm_reduce_kernel<<<(unsigned)ceil_div64(quads, WG), WG, 0, stream>>>(g, (int)p.splits);
        AMSIM_HIP_CHECK(hipGetLastError());
    }
    return AMSIM_OK;
}

int check_product(int64_t m, int64_t n, int64_t k, const void *bias, int bias_dtype, int act, const void *out, int out_dtype)
{
    if (!known_dtype(out_dtype) || (bias && !known_dtype(bias_dtype))) return fail(AMSIM_ERR_INVALID, "mxfp4: unknown element type");
    if (act != AMSIM_ACT_NONE && act != AMSIM_ACT_RELU) return fail(AMSIM_ERR_INVALID, "mxfp4: unknown activation");
    if (!mx_extents_fit(m, k) || !mx_extents_fit(n, k) || !mx_extents_fit(m, n)) return fail(AMSIM_ERR_UNSUPPORTED, "mxfp4: extents out of range");
    if (m == 0 || n == 0 || k == 0) return fail(AMSIM_ERR_INVALID, "mxfp4: empty product");
    if (!out) return fail(AMSIM_ERR_INVALID, "mxfp4: null pointer");
    if ((uintptr_t)out & 15) return fail(AMSIM_ERR_INVALID, "mxfp4: misaligned pointer");
    if (bias && ((uintptr_t)bias & (element_bytes(bias_dtype) - 1))) return fail(AMSIM_ERR_INVALID, "mxfp4: misaligned pointer");
    return AMSIM_OK;
}

int check_workspace(const void *workspace, size_t have, size_t need)
{
    if (need && (!workspace || have < need || ((uintptr_t)workspace & 255))) return fail(AMSIM_ERR_WORKSPACE, "mxfp4: workspace missing, misaligned or too small");
    return AMSIM_OK;
}

// bytes of the quantised activations at the start of amsim_mxfp4_linear's workspace
size_t activation_bytes(int64_t m, int64_t k) { return (size_t)(mx_code_bytes(m, k) + mx_scale_bytes(m, k)); }

}  // namespace

}  // namespace amsim

using namespace amsim;

extern "C" {

size_t amsim_mxfp4_matmul_workspace_bytes(int64_t m, int64_t n, int64_t k)
{
    return mx_extents_fit(m, k) && mx_extents_fit(n, k) && mx_extents_fit(m, n) && m && n && k ? product_workspace(m, n, k) : 0;
}

int amsim_mxfp4_matmul(const void *a, const void *b, int64_t m, int64_t n, int64_t k, const void *bias, int bias_dtype, int act,
                       void *out, int out_dtype, void *workspace, size_t workspace_bytes, void *stream)
{
    if (int rc = check_product(m, n, k, bias, bias_dtype, act, out, out_dtype)) return rc;
    if (!a || !b) return fail(AMSIM_ERR_INVALID, "mxfp4: null pointer");
    if (((uintptr_t)a & 15) || ((uintptr_t)b & 15)) return fail(AMSIM_ERR_INVALID, "mxfp4: misaligned pointer");
    if (int rc = check_workspace(workspace, workspace_bytes, product_workspace(m, n, k))) return rc;
    return product(operand(a, m, k), operand(b, n, k), k, bias, bias_dtype, act, out, out_dtype, workspace, (hipStream_t)stream);
}

size_t amsim_mxfp4_linear_workspace_bytes(int64_t m, int64_t n, int64_t k)
{
    if (!(mx_extents_fit(m, k) && mx_extents_fit(n, k) && mx_extents_fit(m, n) && m && n && k)) return 0;
    return activation_bytes(m, k) + product_workspace(m, n, k);
}

int amsim_mxfp4_linear(const void *x, int dtype, int64_t row_stride, const void *w, int64_t m, int64_t n, int64_t k, const void *bias,
                       int bias_dtype, int act, void *out, void *workspace, size_t workspace_bytes, void *stream)
{
    if (int rc = check_product(m, n, k, bias, bias_dtype, act, out, dtype)) return rc;
    if (!x || !w) return fail(AMSIM_ERR_INVALID, "mxfp4: null pointer");
    if (row_stride < k && m > 1) return fail(AMSIM_ERR_INVALID, "mxfp4: rows overlap");
    if (((uintptr_t)x & (element_bytes(dtype) - 1)) || ((uintptr_t)w & 15)) return fail(AMSIM_ERR_INVALID, "mxfp4: misaligned pointer");
    if (int rc = check_workspace(workspace, workspace_bytes, amsim_mxfp4_linear_workspace_bytes(m, n, k))) return rc;
    if (int rc = mx_quantize(x, dtype, m, k, row_stride, workspace, nullptr, (hipStream_t)stream)) return rc;
    return product(operand(workspace, m, k), operand(w, n, k), k, bias, bias_dtype, act, out, dtype,
                   (char *)workspace + activation_bytes(m, k), (hipStream_t)stream);
}

}  // extern "C"
