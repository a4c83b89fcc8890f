// One AdamW step over many tensors, with the moments in 32 bits or in 8.
//
//   g = grad [* grad_scale]      m' = beta1 m + (1 - beta1) g      v' = beta2 v + ((1 - beta2) g) g
//   p' = p (1 - lr decay) - (m' / (sqrt(v') / sqrt(1 - beta2^t) + eps)) * lr / (1 - beta1^t)
//
// Every operation is one rounding in 32 bits (no contraction), in this order.  28 bytes per element with 32-bit
// parameters, gradients and moments, 16 with 8-bit moments, each read and written once.
// One launch serves as many tensors as its arguments hold: a tensor is an entry of 24 bytes, and the moments of
// all tensors lie in one buffer, each tensor from a multiple of 256 elements on, so that no table has to be
// sent to the device ahead of the kernel.  A wavefront updates one block of 256 and ends (four one after the other
// took 6% longer with 8-bit moments), and finds its tensor in two loads (a binary search over the arguments took 14%
// longer with 32-bit ones).
// 32-bit moments are bound by memory: 101M elements with 16-bit gradients 440 us, 6.0 TB/s.  With 8-bit moments the
// arithmetic has to stay out of memory's way and just about does: 25.5M elements in 161 tensors take 69 us in a row (5.9
// TB/s) and 79 behind other kernels, the vector units busy throughout (458 instructions a block).  The full divisions and
// roots of the language and shuffles through LDS took 97.
//
// 8-bit moments: a wavefront's 256 elements share a 32-bit scale, the largest magnitude among them.  m is held as
// sign, 4 bits of exponent and 3 of mantissa of |m| / scale; v as its root r = sqrt(v), which halves the binades
// to cover, with 4 and 4 bits.  A code is the upper bits of the relative magnitude's 32-bit form, rounded to nearest-even,
// counted down from 1.0 at the largest code: 16 binades.  An |m| below half the smallest code becomes 0, an
// r above 0 never does: its element would otherwise be divided by eps alone.
#include "amsim_mx.h"

#include <cmath>
#include <type_traits>

namespace amsim {

namespace {

constexpr int WG = 256;
constexpr int BLOCK = 256;             // elements that share a scale: a wavefront's
constexpr int CHUNK = 4;               // blocks of a workgroup
constexpr int TABLE = 120;             // tensors per launch (arguments: below 4 KB)

struct Entry {
    void *p;
    const void *g;
    int64_t n;
};
struct AdamWArgs {
    Entry t[TABLE];
    int first_chunk[TABLE + 1];        // workgroups before each tensor's
    int blocks_before[TABLE];          // blocks of the moments' buffer from first_block to each tensor's
    int count;
    int64_t first_block;               // of the moments' buffer, where this launch's tensors begin
    void *m, *v;
    float *m_scale, *v_scale;
    const float *grad_scale;
    float keep, beta1, grad1, beta2, grad2, inv_root2, step_size, eps;
};

// the largest of a wavefront's magnitudes (as whole numbers: a NaN is above all others), the same in every lane
__device__ __forceinline__ float wave_max(float v)
{
    uint32_t m = __float_as_uint(v);
    m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xf, 0xf, true));          // lanes 1 0 3 2 of every four
    m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x4E, 0xf, 0xf, true));          // lanes 2 3 0 1
    m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x141, 0xf, 0xf, true));         // eight lanes mirrored
    m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x140, 0xf, 0xf, true));         // sixteen mirrored
    const uint32_t a = __builtin_amdgcn_readlane(m, 0), b = __builtin_amdgcn_readlane(m, 16), c = __builtin_amdgcn_readlane(m, 32),
                   d = __builtin_amdgcn_readlane(m, 48);
    return __uint_as_float(max(max(a, b), max(c, d)));
}

// a / s, rounded as a division rounds, for 0 <= a <= s and s from 2^-60 to 2^60 of which y is the reciprocal rounded: the
// estimate is corrected by its own remainder, exact in an fma, twice (P. Markstein, "Computation of elementary functions on
// the IBM RISC System/6000 processor", 1990).  Quotients below 2^-40, where the remainder may lose bits, have no code of
// their own: a first moment's becomes 0, and a root's, 2^-75 or more unless it is 0, stays above zero.
__device__ __forceinline__ float quotient(float a, float s, float y)
{
    float q = a * y;
    q = __builtin_fmaf(__builtin_fmaf(-s, q, a), y, q);
    return __builtin_fmaf(__builtin_fmaf(-s, q, a), y, q);
}

// sqrt(x) rounded to nearest for x = 0, x >= 2^-96, infinities and NaN, by Markstein's iteration (in the same paper): g goes to
// sqrt(x) and h to 1 / (2 sqrt(x)) together from one estimate, and g's remainder, exact in an fma, corrects it.  (All floats
// of that range were compared with the root in 64 bits.  The language's root instead: 69.7 us for 68.9, 25.5M elements in 161
// tensors, and 71.5 for 67.9 in one; below 2^-96, where the remainder may lose bits, it is what is called.)
__device__ __forceinline__ float root(float x)
{
    const float y = __builtin_amdgcn_rsqf(fmaxf(x, 0x1p-126f));
    float g = x * y, h = 0.5f * y;
    const float e = __builtin_fmaf(-g, h, 0.5f);
    g = __builtin_fmaf(g, e, g);
    h = __builtin_fmaf(h, e, h);
    const float r = __builtin_fmaf(__builtin_fmaf(-g, g, x), h, g);
    return x < __builtin_inff() ? r : x;
}
// above 0 and below 2^-96
__device__ __forceinline__ bool root_is_out_of_range(float x) { return __float_as_uint(x) - 1u < 0x0f800000u - 1u; }

template <int SHIFT, int BASE> __device__ __forceinline__ float magnitude(uint32_t code)
{
    return code ? __uint_as_float((code + BASE) << SHIFT) : 0.0f;
}
template <int SHIFT, int BASE, int LARGEST> __device__ __forceinline__ uint32_t code_of(float t)
{
    const uint32_t bits = __float_as_uint(t);
    const int c = (int)((bits + ((1u << (SHIFT - 1)) - 1) + ((bits >> SHIFT) & 1)) >> SHIFT) - BASE;
    return (uint32_t)min(max(c, 1), LARGEST);
}
constexpr int M_SHIFT = 20, M_BASE = 889, M_LARGEST = 127;    // 1.0 is 1016 << 20
constexpr int R_SHIFT = 19, R_BASE = 1777, R_LARGEST = 255;   // 1.0 is 2032 << 19

__device__ __forceinline__ float m_value(uint32_t c, float scale)
{
    const float v = magnitude<M_SHIFT, M_BASE>(c & 127) * scale;
    return c & 128 ? -v : v;
}
__device__ __forceinline__ float r_value(uint32_t c, float scale) { return magnitude<R_SHIFT, R_BASE>(c) * scale; }
__device__ __forceinline__ uint32_t m_code(float m, float t)
{
    const uint32_t c = t < magnitude<M_SHIFT, M_BASE>(1) * 0.5f ? 0 : code_of<M_SHIFT, M_BASE, M_LARGEST>(t);
    return m < 0.0f ? c | 128 : c;
}
__device__ __forceinline__ uint32_t r_code(float t) { return t == 0.0f ? 0 : code_of<R_SHIFT, R_BASE, R_LARGEST>(t); }

// the codes of four magnitudes relative to `scale`, the largest of the block
template <bool ROOTS> __device__ __forceinline__ uint32_t encode4(const float (&x)[4], float scale)
{
    float t[4];
    if (scale >= 0x1p-60f && scale <= 0x1p60f) {  // (the same in all lanes)
        const float y = 1.0f / scale;
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = quotient(fabsf(x[e]), scale, y);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = scale > 0.0f ? fabsf(x[e]) / scale : 0.0f;
    }
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) w |= (ROOTS ? r_code(t[e]) : m_code(x[e], t[e])) << (8 * e);
    return w;
}

// Past the last-level cache, or through it: all that a step reads (parameters, gradients, moments) goes past it where that is
// more than it can hold, as nothing is there then when a step comes to it, and nothing it leaves there is read before it is
// displaced.  us of one tensor, through and past; in brackets where its gradients were written just before:
//   MB of a step          256          280          320          336          384          400          512
//   32 bits, f32      68/74 (88/94)              90/92 (118/115)           128/110 (147/137)          174/147 (213/182)
//   32 bits, bf16 grads       81/85 (97/101)             112/104 (125/122)
//   8 bits, f32                                  93/94 (127/127)                       121/118 (167/162)
//   8 bits, bf16 grads 82/90 (103/105)           117/113 (137/137)                                     185/180 (223/216)
// Behind 256 MB of other work (that copy's time taken in) past is quicker at all sizes: 32 bits, f32, 128 MB 96/81, 256 MB
// 139/115.
inline bool step_goes_around(double bytes) { return bytes >= 320 << 20; }
template <bool AROUND, typename V> __device__ __forceinline__ V get(const void *p)
{
    return AROUND ? __builtin_nontemporal_load((const V *)p) : *(const V *)p;
}
template <bool AROUND, typename V> __device__ __forceinline__ void put(void *p, V v)
{
    if constexpr (AROUND) __builtin_nontemporal_store(v, (V *)p);
    else *(V *)p = v;
}

// four neighbouring elements, of which `count` exist
template <typename T> using Quad = std::conditional_t<sizeof(T) == 4, v4i, v2i>;
template <bool AROUND, typename T> __device__ __forceinline__ void load4(const T *p, int count, float (&v)[4])
{
    T t[4] = {(T)0.0f, (T)0.0f, (T)0.0f, (T)0.0f};
    if (count == 4 && ((uintptr_t)p & (4 * sizeof(T) - 1)) == 0) {
        const Quad<T> q = get<AROUND, Quad<T>>(p);
        __builtin_memcpy(t, &q, sizeof(t));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < count) t[i] = p[i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = to_float(t[i]);
}
template <bool AROUND, typename T> __device__ __forceinline__ void store4(T *p, int count, const float (&v)[4])
{
    T t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = from_float<T>(v[i]);
    if (count == 4 && ((uintptr_t)p & (4 * sizeof(T) - 1)) == 0) {
        Quad<T> q;
        __builtin_memcpy(&q, t, sizeof(t));
        put<AROUND>(p, q);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < count) p[i] = t[i];
    }
}

template <typename P, typename G, bool BITS8, bool AROUND>
__global__ __launch_bounds__(WG) void adamw_kernel(AdamWArgs a)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // the tensor whose chunk this is, the last that begins at or before it: a lane looks at two of the table's entries
    const int here = (int)blockIdx.x;
    const bool first = lane < a.count && a.first_chunk[lane] <= here, second = 64 + lane < a.count && a.first_chunk[64 + lane] <= here;
    const int lo = __popcll(__builtin_amdgcn_ballot_w64(first)) + __popcll(__builtin_amdgcn_ballot_w64(second)) - 1;
    const Entry t = a.t[lo];
    const int64_t before = a.first_block + a.blocks_before[lo];
    const float scale_g = a.grad_scale ? *a.grad_scale : 1.0f;
    const int64_t b = (int64_t)((int)blockIdx.x - a.first_chunk[lo]) * CHUNK + wave;
    if (b * BLOCK >= t.n) return;
    const int64_t i = b * BLOCK + lane * 4, s = (before + b) * BLOCK + lane * 4;
    const int count = (int)(t.n - i >= 4 ? 4 : t.n - i > 0 ? t.n - i : 0);
    float p[4], g[4], m[4], v[4];
    load4<AROUND>((const P *)t.p + i, count, p);
    load4<AROUND>((const G *)t.g + i, count, g);
    uint32_t mc = 0, rc = 0;
    float ms = 0, rs = 0;
    if (BITS8) {
        mc = get<AROUND, uint32_t>((const uint8_t *)a.m + s);
        rc = get<AROUND, uint32_t>((const uint8_t *)a.v + s);
        ms = a.m_scale[before + b];
        rs = a.v_scale[before + b];
    } else {
        const v4f mv = get<AROUND, v4f>((const float *)a.m + s), vv = get<AROUND, v4f>((const float *)a.v + s);
#pragma unroll
        for (int e = 0; e < 4; ++e) m[e] = mv[e], v[e] = vv[e];
    }
    float r[4];
    bool small = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (BITS8) {
            m[e] = m_value((mc >> (8 * e)) & 255, ms);
            v[e] = r_value((rc >> (8 * e)) & 255, rs);
            v[e] = v[e] * v[e];
        }
        if (a.grad_scale) g[e] = g[e] * scale_g;
        m[e] = m[e] * a.beta1 + g[e] * a.grad1;
        v[e] = v[e] * a.beta2 + (g[e] * a.grad2) * g[e];
        small |= root_is_out_of_range(v[e]);
    }
    if (!BITS8 || __builtin_amdgcn_ballot_w64(small)) {  // (the same in all lanes)
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = sqrtf(v[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = root(v[e]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float denominator = r[e] * a.inv_root2 + a.eps;
        p[e] = p[e] * a.keep - (m[e] / denominator) * a.step_size;
    }
    store4<AROUND>((P *)t.p + i, count, p);
    if (BITS8) {
        uint32_t mx = 0, rx = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (e >= count) m[e] = r[e] = 0.0f;
            mx = max(mx, __float_as_uint(fabsf(m[e])));
            rx = max(rx, __float_as_uint(fabsf(r[e])));
        }
        ms = wave_max(__uint_as_float(mx));
        rs = wave_max(__uint_as_float(rx));
        mc = encode4<false>(m, ms);
        rc = encode4<true>(r, rs);
        put<AROUND>((uint8_t *)a.m + s, mc);
        put<AROUND>((uint8_t *)a.v + s, rc);
        if (lane == 0) {
            a.m_scale[before + b] = ms;
            a.v_scale[before + b] = rs;
        }
    } else {
        v4f mv, vv;
#pragma unroll
        for (int e = 0; e < 4; ++e) mv[e] = e < count ? m[e] : 0.0f, vv[e] = e < count ? v[e] : 0.0f;
        put<AROUND>((float *)a.m + s, mv);
        put<AROUND>((float *)a.v + s, vv);
    }
}

template <bool ROOTS>
__global__ __launch_bounds__(WG) void state_values_kernel(const uint8_t *codes, const float *scales, int64_t quads, float *out)
{
    const int64_t q = (int64_t)blockIdx.x * WG + threadIdx.x;
    if (q >= quads) return;
    const uint32_t c = ((const uint32_t *)codes)[q];
    const float s = scales[q / (BLOCK / 4)];
    v4f v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = ROOTS ? r_value((c >> (8 * e)) & 255, s) : m_value((c >> (8 * e)) & 255, s);
    ((v4f *)out)[q] = v;
}

template <typename P, typename G> void launch_adamw(const AdamWArgs &a, int state_bits, bool around, hipStream_t stream)
{
    const auto kernel = state_bits == 8 ? (around ? adamw_kernel<P, G, true, true> : adamw_kernel<P, G, true, false>)
                                        : (around ? adamw_kernel<P, G, false, true> : adamw_kernel<P, G, false, false>);
    kernel<<<(unsigned)a.first_chunk[a.count], WG, 0, stream>>>(a);
}
template <typename P> void launch_adamw_grad(const AdamWArgs &a, int grad_dtype, int state_bits, bool around, hipStream_t stream)
{
    switch (grad_dtype) {
    case AMSIM_DTYPE_F32: launch_adamw<P, float>(a, state_bits, around, stream); break;
    case AMSIM_DTYPE_BF16: launch_adamw<P, __bf16>(a, state_bits, around, stream); break;
    default: launch_adamw<P, _Float16>(a, state_bits, around, stream); break;
    }
}

}  // namespace

}  // namespace amsim

using namespace amsim;

extern "C" {

int amsim_adamw_step(int count, void *const *params, const void *const *grads, const int64_t *sizes, int param_dtype, int grad_dtype,
                     int state_bits, void *m, void *v, float *m_scale, float *v_scale, const amsim_adamw_hyper *hyper,
                     const float *grad_scale, void *stream)
{
    if (!known_dtype(param_dtype) || !known_dtype(grad_dtype)) return fail(AMSIM_ERR_INVALID, "adamw: unknown element type");
    if (state_bits != 32 && state_bits != 8) return fail(AMSIM_ERR_INVALID, "adamw: states have 32 or 8 bits");
    if (count < 0 || !hyper || (count && (!params || !grads || !sizes))) return fail(AMSIM_ERR_INVALID, "adamw: negative count or null pointer");
    const double lr = hyper->lr, beta1 = hyper->beta1, beta2 = hyper->beta2, eps = hyper->eps, weight_decay = hyper->weight_decay;
    const int64_t step = hyper->step;
    if (step < 1) return fail(AMSIM_ERR_INVALID, "adamw: step below 1");
    if (!(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0 && eps >= 0.0)) return fail(AMSIM_ERR_INVALID, "adamw: betas or eps out of range");
    int64_t all_blocks = 0, stepped = 0;  // (stepped: of tensors that have gradients)
    for (int i = 0; i < count; ++i) {
        if (sizes[i] < 0) return fail(AMSIM_ERR_INVALID, "adamw: negative size");
        if (sizes[i] && !params[i]) return fail(AMSIM_ERR_INVALID, "adamw: null pointer");
        if (((uintptr_t)params[i] & (element_bytes(param_dtype) - 1)) || ((uintptr_t)grads[i] & (element_bytes(grad_dtype) - 1)))
            return fail(AMSIM_ERR_INVALID, "adamw: misaligned pointer");
        if (sizes[i] > (1ll << 33)) return fail(AMSIM_ERR_UNSUPPORTED, "adamw: tensor of more than 2^33 elements");
        all_blocks += ceil_div64(sizes[i], BLOCK);
        if (grads[i]) stepped += ceil_div64(sizes[i], BLOCK);
    }
    if (all_blocks == 0) return AMSIM_OK;
    if (!m || !v || (state_bits == 8 && (!m_scale || !v_scale))) return fail(AMSIM_ERR_INVALID, "adamw: null pointer");
    if (((uintptr_t)m & 15) || ((uintptr_t)v & 15)) return fail(AMSIM_ERR_INVALID, "adamw: misaligned pointer");
    AdamWArgs a{};
    a.m = m, a.v = v, a.m_scale = m_scale, a.v_scale = v_scale, a.grad_scale = grad_scale;
    a.keep = (float)(1.0 - lr * weight_decay);
    a.beta1 = (float)beta1, a.grad1 = (float)(1.0 - beta1), a.beta2 = (float)beta2, a.grad2 = (float)(1.0 - beta2);
    a.inv_root2 = (float)(1.0 / std::sqrt(1.0 - std::pow(beta2, (double)step)));
    a.step_size = (float)(lr / (1.0 - std::pow(beta1, (double)step)));
    a.eps = (float)eps;
    const bool around = step_goes_around((double)stepped * BLOCK * (element_bytes(param_dtype) + element_bytes(grad_dtype) + (state_bits == 8 ? 2 : 8)));
    int64_t block = 0;
    for (int i = 0; i < count;) {
        a.count = 0;
        a.first_block = block;
        int64_t here = 0, blocks = 0;
        for (; i < count && a.count < TABLE; ++i) {
            const int64_t n = ceil_div64(sizes[i], BLOCK), c = ceil_div64(n, CHUNK);
            if (here + c >= (1ll << 24) || blocks + n >= (1ll << 31)) break;
            if (sizes[i] && grads[i]) {
                a.t[a.count] = Entry{params[i], grads[i], sizes[i]};
                a.blocks_before[a.count] = (int)blocks;
                a.first_chunk[a.count++] = (int)here;
                here += c;
            }
            blocks += n;
        }
        block += blocks;
        a.first_chunk[a.count] = (int)here;
        if (a.count == 0) continue;
        switch (param_dtype) {
        case AMSIM_DTYPE_F32: launch_adamw_grad<float>(a, grad_dtype, state_bits, around, (hipStream_t)stream); break;
        case AMSIM_DTYPE_BF16: launch_adamw_grad<__bf16>(a, grad_dtype, state_bits, around, (hipStream_t)stream); break;
        default: launch_adamw_grad<_Float16>(a, grad_dtype, state_bits, around, (hipStream_t)stream); break;
        }
        AMSIM_HIP_CHECK(hipGetLastError());
    }
    return AMSIM_OK;
}

int amsim_adamw_state_values(const void *codes, const float *scales, int64_t blocks, int roots, float *out, void *stream)
{
    if (blocks < 0) return fail(AMSIM_ERR_INVALID, "adamw: negative size");
    if (!codes || !scales || !out) return fail(AMSIM_ERR_INVALID, "adamw: null pointer");
    if (blocks == 0) return AMSIM_OK;
    if (((uintptr_t)codes & 3) || ((uintptr_t)out & 15)) return fail(AMSIM_ERR_INVALID, "adamw: misaligned pointer");
    const int64_t quads = blocks * (BLOCK / 4), groups = ceil_div64(quads, WG);
    if (groups >= (1ll << 24)) return fail(AMSIM_ERR_UNSUPPORTED, "adamw: more blocks than one launch takes");
    if (roots) state_values_kernel<true><<<(unsigned)groups, WG, 0, (hipStream_t)stream>>>((const uint8_t *)codes, scales, quads, out);
    else state_values_kernel<false><<<(unsigned)groups, WG, 0, (hipStream_t)stream>>>((const uint8_t *)codes, scales, quads, out);
    AMSIM_HIP_CHECK(hipGetLastError());
    return AMSIM_OK;
}

}  // extern "C"
